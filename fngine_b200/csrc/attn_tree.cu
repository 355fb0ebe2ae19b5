// Attention of a few drafted tokens per sequence over a paged cache (one token per sequence: plain decoding).
//
//   out[i] = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that token i sees: all ctx keys of the context, and of the
//   drafted tokens, whose keys follow the context's in the cache, those in its mask.
//
// Bound by the cache's bytes: each key and value is read once for all rows (tokens x query heads of a group) of a key head. Up to
// 128 rows are a block's row tile; the tiles of keys of all (sequence, key head, row tile) segments are one sequence that is cut
// evenly over the multiprocessors, so that sequences of different lengths leave none of them idle, whatever lengths the
// device finds (the host does not know them). A segment that several blocks share is joined by the last of them to arrive, in
// block order: results do not depend on timing. Inside a block RW warps share the rows and 8 / RW the keys of a tile; with few rows
// every warp has 16 keys of its own and the warps' running maxima, sums and outputs meet once per segment. Keys arrive by
// cp.async some tiles ahead; the products are mma.sync m16n8k16: at 16 to 128 rows per key they need 2 to 13 % of what tcgen05
// gives, and fragments in registers spare the trip of scores and weights through tensor memory.
#include "attn_common.cuh"

namespace fb {
namespace {

constexpr int kTreeWarps = 8;
constexpr int kTreeThreads = 32 * kTreeWarps;
constexpr int kTreeMaxDrafted = 64;
constexpr int kTreeMaxSms = 256;  // partial results are sized for this many blocks

struct TreeArgs {
  const void* q;
  void* out;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* contexts;
  const uint64_t* mask;
  int64_t q_stride, out_stride;  // elements between tokens
  int64_t n_pages;
  int64_t table_stride;
  int32_t* counters;  // [segments]
  float* partial;     // [2 * blocks][16 RW][D + 2]
  float scale_log2;
  int n_seqs, drafted, kv_heads, group, page_size, page_shift, row_tiles;
};

__device__ __forceinline__ void tree_cp16(uint32_t dst, const void* src, bool there) {
  // (a source size of zero writes zeros and reads nothing)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void tree_cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tree_ldm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tree_ldm_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <class T>
__device__ __forceinline__ void tree_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, int RW>
struct TreeShape {
  static constexpr int kKeys = RW <= 2 ? 128 : 64;  // keys per tile
  static constexpr int kStages = RW <= 2 ? 3 : 4;
  static constexpr int kKeyWarps = kTreeWarps / RW;
  static constexpr int kWarpKeys = kKeys / kKeyWarps;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kMergeWords = (D / 2 + 4) * 32;  // a warp's outputs, maxima and sums
  static constexpr int kMergeBytes = (kKeyWarps > 1 ? kTreeWarps / 2 : 1) * kMergeWords * 4;
  static constexpr int kSmem = kStages * 2 * kTileBytes + kMergeBytes;
};

// Walks through the tiles of the segments in their order.
struct TreeCursor {
  int seq, part, tile;       // part: key head * row tiles + row tile
  int tiles, ctx, length;    // of the sequence
  uint64_t seen;             // drafted tokens that some token of the sequence sees
};

template <class T, int D, int RW>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_kernel(const TreeArgs a) {
  using S = TreeShape<D, RW>;
  constexpr int kKeys = S::kKeys, kStages = S::kStages, kKeyWarps = S::kKeyWarps, kWarpKeys = S::kWarpKeys;
  constexpr int kChunks = D / 8;                         // 16-byte chunks of a key
  constexpr int kRowsPerPass = kTreeThreads / kChunks;   // keys per pass of the copying threads
  constexpr int kPasses = kKeys / kRowsPerPass;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + kStages * 2 * S::kTileBytes);
  __shared__ int last_block;
  __shared__ int64_t found[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rw = warp / kKeyWarps, kw = warp % kKeyWarps;
  const int parts = a.kv_heads * a.row_tiles, rows_all = a.drafted * a.group;
  const int64_t room = a.table_stride * a.page_size;  // keys that the table can hold
  pdl_wait_prior();
  pdl_launch_dependents();

  auto length_of = [&](int seq, int* ctx) {
    int c = a.contexts[seq];
    c = c < 0 ? 0 : c;
    if (c > room) c = int(room);
    *ctx = c;
    const int64_t n = int64_t(c) + a.drafted;
    return int(n < room ? n : room);
  };
  auto tiles_of = [&](int seq) {
    int c;
    const int n = (length_of(seq, &c) + kKeys - 1) / kKeys;
    return n > 0 ? n : 1;
  };

  // All tiles, and the sequence that this block's first one lies in.
  int64_t total = 0;
  {
    int64_t* sums = reinterpret_cast<int64_t*>(merge);
    int64_t mine = 0;
    for (int s = tid; s < a.n_seqs; s += kTreeThreads) mine += tiles_of(s);
#pragma unroll
    for (int m = 16; m; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    for (int w = 0; w < kTreeWarps; ++w) total += sums[w];
    __syncthreads();
  }
  total *= parts;
  const int blocks = int(total < int64_t(gridDim.x) ? total : int64_t(gridDim.x));
  if (int(blockIdx.x) >= blocks) return;
  const int64_t begin = int64_t(blockIdx.x) * total / blocks, end = int64_t(blockIdx.x + 1) * total / blocks;
  int64_t seq_begin = 0;  // first tile of the sequence of the products' cursor
  {
    int64_t* sums = reinterpret_cast<int64_t*>(merge);
    int64_t before = 0;
    for (int base = 0; base < a.n_seqs; base += kTreeThreads) {
      const int s = base + tid;
      const int64_t n = s < a.n_seqs ? int64_t(tiles_of(s)) * parts : 0;
      int64_t upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t other = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += other;
      }
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      int64_t all = 0;
      for (int w = 0; w < kTreeWarps; ++w) {
        if (w < warp) upto += sums[w];
        all += sums[w];
      }
      if (n && before + upto > begin && before + upto - n <= begin) {
        found[0] = s;
        found[1] = before + upto - n;
      }
      before += all;
      __syncthreads();
      if (before > begin) break;
    }
  }
  auto enter = [&](TreeCursor& c) {
    c.length = length_of(c.seq, &c.ctx);
    const int n = (c.length + kKeys - 1) / kKeys;
    c.tiles = n > 0 ? n : 1;
    c.seen = 0;
    if (a.mask) {
      uint64_t m = 0;
      for (int i = lane; i < a.drafted; i += 32) m |= a.mask[int64_t(c.seq) * a.drafted + i];
      const uint32_t lo = __reduce_or_sync(0xffffffffu, uint32_t(m)), hi = __reduce_or_sync(0xffffffffu, uint32_t(m >> 32));
      c.seen = (uint64_t(hi) << 32) | lo;
    } else {
      c.seen = ~0ull;
    }
  };
  auto advance = [&](TreeCursor& c) {  // true: a new segment
    if (++c.tile < c.tiles) return false;
    c.tile = 0;
    if (++c.part == parts) {
      c.part = 0;
      ++c.seq;
      if (c.seq < a.n_seqs) enter(c);
    }
    return true;
  };

  TreeCursor now;
  now.seq = int(found[0]);
  seq_begin = found[1];
  enter(now);
  now.part = int((begin - seq_begin) / now.tiles);
  now.tile = int((begin - seq_begin) % now.tiles);
  TreeCursor ahead = now;
  const int n_tiles = int(end - begin);

  // Page numbers of the tile to be copied next: asked for a tile before they are used.
  const int my_chunk = tid % kChunks, my_row = tid / kChunks;
  int pages[kPasses];
  auto ask = [&] {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int key = ahead.tile * kKeys + i * kRowsPerPass + my_row;
      const int d = key - ahead.ctx;
      const bool seen = key < ahead.length && (d < 0 || ((ahead.seen >> (d & 63)) & 1));
      const int index = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
      pages[i] = seen ? a.table[ahead.seq * a.table_stride + index] : -1;
    }
  };
  const uint32_t ring = smem_u32(smem);
  const size_t key_elems = size_t(a.kv_heads) * D;
  int asked = 0, put_stage = 0;
  auto copy = [&] {
    if (asked < n_tiles) {
      const uint32_t stage = ring + put_stage * (2 * S::kTileBytes);
      const size_t head = size_t(ahead.part / a.row_tiles) * D + my_chunk * 8;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int row = i * kRowsPerPass + my_row, key = ahead.tile * kKeys + row;
        const int index = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
        // A page outside of the cache reads as zeros, as does a drafted token that nobody sees.
        const bool there = pages[i] >= 0 && pages[i] < a.n_pages;
        const size_t at = there ? (size_t(pages[i]) * a.page_size + size_t(key - index * a.page_size)) * key_elems + head : 0;
        const uint32_t dst = stage + row * (D * 2) + ((my_chunk ^ (row & 7)) << 4);
        tree_cp16(dst, static_cast<const T*>(a.k) + at, there);
        tree_cp16(dst + S::kTileBytes, static_cast<const T*>(a.v) + at, there);
      }
      ++asked;
      if (asked < n_tiles) {
        advance(ahead);
        ask();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put_stage = put_stage + 1 == kStages ? 0 : put_stage + 1;
  };
  ask();
  for (int i = 0; i < kStages - 1; ++i) copy();

  uint32_t qf[D / 16][4];
  float o[D / 8][4], m_run[2], l_run[2];
  uint64_t row_mask[2];
  auto begin_segment = [&] {
    const int head0 = (now.part / a.row_tiles) * a.group, row0 = (now.part % a.row_tiles) * (16 * RW) + rw * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + g + 8 * i, token = row / a.group, head = head0 + row - token * a.group;
      const bool real = row < rows_all;
      const T* p = static_cast<const T*>(a.q) + (int64_t(now.seq) * a.drafted + token) * a.q_stride + head * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][i] = real ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 2 * t) : 0u;
        qf[kk][i + 2] = real ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 8 + 2 * t) : 0u;
      }
      row_mask[i] = !real ? 0 : a.mask ? a.mask[int64_t(now.seq) * a.drafted + token]
                                       : token == 63 ? ~0ull : (2ull << token) - 1;
      m_run[i] = -INFINITY;
      l_run[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  };
  begin_segment();

  int stage_at = 0;
  int64_t piece_begin = begin;
  const int lr = (lane & 7) + ((lane >> 4) & 1) * 8, lc = (lane >> 3) & 1;    // K: keys 0-7 | 8-15 by chunk c | c + 1
  const int vr = (lane & 7) + ((lane >> 3) & 1) * 8, vc = (lane >> 4) & 1;    // V: chunk c | c + 1 by keys 0-7 | 8-15
  for (int it = 0; it < n_tiles; ++it) {
    tree_cp_wait<kStages - 2>();
    __syncthreads();
    copy();
    const uint32_t ks = ring + stage_at * (2 * S::kTileBytes) + kw * kWarpKeys * (D * 2), vs = ks + S::kTileBytes;
    stage_at = stage_at + 1 == kStages ? 0 : stage_at + 1;

    float s[kWarpKeys / 8][4];
#pragma unroll
    for (int i = 0; i < kWarpKeys / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int n2 = 0; n2 < kWarpKeys / 16; ++n2) {
        uint32_t b[4];
        const int row = n2 * 16 + lr;
        tree_ldm(b, ks + row * (D * 2) + (((2 * kk + lc) ^ (row & 7)) << 4));
        tree_mma<T>(s[2 * n2], qf[kk], b[0], b[1]);
        tree_mma<T>(s[2 * n2 + 1], qf[kk], b[2], b[3]);
      }
    }
    const int key0 = now.tile * kKeys + kw * kWarpKeys;
    if (key0 + kWarpKeys > now.ctx) {
#pragma unroll
      for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + n * 8 + 2 * t + (j & 1), d = key - now.ctx;
          const bool sees = key < now.length && (d < 0 || ((row_mask[j >> 1] >> (d & 63)) & 1));
          if (!sees) s[n][j] = -INFINITY;
        }
    }
    float base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = m_run[i];
#pragma unroll
      for (int n = 0; n < kWarpKeys / 8; ++n) m = fmaxf(m, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      base[i] = m == -INFINITY ? 0.f : m * a.scale_log2;  // a row that has seen nothing yet
      const float fade = exp2_approx(m_run[i] * a.scale_log2 - base[i]);
      m_run[i] = m;
      l_run[i] *= fade;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][2 * i] *= fade;
        o[n][2 * i + 1] *= fade;
      }
    }
#pragma unroll
    for (int n2 = 0; n2 < kWarpKeys / 16; ++n2) {
      float p[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[h][j] = exp2_approx(fmaf(s[2 * n2 + h][j], a.scale_log2, -base[j >> 1]));
          l_run[j >> 1] += p[h][j];
        }
      // Weights are rounded to the type of v: half a step of them each, averaged over the keys.
      const uint32_t pf[4] = {pack2<T>(p[0][0], p[0][1]), pack2<T>(p[0][2], p[0][3]), pack2<T>(p[1][0], p[1][1]),
                              pack2<T>(p[1][2], p[1][3])};
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b[4];
        const int row = n2 * 16 + vr;
        tree_ldm_trans(b, vs + row * (D * 2) + (((2 * n + vc) ^ (row & 7)) << 4));
        tree_mma<T>(o[2 * n], pf, b[0], b[1]);
        tree_mma<T>(o[2 * n + 1], pf, b[2], b[3]);
      }
    }

    const int64_t at = begin + it;  // this tile
    const bool segment_ends = now.tile + 1 == now.tiles;
    if (segment_ends || it + 1 == n_tiles) {
      const int64_t segment_begin = seq_begin + int64_t(now.part) * now.tiles;
      // Sums of the four lanes that share a row.
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      }
      // The warps that share rows meet pairwise.
#pragma unroll
      for (int half = kKeyWarps / 2; half > 0; half >>= 1) {
        float* slot = merge + (rw * (kKeyWarps / 2) + (kw % half)) * S::kMergeWords + lane;
        if (kw >= half && kw < 2 * half) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) slot[(4 * i + j) * 32] = o[i][j];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            slot[(D / 2 + i) * 32] = m_run[i];
            slot[(D / 2 + 2 + i) * 32] = l_run[i];
          }
        }
        __syncthreads();
        if (kw < half) {
          float mine[2], theirs[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float m2 = slot[(D / 2 + i) * 32], l2 = slot[(D / 2 + 2 + i) * 32], m = fmaxf(m_run[i], m2);
            const float b = m == -INFINITY ? 0.f : m;
            mine[i] = exp2_approx((m_run[i] - b) * a.scale_log2);
            theirs[i] = exp2_approx((m2 - b) * a.scale_log2);
            m_run[i] = m;
            l_run[i] = l_run[i] * mine[i] + l2 * theirs[i];
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              o[i][j] = o[i][j] * mine[j >> 1] + slot[(4 * i + j) * 32] * theirs[j >> 1];
        }
        __syncthreads();
      }
      const bool whole = piece_begin == segment_begin && segment_ends;
      const int head0 = (now.part / a.row_tiles) * a.group, row0 = (now.part % a.row_tiles) * (16 * RW);
      if (whole) {
        if (kw == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = row0 + rw * 16 + g + 8 * i;
            if (row >= rows_all) continue;
            const int token = row / a.group, head = head0 + row - token * a.group;
            const float inv = l_run[i] > 0.f || l_run[i] != l_run[i] ? 1.f / l_run[i] : 0.f;  // a row that sees nothing: zeros
            T* p = static_cast<T*>(a.out) + (int64_t(now.seq) * a.drafted + token) * a.out_stride + head * D;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<uint32_t*>(p + n * 8 + 2 * t) = pack2<T>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
          }
        }
      } else {
        constexpr size_t kSlot = size_t(16 * RW) * (D + 2);
        // A block has at most two pieces that are not whole: one that begins with its segment, one that does not.
        float* mine = a.partial + (2 * size_t(blockIdx.x) + (piece_begin == segment_begin ? 1 : 0)) * kSlot;
        if (kw == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = rw * 16 + g + 8 * i;
            if (t == 0) {
              mine[row] = m_run[i];
              mine[16 * RW + row] = l_run[i];
            }
            float* p = mine + 32 * RW + row * D + 2 * t;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(p + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
          }
        }
        __threadfence();
        __syncthreads();
        const int64_t segment_end = segment_begin + now.tiles;
        const int first = int(((segment_begin + 1) * blocks - 1) / total), last = int((segment_end * blocks - 1) / total);
        int32_t* counter = a.counters + int64_t(now.seq) * parts + now.part;
        if (tid == 0) {
          last_block = atomicAdd(counter, 1) == last - first;
          if (last_block) *counter = 0;  // for the next call
        }
        __syncthreads();
        if (last_block) {
          __threadfence();
          const float* head_piece = a.partial + (2 * size_t(first) + 1) * kSlot;
          for (int i = tid; i < 16 * RW * (D / 4); i += kTreeThreads) {
            const int r = i / (D / 4), c = 4 * (i % (D / 4)), row = row0 + r;
            if (row >= rows_all) break;
            float m = -INFINITY, l = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int b = first; b <= last; ++b) {
              const float* piece = b == first ? head_piece : a.partial + 2 * size_t(b) * kSlot;
              const float m2 = __ldcg(piece + r), l2 = __ldcg(piece + 16 * RW + r);
              const float4 x = __ldcg(reinterpret_cast<const float4*>(piece + 32 * RW + r * D + c));
              const float top = fmaxf(m, m2), zero = top == -INFINITY ? 0.f : top;
              const float f1 = exp2_approx((m - zero) * a.scale_log2), f2 = exp2_approx((m2 - zero) * a.scale_log2);
              m = top;
              l = l * f1 + l2 * f2;
              sum.x = sum.x * f1 + x.x * f2;
              sum.y = sum.y * f1 + x.y * f2;
              sum.z = sum.z * f1 + x.z * f2;
              sum.w = sum.w * f1 + x.w * f2;
            }
            const int token = row / a.group, head = head0 + row - token * a.group;
            const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
            T* p = static_cast<T*>(a.out) + (int64_t(now.seq) * a.drafted + token) * a.out_stride + head * D + c;
            *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
          }
        }
        __syncthreads();
      }
      piece_begin = at + 1;
    }
    if (it + 1 < n_tiles) {
      const int seq = now.seq, tiles = now.tiles;
      if (advance(now)) {
        if (now.seq != seq) seq_begin += int64_t(tiles) * parts;
        begin_segment();
      }
    }
  }
  tree_cp_wait<0>();
}

// Row warps: enough for the rows of a key head, up to eight.
int tree_row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

template <class T, int D, int RW>
cudaError_t launch_tree(const TreeArgs& a, cudaStream_t s) {
  constexpr int smem = TreeShape<D, RW>::kSmem;
  static PerDeviceOnce once;
  const cudaError_t e = per_device_once(once, [] { return opt_in_smem(tree_kernel<T, D, RW>, smem); });
  if (e != cudaSuccess) return e;
  return launch_pdl(tree_kernel<T, D, RW>, dim3(unsigned(sm_count())), dim3(kTreeThreads), size_t(smem), s, a);
}
template <class T, int D>
cudaError_t launch_tree_rows(const TreeArgs& a, int rw, cudaStream_t s) {
  return rw == 1 ? launch_tree<T, D, 1>(a, s) : rw == 2 ? launch_tree<T, D, 2>(a, s) : rw == 4 ? launch_tree<T, D, 4>(a, s)
                                                                                             : launch_tree<T, D, 8>(a, s);
}
size_t tree_counter_bytes(int64_t n_seqs, int drafted, int heads, int kv_heads) {
  const int rows = drafted * (heads / kv_heads), tile = 16 * tree_row_warps(rows);
  return (size_t(n_seqs) * kv_heads * ((rows + tile - 1) / tile) * 4 + 255) & ~size_t(255);
}
bool tree_shape_ok(int n_seqs, int drafted, int heads, int kv_heads, int dim) {
  return n_seqs >= 0 && drafted >= 1 && drafted <= kTreeMaxDrafted && kv_heads >= 1 && heads >= kv_heads && heads <= 1024 &&
         heads % kv_heads == 0 && (dim == 64 || dim == 128);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

size_t fb_attn_tree_workspace_bytes(int32_t n_seqs, int32_t drafted, int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (!tree_shape_ok(n_seqs, drafted, heads, kv_heads, head_dim)) return 0;
  const int tile = 16 * tree_row_warps(drafted * (heads / kv_heads));
  return tree_counter_bytes(n_seqs, drafted, heads, kv_heads) + size_t(2 * kTreeMaxSms) * tile * (head_dim + 2) * 4;
}

int32_t fb_attn_tree_decode(const void* q, int64_t q_stride, int32_t heads, int32_t n_seqs, int32_t drafted,
                            const fb_kv_cache* cache, const int32_t* block_table, int64_t table_stride, const int32_t* contexts,
                            const uint64_t* mask, float scale, void* out, int64_t out_stride, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (!cache) return invalid("attn_tree_decode: null argument");
  const int dim = cache->head_dim, kv = cache->kv_heads;
  if (cache->dtype != FB_DT_BF16 && cache->dtype != FB_DT_F16) return invalid("attn_tree_decode: bf16 or fp16");
  if (drafted < 1 || drafted > kTreeMaxDrafted) return invalid("attn_tree_decode: 1..64 drafted tokens per sequence");
  if (!tree_shape_ok(n_seqs, drafted, heads, kv, dim))
    return invalid("attn_tree_decode: unsupported shape (head_dim 64 or 128, heads a multiple of kv_heads up to 1024)");
  if (!n_seqs) return 0;
  if (!q || !out || !block_table || !contexts || !cache->k || !cache->v) return invalid("attn_tree_decode: null argument");
  if (cache->page_size < 1 || cache->n_pages < 1) return invalid("attn_tree_decode: a cache without pages");
  if (table_stride < 1) return invalid("attn_tree_decode: a table without columns");
  if (table_stride > INT32_MAX / 2 / cache->page_size) return invalid("attn_tree_decode: more than 2^30 keys per sequence");
  if (q_stride < int64_t(heads) * dim || out_stride < int64_t(heads) * dim)
    return invalid("attn_tree_decode: a stride is smaller than a token's heads");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache->k) |
       reinterpret_cast<uintptr_t>(cache->v)) & 15 || q_stride % 8 || out_stride % 8)
    return invalid("attn_tree_decode: tensors start on 16 bytes and tokens lie a multiple of 8 elements apart");
  if ((reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(contexts)) & 3 || reinterpret_cast<uintptr_t>(mask) & 7)
    return invalid("attn_tree_decode: table, contexts or mask are not aligned to their elements");
  if (!(scale > 0.f && scale <= 1.0e30f)) return invalid("attn_tree_decode: scale is not positive and finite");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < fb_attn_tree_workspace_bytes(n_seqs, drafted, heads, kv, dim))
    return invalid("attn_tree_decode: workspace missing, misaligned (256 B) or smaller than fb_attn_tree_workspace_bytes");
  if (sm_count() > kTreeMaxSms) return invalid("attn_tree_decode: more than 256 multiprocessors");
  TreeArgs a;
  a.q = q;
  a.out = out;
  a.k = cache->k;
  a.v = cache->v;
  a.table = block_table;
  a.contexts = contexts;
  a.mask = mask;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_pages = cache->n_pages;
  a.table_stride = table_stride;
  a.counters = static_cast<int32_t*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + tree_counter_bytes(n_seqs, drafted, heads, kv));
  a.scale_log2 = scale * 1.4426950408889634f;  // scores are kept in powers of two
  a.n_seqs = n_seqs;
  a.drafted = drafted;
  a.kv_heads = kv;
  a.group = heads / kv;
  a.page_size = cache->page_size;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (cache->page_size == 1 << i) a.page_shift = i;
  const int rows = drafted * a.group, rw = tree_row_warps(rows);
  a.row_tiles = (rows + 16 * rw - 1) / (16 * rw);
  cudaStream_t s = as_stream(stream);
  const bool bf = cache->dtype == FB_DT_BF16;
  const cudaError_t e = dim == 64 ? (bf ? launch_tree_rows<__nv_bfloat16, 64>(a, rw, s) : launch_tree_rows<__half, 64>(a, rw, s))
                                  : (bf ? launch_tree_rows<__nv_bfloat16, 128>(a, rw, s) : launch_tree_rows<__half, 128>(a, rw, s));
  const int32_t st = check_launch("attn_tree_decode");
  return st ? st : int32_t(e);
}

}  // extern "C"
