// Attention of a few drafted tokens per sequence over a paged cache (one token per sequence: plain decoding), on tcgen05.
//
//   out[i] = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that token i sees: all ctx keys of the context, and of the
//   drafted tokens, whose keys follow the context's in the cache, those in its mask.
//
// Bound by the cache's bytes: each key and value is read once for all rows (tokens x query heads of a group) of a key head. The
// rows, up to 128, are the lanes of the products' results in tensor memory, whether they are 4 or 128: a block of 128 keys costs the
// tensor core 1024 cycles at head_dim 128 and a multiprocessor's share of the memory bandwidth 2800. (Products by mma.sync with
// fragments in registers, 16 to 128 rows, were bound by the latencies of eight warps: 446 us for 32 sequences of up to 16384 keys
// and four tokens, 87 for eight of 4096 and sixteen.)
//   S = Q K^T   both operands in shared memory, fp32 S in tensor memory
//   P = 2^(c S - c m) over S in the type of v, by a thread per row; only warps that hold rows read S
//   O += P V    fp32 in tensor memory; multiplied only when a maximum rises by more than 2^8 above the one in use
// A block of keys keeps its softmax warps and its products longer than its bytes take. So even and odd blocks are two streams with
// warps, S, O, maxima and sums of their own, which meet where a segment ends: each O is read there by both, half of the columns each.
// And a warp reaches only its 32 lanes of tensor memory: up to 32 rows lie there four times (up to 64 twice), and each copy takes a part of a
// block's keys, with zeros for weights of the others, and a maximum, a sum and an O of its own until the segment ends.
// 32 sequences of up to 16384 keys, four tokens, 32 heads of 128: 268 us = 6.25 TB/s (302 without the copies of rows; head_dim 64 207
// and 244); eight of 4096 keys, sixteen tokens, 48 heads: 41 us; one token and 1003 keys: 12.
// Blocks of context keys come by TMA, a box per run of slots that a page holds (up to 128, the power of two in the page size). The
// block where the context ends, and all blocks where that power is below kTreeMinBox, come by cp.async, 16 bytes a thread: any slots, and
// what is not to be read is written as zeros. (cp.async alone moves 4.4 TB/s; TMA gathers of four cache rows took 41 ns each per
// multiprocessor, 512 bytes.) The blocks of keys of all (sequence, key head, row tile) segments are one sequence that is cut
// evenly over the multiprocessors, so that sequences of different lengths leave none of them idle, whatever lengths the
// device finds (the host does not know them). A segment that several blocks share is joined by the last of them to arrive, in
// block order: results do not depend on timing.
#include "attn_common.cuh"

namespace fb {
namespace {

constexpr int kTreeThreads = 512;        // two streams of four softmax warps, four that copy, one each that issues scores and outputs, two idle
constexpr int kTreeWarps = kTreeThreads / 32;
constexpr int kTreeRows = 128;           // rows of a tile
constexpr int kTreeKeys = 128;           // keys of a block
constexpr int kTreeMaxDrafted = 64;
constexpr int kTreeMaxSms = 256;         // partial results are sized for this many blocks
constexpr int kTreeMinBox = 8;           // slots of the smallest box
constexpr int kTreeBarBytes = 3 * 1024;  // for barriers and tables
constexpr float kTreeSlack = 8.f;        // how far (in powers of two) scores may rise above the maximum in use

struct TreeArgs {
  void* out;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* contexts;
  const uint64_t* mask;
  int64_t out_stride;  // elements between tokens
  int64_t table_stride;
  int64_t table_columns;
  uint32_t* status;
  int32_t* counters;   // [segments]
  float* partial;      // [2 * blocks]: outputs [D / 4][128][4], maxima [128], sums [128]
  float scale_log2;
  int n_pages, n_seqs, drafted, kv_heads, group, page_size, page_shift;
  int box;                     // slots of a copied box, 0: no boxes
  int row_tiles, tile_tokens;  // row tiles per key head, drafted tokens per row tile
};
struct TreeMaps {
  CUtensorMap q, k, v;
};

// C copies of a tile's rows in 128 / C lanes each.
template <int D, int C>
struct TreeShape {
  static constexpr int kTileBytes = kTreeKeys * D * 2;
  static constexpr int kHalf = kTreeKeys * 128;  // a tile is D / 64 parts of 128 rows x 128 bytes
  static constexpr int kStages = D == 64 ? 10 : C == 1 ? 5 : 4;
  static constexpr int kMeet = C == 1 ? 0 : 2 * kTreeRows * 32 * 4;  // where copies of rows meet: 32 columns for each stream's warps
  static constexpr int kSmem = (2 + kStages) * kTileBytes + kMeet + kTreeBarBytes;
  static constexpr int kSlot = (D + 2) * kTreeRows;  // floats of a partial result
};

struct TreeBars {
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2], full[10], empty[10], drained;
  float tops[2][kTreeRows], sum_of[2][kTreeRows];  // of the two streams, where they meet
  union {
    int slots[kTreeKeys];  // cache slots of a key block, -1: zeros
    struct {               // before the first of them
      int64_t sums[kTreeWarps];
      int64_t found[2];
    };
  };
  uint32_t tmem;
  int aborted;
  int q_issued;
  int in_flight;  // copies up to the last one made by TMA
  int last_block;
};
static_assert(sizeof(TreeBars) <= kTreeBarBytes, "room behind the ring");
static_assert(TreeShape<128, 1>::kSmem <= 227 * 1024, "all of a multiprocessor's shared memory");

// Walks through the key blocks of the segments in their order.
struct TreeCursor {
  int seq, part, tile;     // part: key head * row tiles + row tile
  int tiles, ctx, length;  // of the sequence
};

template <class T, int D, int C>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_kernel(const TreeArgs a, const __grid_constant__ TreeMaps maps) {
  using S = TreeShape<D, C>;
  constexpr int kStages = S::kStages, kParts = D / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_tiles = smem;
  uint8_t* ring = smem + 2 * S::kTileBytes;
  float4* meet = reinterpret_cast<float4*>(ring + kStages * S::kTileBytes);  // [stream][8 pieces of 4 columns][128 rows]
  TreeBars* bars = reinterpret_cast<TreeBars*>(ring + kStages * S::kTileBytes + S::kMeet);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int parts = a.kv_heads * a.row_tiles;
  const int64_t room = a.table_columns * a.page_size;  // keys that the table can hold
  pdl_wait_prior();
  if (smem_u32(smem) & 1023u) {  // (tiles and their swizzle start on 1024 bytes)
    if (tid == 0) atomicMax(a.status, uint32_t(FB_STATUS_BAD_WORK));
    return;
  }

  auto length_of = [&](int seq, int* ctx) {
    int c = a.contexts[seq];
    c = c < 0 ? 0 : c;
    if (c > room) c = int(room);
    *ctx = c;
    const int64_t n = int64_t(c) + a.drafted;
    return int(n < room ? n : room);
  };
  auto blocks_of = [](int length) { return length > kTreeKeys ? (length + kTreeKeys - 1) / kTreeKeys : 1; };
  auto tiles_of = [&](int seq) {
    int c;
    return blocks_of(length_of(seq, &c));
  };

  // All key blocks, and the sequence that this block's first one lies in.
  int64_t total = 0, begin = 0, end = 0, seq_begin = 0;
  int blocks = 0, first_seq = 0;
  if (a.n_seqs <= 32) {  // every warp for itself
    const int64_t n = lane < a.n_seqs ? int64_t(tiles_of(lane)) * parts : 0;
    int64_t upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    blocks = int(total < int64_t(gridDim.x) ? total : int64_t(gridDim.x));
    if (int(blockIdx.x) >= blocks) return;
    begin = int64_t(blockIdx.x) * total / blocks;
    const uint32_t who = __ballot_sync(0xffffffffu, n && upto > begin && upto - n <= begin);
    first_seq = __ffs(who) - 1;
    seq_begin = __shfl_sync(0xffffffffu, upto - n, first_seq);
  } else {
    int64_t mine = 0;
    for (int s = tid; s < a.n_seqs; s += kTreeThreads) mine += tiles_of(s);
#pragma unroll
    for (int m = 16; m; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
    if (lane == 0) bars->sums[warp] = mine;
    __syncthreads();
    for (int w = 0; w < kTreeWarps; ++w) total += bars->sums[w];
    __syncthreads();
    total *= parts;
    blocks = int(total < int64_t(gridDim.x) ? total : int64_t(gridDim.x));
    if (int(blockIdx.x) >= blocks) return;
    begin = int64_t(blockIdx.x) * total / blocks;
    int64_t before = 0;
    for (int base = 0; base < a.n_seqs && before <= begin; base += kTreeThreads) {
      const int s = base + tid;
      const int64_t n = s < a.n_seqs ? int64_t(tiles_of(s)) * parts : 0;
      int64_t upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t other = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += other;
      }
      if (lane == 31) bars->sums[warp] = upto;
      __syncthreads();
      int64_t all = 0;
      for (int w = 0; w < kTreeWarps; ++w) {
        if (w < warp) upto += bars->sums[w];
        all += bars->sums[w];
      }
      if (n && before + upto > begin && before + upto - n <= begin) {
        bars->found[0] = s;
        bars->found[1] = before + upto - n;
      }
      before += all;
      __syncthreads();
    }
    first_seq = int(bars->found[0]);
    seq_begin = bars->found[1];
  }
  end = int64_t(blockIdx.x + 1) * total / blocks;
  const int n_tiles = int(end - begin);

  TreeCursor now;
  now.seq = first_seq;
  now.length = length_of(now.seq, &now.ctx);
  now.tiles = blocks_of(now.length);
  now.part = int((begin - seq_begin) / now.tiles);
  now.tile = int((begin - seq_begin) % now.tiles);
  auto advance = [&](TreeCursor& c) {  // true: a new segment
    if (++c.tile < c.tiles) return false;
    c.tile = 0;
    if (++c.part == parts) {
      c.part = 0;
      if (++c.seq < a.n_seqs) {
        c.length = length_of(c.seq, &c.ctx);
        c.tiles = blocks_of(c.length);
      }
    }
    return true;
  };

  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], kTreeRows);
      mbar_init(&bars->o_done[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars->full[i], kTreeKeys);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->drained, 2);
    bars->aborted = 0;
    bars->q_issued = 0;
    bars->in_flight = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (not before the allocation: a block of the next kernel that took tensor memory and then waited for this one would hold it up)
  pdl_launch_dependents();
  // All 512 columns: their address is 0, and every address in tensor memory a constant.
  if (bars->tmem != 0 && tid == 0) atomicMax(a.status, uint32_t(FB_STATUS_BAD_WORK));
  constexpr uint32_t kS = 0, kO = 256;  // stream t: S in columns 128 t, O in 256 + 128 t

  // 256 threads x 168 and 256 x 88 registers are the 512 x 128 of the launch.
  if (warp >= 8 && warp < 12) {
    regs_down<88>();
    // ------------------------------------------------------------------ copies
    const int me = tid - 256;  // looks up key `me` of a block
    uint64_t seen = 0;         // drafted tokens that some token of the sequence sees
    auto look = [&](int seq) {
      seen = ~0ull;
      if (!a.mask) return;
      uint64_t m = 0;
      for (int i = lane; i < a.drafted; i += 32) m |= a.mask[int64_t(seq) * a.drafted + i];
      const uint32_t lo = __reduce_or_sync(0xffffffffu, uint32_t(m)), hi = __reduce_or_sync(0xffffffffu, uint32_t(m >> 32));
      seen = (uint64_t(hi) << 32) | lo;
    };
    int page = -1;  // of the block to be copied next
    auto ask = [&] {
      const int key = now.tile * kTreeKeys + me, d = key - now.ctx;
      const bool read = key < now.length && (d < 0 || ((seen >> (d & 63)) & 1));
      const int index = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
      page = read ? a.table[now.seq * a.table_stride + index] : -1;
    };
    constexpr int kChunks = D / 8, kPerPass = kTreeKeys / kChunks, kPasses = kTreeKeys / kPerPass;
    const int chunk = me % kChunks, row = me / kChunks;
    const uint32_t put = uint32_t((chunk / 8) * S::kHalf + ((((chunk & 7) ^ (row & 7)) << 4) + row * 128));
    const size_t slot_values = size_t(a.kv_heads) * D;
    static_assert(kPerPass % 8 == 0, "a thread's rows have one place in their 128-byte swizzle");
    look(now.seq);
    ask();
    bool ok = true, fresh = true;
    int segment = 0;
    // (after a wait that ran out the loop goes on without copies: all four warps meet at the same barriers)
    for (int it = 0; it < n_tiles; ++it) {
      const int head = now.part / a.row_tiles;
      if (fresh) {
        const int b = segment & 1;
        if (segment >= 2) ok = ok && bounded_wait_warp(&bars->aborted, a.status, &bars->q_empty[b], uint32_t(segment / 2 - 1) & 1);
        if (ok && me == 0) {
          const int token = now.seq * a.drafted + (now.part % a.row_tiles) * a.tile_tokens;
          mbar_expect_tx(&bars->q_full[b], uint32_t(C * a.tile_tokens * a.group) * D * 2);
          for (int c = 0; c < C; ++c)
            for (int p = 0; p < kParts; ++p)
              tma_load_3d(smem_u32(q_tiles + b * S::kTileBytes) + p * S::kHalf + c * (kTreeRows / C) * 128, &maps.q, p * 64, head * a.group, token,
                          &bars->q_full[b]);
          bars->q_issued = segment + 1;
        }
        ++segment;
      }
      // A page outside of the cache reads as zeros, as does a drafted token that nobody sees.
      const int key = now.tile * kTreeKeys + me, index = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
      const int mine = page >= 0 && page < a.n_pages ? page * a.page_size + (key - index * a.page_size) : -1;
      const bool boxes = a.box && (now.tile + 1) * kTreeKeys <= now.ctx;  // (the same for all)
      if (!boxes) bars->slots[me] = mine;
      if (it + 1 < n_tiles) {
        const int seq = now.seq;
        fresh = advance(now);
        if (now.seq != seq) look(now.seq);
        ask();
      }
      if (!boxes) warps_sync(2, kTreeKeys);
      const int* slots = &bars->slots[row];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int i = 2 * it + kv, at = i % kStages;
        if (i >= kStages) ok = ok && bounded_wait_warp(&bars->aborted, a.status, &bars->empty[at], uint32_t(i / kStages - 1) & 1);
        // Each thread makes one of the slot's 128 arrivals.
        if (boxes) {
          if (ok && me == 0) {
            mbar_expect_tx(&bars->full[at], S::kTileBytes);
            bars->in_flight = i + 1;
          } else {
            mbar_arrive(&bars->full[at]);
          }
          if (ok && me % a.box == 0) {
            const uint32_t dst = smem_u32(ring + at * S::kTileBytes) + me * 128;
#pragma unroll
            for (int p = 0; p < kParts; ++p)
              tma_load_2d(dst + p * S::kHalf, kv ? &maps.v : &maps.k, head * D + p * 64, mine >= 0 ? mine : a.n_pages * a.page_size, &bars->full[at]);
          }
          __syncwarp();
        } else {
          if (ok) {
            const T* from = static_cast<const T*>(kv ? a.v : a.k) + head * D + chunk * 8;
            const uint32_t dst = smem_u32(ring + at * S::kTileBytes) + put;
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
              const int slot = slots[p * kPerPass];
              const T* src = from + size_t(slot < 0 ? 0 : slot) * slot_values;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + p * (kPerPass * 128)), "l"(src), "r"(slot < 0 ? 0 : 16)
                           : "memory");
            }
          }
          // (made when this thread's copies have landed)
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars->full[at])) : "memory");
        }
      }
      if (!boxes) warps_sync(2, kTreeKeys);  // the slots have been read
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 12) {
    regs_down<88>();
    // ------------------------------------------------------------------ products: a thread for the scores, one for the outputs
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t kIdesc = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kTreeRows >> 4) << 24);
    constexpr uint32_t kIdescQk = kIdesc | (uint32_t(kTreeKeys >> 3) << 17);
    constexpr uint32_t kIdescPv = kIdesc | (uint32_t(D >> 3) << 17) | (1u << 16);  // V runs along N
    if (warp < 14 && elect_one()) {
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && bounded_spin(&bars->aborted, a.status, bar, parity); };
      int segment = 0, piece = 0;  // piece: first block of the segment in this block's share
      for (int it = 0; it < n_tiles && ok; ++it) {
        const bool first = it == piece, last = now.tile + 1 == now.tiles;
        const uint32_t t = uint32_t(it & 1);
        if (warp == 12) {
          const int slot = (2 * it) % kStages, b = segment & 1;
          if (first) wait(&bars->q_full[b], uint32_t(segment / 2) & 1);
          wait(&bars->full[slot], uint32_t(2 * it / kStages) & 1);
          if (it >= 2) wait(&bars->o_done[t], uint32_t((it >> 1) - 1) & 1);  // the stream's last weights, which lie over S, are used
          if (!ok) break;
          fence_proxy_async();  // (cp.async writes by the generic proxy, the product reads through the other)
          tc_fence_after();
          const uint32_t qd = umma_desc_lo(smem_u32(q_tiles + b * S::kTileBytes), 1), kd = umma_desc_lo(smem_u32(ring + slot * S::kTileBytes), 1);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k / 4) * (S::kHalf >> 4) + (k % 4) * 2;
            umma_ss<kIdescQk>(kS + 128 * t, qd + at, kd + at, k > 0);
          }
          umma_commit(&bars->s_full[t]);
          umma_commit(&bars->empty[slot]);
          if (last) umma_commit(&bars->q_empty[b]);
        } else {
          const int slot = (2 * it + 1) % kStages;
          wait(&bars->full[slot], uint32_t((2 * it + 1) / kStages) & 1);
          wait(&bars->p_full[t], uint32_t(it >> 1) & 1);
          if (!ok) break;
          fence_proxy_async();
          tc_fence_after();
          const uint32_t vd = umma_desc_lo(smem_u32(ring + slot * S::kTileBytes), S::kHalf >> 4);
          const uint32_t d = kO + 128 * t, p = kS + 128 * t;
          umma_ts<kIdescPv>(d, p, vd, it - piece >= 2);
#pragma unroll
          for (int k = 1; k < kTreeKeys / 16; ++k) umma_ts<kIdescPv>(d, p + 8 * k, vd + k * (2048 >> 4), true);
          umma_commit(&bars->o_done[t]);
          umma_commit(&bars->empty[slot]);
        }
        if (last) ++segment;
        if (it + 1 < n_tiles && advance(now)) piece = it + 1;
      }
      // Nothing issued here is still running when the tensor memory is given back.
      umma_commit(&bars->drained);
    }
    __syncwarp();
    for (uint32_t n = 0; n < (1u << 16) && !__all_sync(0xffffffffu, mbar_try_wait_hint(&bars->drained, 0)); ++n) {}
  } else {
    regs_up<168>();
    // ------------------------------------------------------------------ softmax: thread = row, warps 4 t .. 4 t + 3 take stream t
    const int t = warp >> 2, row = tid & (kTreeRows - 1), lane_row = 32 * (warp & 3);
    const uint32_t lanes = uint32_t(lane_row) << 16;
    const uint32_t s_at = lanes + kS + 128 * t, o_at = lanes + kO + 128 * t;
    const uint64_t scale = pair_of(a.scale_log2, a.scale_log2);
    // Copy c of the rows has its keys: the c-th part of a block's, in steps of 32.
    constexpr int span = kTreeRows / C, kSteps = 4 / C;
    const int copy = row / span, place = row % span, step0 = copy * kSteps;
    bool ok = true, fresh = true;
    float top = -INFINITY, sum = 0.f;
    int rows = 0, head0 = 0;
    int64_t token0 = 0;
    uint64_t sees = 0;
    int piece = 0;  // first block of the segment in this block's share
    // (after a wait that ran out the loop goes on without work: all eight warps meet at the same barriers)
    for (int it = 0; it < n_tiles; ++it) {
      if (fresh) {
        fresh = false;
        piece = it;
        top = -INFINITY;
        sum = 0.f;
        const int first = (now.part % a.row_tiles) * a.tile_tokens;
        const int tokens = a.drafted - first < a.tile_tokens ? a.drafted - first : a.tile_tokens;
        rows = tokens * a.group;
        head0 = (now.part / a.row_tiles) * a.group;
        token0 = int64_t(now.seq) * a.drafted + first;
        sees = 0;
        const int token = place / a.group;
        if (place < rows) sees = a.mask ? a.mask[token0 + token] : first + token == 63 ? ~0ull : (2ull << (first + token)) - 1;
        const int there = now.length - now.ctx;  // drafted tokens that the table has room for
        if (there < 64) sees &= (1ull << there) - 1;
      }
      const bool segment_ends = now.tile + 1 == now.tiles, piece_ends = segment_ends || it + 1 == n_tiles;
      if ((it & 1) == t) {
        ok = ok && bounded_wait_warp(&bars->aborted, a.status, &bars->s_full[t], uint32_t(it >> 1) & 1);
        if (ok && lane_row % span < rows) {
          tc_fence_after();
          // (The scores are read twice, once for the maximum and once for the weights: 130 cycles of 3300, for 64 registers.)
          const int off = now.ctx - now.tile * kTreeKeys;  // first column behind the context
          auto unseen = [&](int i, float (&s)[32]) {
            if (off >= kTreeKeys) return;
            const int sh = off - 32 * i;  // bit of this word that drafted token 0 has
            uint32_t bits;
            if (sh >= 32) bits = 0xffffffffu;
            else if (sh >= 0) bits = uint32_t(sees << sh) | ((1u << sh) - 1u);
            else bits = -sh < 64 ? uint32_t(sees >> -sh) : 0u;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!((bits >> c) & 1)) s[c] = -INFINITY;
          };
          // Loops of two steps of 32 columns, the next on their way: short enough to stay in the instruction cache, where all four steps
          // in a row ran at four cycles per instruction (drafts of 16: 49 us, now 41). What one turn hands to the next has landed.
          float s0[32], s1[32], latest = -INFINITY;
          tmem_ld32(s_at + 32 * step0, s0);
          tmem_ld_wait();
          tmem_landed(s0);
#pragma unroll 1
          for (int i = step0; i < step0 + kSteps; i += 2) {
            if (kSteps > 1) tmem_ld32(s_at + 32 * (i + 1), s1);
            unseen(i, s0);
            latest = scores_max(s0, latest);
            if (kSteps > 1) {
              tmem_ld_wait();
              tmem_landed(s1);
              tmem_ld32(s_at + 32 * (kSteps > 2 ? (i + 2) & 3 : step0), s0);  // (at the end the first columns again: the weights begin with them)
              unseen(i + 1, s1);
              latest = scores_max(s1, latest);
              tmem_ld_wait();
              tmem_landed(s0);
            }
          }
          // (no for a row that has seen nothing yet; rows behind the last one are nobody's and decide nothing)
          const bool rises = place < rows && (latest - top) * a.scale_log2 > kTreeSlack;
          if (__any_sync(0xffffffffu, rises)) {
            const float up = fmaxf(latest, top);
            const float fade = up == -INFINITY ? 1.f : exp2_approx((top - up) * a.scale_log2);
            top = up;
            sum *= fade;
            if (it - piece >= 2) {  // (the stream's last outputs are done: these scores were issued after that)
#pragma unroll 1
              for (int i = 0; i < D / 32; ++i) {
                float o[32];
                tmem_ld32(o_at + 32 * i, o);
                tmem_ld_wait();
                tmem_landed(o);
                uint32_t r[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(o[c] * fade);
                tmem_st16(o_at + 32 * i, r);
                tmem_st16(o_at + 32 * i + 16, r + 16);
              }
            }
          }
          const float base = (top == -INFINITY ? 0.f : top * a.scale_log2) - kLift<T>;
          const uint64_t minus = pair_of(-base, -base);
          uint64_t part[2] = {0, 0};
#pragma unroll 1
          for (int i = step0; i < step0 + kSteps; i += 2) {
            uint32_t p[16];
            if (kSteps > 1) tmem_ld32(s_at + 32 * (i + 1), s1);
            if (kSteps > 1) unseen(i, s0);
            scores_exp<T, false>(s0, scale, minus, p, part);
            if (kSteps > 1) {
              tmem_ld_wait();
              tmem_landed(s1);
              tmem_st16(s_at + 16 * i, p);  // (over scores that have been read)
              if (kSteps > 2) tmem_ld32(s_at + 64, s0);  // (of no use in the second turn, whose weights begin at column 32)
              unseen(i + 1, s1);
              scores_exp<T, false>(s1, scale, minus, p, part);
              tmem_st16(s_at + 16 * (i + 1), p);
              if (kSteps > 2) {
                tmem_ld_wait();
                tmem_landed(s0);
              }
            } else {
              tmem_st16(s_at + 16 * i, p);
            }
          }
          if (C > 1) {  // the other copies' keys
            const uint32_t none[16] = {};
#pragma unroll
            for (int i = 1; i < C; ++i)
#pragma unroll
              for (int e = 0; e < kSteps; ++e) tmem_st16(s_at + 16 * (((copy + i) % C) * kSteps + e), none);
          }
          sum += pairs_sum(part);
          tmem_st_wait();
          tc_fence_before();
        }
        mbar_arrive(&bars->p_full[t]);
      }

      if (piece_ends) {
        // The stream's last block of this segment, if it has one. Its scores were issued when the outputs of the one before were done, so
        // the barrier is not two phases behind, and not ahead: the next outputs need this warp's weights.
        const int last_own = (it & 1) == t ? it : it - 1;
        if (last_own >= piece) ok = ok && bounded_wait_warp(&bars->aborted, a.status, &bars->o_done[t], uint32_t(last_own >> 1) & 1);
        tc_fence_after();
        bars->tops[t][row] = top;
        bars->sum_of[t][row] = sum;
        warps_sync(1, 2 * kTreeRows);
        const int64_t segment_begin = seq_begin + int64_t(now.part) * now.tiles, piece_begin = begin + piece;
        const bool whole = piece_begin == segment_begin && segment_ends;
        // A block has at most two pieces that are not whole: one that begins with its segment, one that does not.
        float* mine = a.partial + (2 * size_t(blockIdx.x) + (piece_begin == segment_begin ? 1 : 0)) * S::kSlot;
        if (C == 1) {
          if (ok && lane_row < rows) {
            const float m0 = bars->tops[0][row], m1 = bars->tops[1][row], up = fmaxf(m0, m1), zero = up == -INFINITY ? 0.f : up;
            float f[2] = {exp2_approx((m0 - zero) * a.scale_log2), exp2_approx((m1 - zero) * a.scale_log2)};
            const float l = bars->sum_of[0][row] * f[0] + bars->sum_of[1][row] * f[1];
            if (whole) {
              const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees nothing: zeros
              f[0] *= inv;
              f[1] *= inv;
            } else if (t == 0) {
              mine[D * kTreeRows + row] = up;
              mine[(D + 1) * kTreeRows + row] = l;
            }
            T* to = static_cast<T*>(a.out) + (token0 + row / a.group) * a.out_stride + int64_t(head0 + row % a.group) * D;
#pragma unroll
            for (int i = t * (D / 64); i < (t + 1) * (D / 64); ++i) {
              float o[32], x[32];
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] = 0.f;
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                if (it == piece && w != (it & 1)) continue;  // one block: one stream
                tmem_ld32(lanes + kO + 128 * w + 32 * i, o);
                tmem_ld_wait();
                tmem_landed(o);
#pragma unroll
                for (int c = 0; c < 32; ++c) x[c] = fmaf(o[c], f[w], x[c]);
              }
              if (row < rows) {
                if (whole) {
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    uint4 v;
                    v.x = pack2<T>(x[8 * c], x[8 * c + 1]);
                    v.y = pack2<T>(x[8 * c + 2], x[8 * c + 3]);
                    v.z = pack2<T>(x[8 * c + 4], x[8 * c + 5]);
                    v.w = pack2<T>(x[8 * c + 6], x[8 * c + 7]);
                    *reinterpret_cast<uint4*>(to + 32 * i + 8 * c) = v;
                  }
                } else {
#pragma unroll
                  for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<float4*>(mine + ((8 * i + c) * kTreeRows + row) * 4) = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
                }
              }
              __syncwarp();  // (the next read of tensor memory takes the whole warp)
            }
            tc_fence_before();
          }
        } else {
          const bool works = ok && lane_row % span < rows;
          float f[2] = {0.f, 0.f};
          T* to = static_cast<T*>(a.out) + (token0 + place / a.group) * a.out_stride + int64_t(head0 + place % a.group) * D;
          if (works) {
            float up = -INFINITY, l = 0.f;
            for (int r = place; r < kTreeRows; r += span) up = fmaxf(up, fmaxf(bars->tops[0][r], bars->tops[1][r]));
            const float zero = up == -INFINITY ? 0.f : up;
            for (int r = place; r < kTreeRows; r += span)
              l += bars->sum_of[0][r] * exp2_approx((bars->tops[0][r] - zero) * a.scale_log2) +
                   bars->sum_of[1][r] * exp2_approx((bars->tops[1][r] - zero) * a.scale_log2);
            f[0] = exp2_approx((bars->tops[0][row] - zero) * a.scale_log2);
            f[1] = exp2_approx((bars->tops[1][row] - zero) * a.scale_log2);
            if (whole) {
              const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees nothing: zeros
              f[0] *= inv;
              f[1] *= inv;
            } else if (t == 0 && copy == 0) {
              mine[D * kTreeRows + place] = up;
              mine[(D + 1) * kTreeRows + place] = l;
            }
          }
          // Four columns of a row, where they go.
          auto put = [&](int column, const float4& x) {
            if (!works || place >= rows) return;
            if (whole) {
              *reinterpret_cast<uint2*>(to + column) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
            } else {
              *reinterpret_cast<float4*>(mine + (column / 4 * kTreeRows + place) * 4) = x;
            }
          };
#pragma unroll 1
          for (int i = t * (D / 64); i < (t + 1) * (D / 64); ++i) {
            float x[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = 0.f;
            if (works) {
              __syncwarp();
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                if (it == piece && w != (it & 1)) continue;  // one block: one stream
                float o[32];
                tmem_ld32(lanes + kO + 128 * w + 32 * i, o);
                tmem_ld_wait();
                tmem_landed(o);
#pragma unroll
                for (int c = 0; c < 32; ++c) x[c] = fmaf(o[c], f[w], x[c]);
              }
            }
            // Each copy adds a part of the columns, in the order of the copies.
            float4* at = meet + t * (8 * kTreeRows);
#pragma unroll
            for (int c = 0; c < 8; ++c) at[c * kTreeRows + row] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
            warps_sync(3 + t, kTreeRows);
            for (int c = copy * (8 / C); c < (copy + 1) * (8 / C); ++c) {
              float4 all = at[c * kTreeRows + place];
              for (int r = place + span; r < kTreeRows; r += span) {
                const float4 v = at[c * kTreeRows + r];
                all.x += v.x;
                all.y += v.y;
                all.z += v.z;
                all.w += v.w;
              }
              put(32 * i + 4 * c, all);
            }
            warps_sync(3 + t, kTreeRows);
          }
          if (works) tc_fence_before();
        }
        if (!whole) {
          __threadfence();
          warps_sync(1, 2 * kTreeRows);
          const int64_t segment_end = segment_begin + now.tiles;
          const int first = int(((segment_begin + 1) * blocks - 1) / total), last = int((segment_end * blocks - 1) / total);
          if (tid == 0) {
            int32_t* counter = a.counters + int64_t(now.seq) * parts + now.part;
            bars->last_block = atomicAdd(counter, 1) == last - first;
            if (bars->last_block) *counter = 0;  // for the next call
          }
          warps_sync(1, 2 * kTreeRows);
          if (bars->last_block) {
            __threadfence();
            // 256 / rows threads to a row, rows along the lanes, up to four 16-byte pieces of it at a time.
            const int per_row = 2 * kTreeRows / rows, r = tid % rows, sub = tid / rows;
            if (sub < per_row) {
              // Piece b of the segment is block b's: the first begins with the segment, the others do not.
              const float* head_piece = a.partial + (2 * size_t(first) + 1) * S::kSlot;
              const float* piece0 = a.partial + 2 * size_t(first) * S::kSlot;
              // The first pieces, which most segments have no more than, in one go: their weights first, then rounds of 16 loads. (A piece that is
              // not there is the first one again, with a weight of zero.)
              constexpr int kFirst = 4;
              const int pieces = last - first + 1;
              const float* from[kFirst];
              float f[kFirst], l = 0.f, up = -INFINITY;
#pragma unroll
              for (int b = 0; b < kFirst; ++b) {
                from[b] = b && b < pieces ? piece0 + size_t(2 * b) * S::kSlot : head_piece;
                f[b] = __ldcg(from[b] + D * kTreeRows + r);
              }
              float sums[kFirst];
#pragma unroll
              for (int b = 0; b < kFirst; ++b) sums[b] = __ldcg(from[b] + (D + 1) * kTreeRows + r);
#pragma unroll
              for (int b = 0; b < kFirst; ++b) up = fmaxf(up, f[b]);
#pragma unroll 4
              for (int b = kFirst; b < pieces; ++b) up = fmaxf(up, __ldcg(piece0 + size_t(2 * b) * S::kSlot + D * kTreeRows + r));
              if (up == -INFINITY) up = 0.f;  // a row that sees nothing
#pragma unroll
              for (int b = 0; b < kFirst; ++b) {
                f[b] = b < pieces ? exp2_approx((f[b] - up) * a.scale_log2) : 0.f;
                l = fmaf(sums[b], f[b], l);
              }
#pragma unroll 4
              for (int b = kFirst; b < pieces; ++b) {
                const float* at = piece0 + size_t(2 * b) * S::kSlot + D * kTreeRows + r;
                l = fmaf(__ldcg(at + kTreeRows), exp2_approx((__ldcg(at) - up) * a.scale_log2), l);
              }
              const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
              T* to = static_cast<T*>(a.out) + (token0 + r / a.group) * a.out_stride + int64_t(head0 + r % a.group) * D;
              auto add = [](float4& x, const float4& o, float w) {
                x.x = fmaf(o.x, w, x.x);
                x.y = fmaf(o.y, w, x.y);
                x.z = fmaf(o.z, w, x.z);
                x.w = fmaf(o.w, w, x.w);
              };
              for (int c0 = sub; c0 < D / 4; c0 += 4 * per_row) {
                float4 x[4], o[kFirst][4];
#pragma unroll
                for (int b = 0; b < kFirst; ++b)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int c = c0 + e * per_row;
                    o[b][e] = __ldcg(reinterpret_cast<const float4*>(from[b] + ((c < D / 4 ? c : c0) * kTreeRows + r) * 4));
                  }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int b = 0; b < kFirst; ++b)
#pragma unroll
                  for (int e = 0; e < 4; ++e) add(x[e], o[b][e], f[b]);
#pragma unroll 2
                for (int b = kFirst; b < pieces; ++b) {
                  const float* at = piece0 + size_t(2 * b) * S::kSlot;
                  const float w = exp2_approx((__ldcg(at + D * kTreeRows + r) - up) * a.scale_log2);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int c = c0 + e * per_row;
                    if (c < D / 4) add(x[e], __ldcg(reinterpret_cast<const float4*>(at + (c * kTreeRows + r) * 4)), w);
                  }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int c = c0 + e * per_row;
                  if (c < D / 4)
                    *reinterpret_cast<uint2*>(to + 4 * c) = make_uint2(pack2<T>(x[e].x * inv, x[e].y * inv), pack2<T>(x[e].z * inv, x[e].w * inv));
                }
              }
            }
          }
        }
        warps_sync(1, 2 * kTreeRows);  // both streams' outputs have been read
      }
      if (it + 1 < n_tiles) {
        const int seq = now.seq, tiles = now.tiles;
        fresh = advance(now);
        if (now.seq != seq) seq_begin += int64_t(tiles) * parts;
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (bars->aborted && tid == 0) {  // copies that nobody waited for
    const int issued = bars->in_flight, q_issued = bars->q_issued;
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
      for (uint32_t n = 0; n < (1u << 16) && !mbar_try_wait_hint(&bars->full[i % kStages], uint32_t(i / kStages) & 1); ++n) {}
    for (int i = q_issued > 2 ? q_issued - 2 : 0; i < q_issued; ++i)
      for (uint32_t n = 0; n < (1u << 16) && !mbar_try_wait_hint(&bars->q_full[i & 1], uint32_t(i / 2) & 1); ++n) {}
  }
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(bars->tmem), "r"(512) : "memory");
}

template <class T, int D, int C>
cudaError_t launch_tree_copies(const TreeArgs& a, const TreeMaps& maps, cudaStream_t s) {
  static PerDeviceOnce once;
  const cudaError_t e = per_device_once(once, [] { return opt_in_smem(tree_kernel<T, D, C>, TreeShape<D, C>::kSmem); });
  if (e != cudaSuccess) return e;
  return launch_pdl(tree_kernel<T, D, C>, dim3(unsigned(sm_count())), dim3(kTreeThreads), size_t(TreeShape<D, C>::kSmem), s, a, maps);
}
template <class T, int D>
cudaError_t launch_tree(const TreeArgs& a, const TreeMaps& maps, cudaStream_t s) {
  const int rows = a.tile_tokens * a.group;
  return rows <= 32 ? launch_tree_copies<T, D, 4>(a, maps, s) : rows <= 64 ? launch_tree_copies<T, D, 2>(a, maps, s) : launch_tree_copies<T, D, 1>(a, maps, s);
}

// Drafted tokens of a row tile: whole tokens, as many as 128 rows hold.
int tree_tile_tokens(int drafted, int group) {
  const int fit = kTreeRows / group;
  return drafted < fit ? drafted : fit;
}
int tree_row_tiles(int drafted, int group) {
  const int t = tree_tile_tokens(drafted, group);
  return (drafted + t - 1) / t;
}
// Partial results lie in front of the counters, at one size for all shapes: what one call leaves there is no counter of another.
constexpr size_t kTreePartialBytes = size_t(2 * kTreeMaxSms) * kTreeRows * (128 + 2) * 4;
size_t tree_counter_bytes(int64_t n_seqs, int drafted, int heads, int kv_heads) {
  return (size_t(n_seqs) * kv_heads * tree_row_tiles(drafted, heads / kv_heads) * 4 + 255) & ~size_t(255);
}
bool tree_shape_ok(int n_seqs, int drafted, int heads, int kv_heads, int dim) {
  return n_seqs >= 0 && drafted >= 1 && drafted <= kTreeMaxDrafted && kv_heads >= 1 && heads >= kv_heads && heads <= 1024 &&
         heads % kv_heads == 0 && heads / kv_heads <= kTreeRows && (dim == 64 || dim == 128);
}

// The cache's slots as rows of kv_heads * dim values, in boxes of `box` slots x 64 values; slots behind the last one read as zeros.
bool tree_map_cache(CUtensorMap* map, const void* base, bool bf16, int64_t slots, int row, int box_slots) {
  const cuuint64_t dims[2] = {cuuint64_t(row), cuuint64_t(slots)}, strides[1] = {cuuint64_t(row) * 2};
  const cuuint32_t box[2] = {64, cuuint32_t(box_slots)}, elem[2] = {1, 1};
  return encode_tiled_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                           const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [tokens][heads][dim] in boxes of a row tile: its tokens x the heads of a group x 64 values.
bool tree_map_q(CUtensorMap* map, const void* base, bool bf16, int dim, int heads, int64_t tokens, int64_t stride, int group, int tile) {
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(dim) * 2, cuuint64_t(stride) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(group), cuuint32_t(tile)}, elem[3] = {1, 1, 1};
  return encode_tiled_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                           const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

size_t fb_attn_tree_workspace_bytes(int32_t n_seqs, int32_t drafted, int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (!tree_shape_ok(n_seqs, drafted, heads, kv_heads, head_dim)) return 0;
  return 256 + kTreePartialBytes + tree_counter_bytes(n_seqs, drafted, heads, kv_heads);
}

int32_t fb_attn_tree_decode(const void* q, int64_t q_stride, int32_t heads, int32_t n_seqs, int32_t drafted,
                            const fb_kv_cache* cache, const int32_t* block_table, int64_t table_stride, const int32_t* contexts,
                            const uint64_t* mask, float scale, void* out, int64_t out_stride, void* workspace,
                            size_t workspace_bytes, void* stream) {
  return fb_attn_tree_decode_view(q, q_stride, heads, n_seqs, drafted, cache, block_table, table_stride, table_stride, contexts, mask, scale, out,
                                  out_stride, workspace, workspace_bytes, stream);
}

int32_t fb_attn_tree_decode_view(const void* q, int64_t q_stride, int32_t heads, int32_t n_seqs, int32_t drafted,
                                 const fb_kv_cache* cache, const int32_t* block_table, int64_t table_stride, int64_t table_columns,
                                 const int32_t* contexts, const uint64_t* mask, float scale, void* out, int64_t out_stride,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!cache) return invalid("attn_tree_decode: null argument");
  const int dim = cache->head_dim, kv = cache->kv_heads;
  if (cache->dtype != FB_DT_BF16 && cache->dtype != FB_DT_F16) return invalid("attn_tree_decode: bf16 or fp16");
  if (drafted < 1 || drafted > kTreeMaxDrafted) return invalid("attn_tree_decode: 1..64 drafted tokens per sequence");
  if (!tree_shape_ok(n_seqs, drafted, heads, kv, dim))
    return invalid("attn_tree_decode: unsupported shape (head_dim 64 or 128, heads a multiple of kv_heads, up to 1024 and 128 per key head)");
  if (!n_seqs) return 0;
  if (!q || !out || !block_table || !contexts || !cache->k || !cache->v) return invalid("attn_tree_decode: null argument");
  if (cache->page_size < 1 || cache->n_pages < 1) return invalid("attn_tree_decode: a cache without pages");
  if (table_columns < 1) return invalid("attn_tree_decode: a table without columns");
  if (table_columns > INT32_MAX / 2 / cache->page_size) return invalid("attn_tree_decode: more than 2^30 keys per sequence");
  if (table_stride < table_columns) return invalid("attn_tree_decode: rows of the table overlap");
  if (table_stride > INT32_MAX) return invalid("attn_tree_decode: rows of the table lie too far apart");
  if (cache->n_pages > INT32_MAX / cache->page_size) return invalid("attn_tree_decode: a cache of more than 2^31 slots");
  if (int64_t(n_seqs) * drafted > INT32_MAX || q_stride >= int64_t(1) << 38)
    return invalid("attn_tree_decode: q is too large");
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
  if (!encode_tiled_fn()) {
    set_error("attn_tree_decode: cuTensorMapEncodeTiled is not available");
    return int32_t(cudaErrorNotSupported);
  }
  TreeArgs a;
  a.out = out;
  a.k = cache->k;
  a.v = cache->v;
  a.table = block_table;
  a.contexts = contexts;
  a.mask = mask;
  a.out_stride = out_stride;
  a.table_stride = table_stride;
  a.table_columns = table_columns;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  a.status = reinterpret_cast<uint32_t*>(base);
  a.partial = reinterpret_cast<float*>(base + 256);
  a.counters = reinterpret_cast<int32_t*>(base + 256 + kTreePartialBytes);
  a.scale_log2 = scale * 1.4426950408889634f;  // scores are kept in powers of two
  a.n_pages = int(cache->n_pages);
  a.n_seqs = n_seqs;
  a.drafted = drafted;
  a.kv_heads = kv;
  a.group = heads / kv;
  a.page_size = cache->page_size;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (cache->page_size == 1 << i) a.page_shift = i;
  a.tile_tokens = tree_tile_tokens(drafted, a.group);
  a.row_tiles = tree_row_tiles(drafted, a.group);
  const bool bf = cache->dtype == FB_DT_BF16;
  a.box = cache->page_size & -cache->page_size;  // slots that start on a multiple of it lie in one page
  if (a.box > kTreeKeys) a.box = kTreeKeys;
  if (a.box < kTreeMinBox) a.box = 0;
  const int64_t slots = cache->n_pages * cache->page_size;
  TreeMaps maps;
  if (!tree_map_q(&maps.q, q, bf, dim, heads, int64_t(n_seqs) * drafted, q_stride, a.group, a.tile_tokens) ||
      !tree_map_cache(&maps.k, cache->k, bf, slots, kv * dim, a.box ? a.box : kTreeMinBox) ||
      !tree_map_cache(&maps.v, cache->v, bf, slots, kv * dim, a.box ? a.box : kTreeMinBox))
    return invalid("attn_tree_decode: cuTensorMapEncodeTiled failed");
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = dim == 64 ? (bf ? launch_tree<__nv_bfloat16, 64>(a, maps, s) : launch_tree<__half, 64>(a, maps, s))
                                  : (bf ? launch_tree<__nv_bfloat16, 128>(a, maps, s) : launch_tree<__half, 128>(a, maps, s));
  const int32_t st = check_launch("attn_tree_decode");
  return st ? st : int32_t(e);
}

}  // extern "C"
