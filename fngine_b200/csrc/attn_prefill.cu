// Causal attention over packed prompts with grouped heads, on tcgen05.
//
//   out_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j     within a sequence; query head h reads key head h / (heads / kv_heads)
//
// One pass over the keys per query tile with a running maximum and sum. A block takes 256 queries of one head as two tiles of
// 128 (TMEM lanes) and goes through the keys 128 at a time:
//   S = Q K^T   tcgen05 kind::f16, both operands in shared memory, fp32 S in tensor memory (128 columns per tile)
//   P = 2^(c S - c m) in the type of v, to tensor memory by the tile's four softmax warps, a thread per row: no shuffles
//   O += P V    P from tensor memory, V as it lies in memory (keys x head_dim: the operand's N-major form), fp32 O in tensor memory
// The two tiles are half a step apart and take turns with S, which a softmax thread has in registers 70 cycles after it is complete:
// from then on the other tile's scores are made there, so neither softmax waits for the tensor core.
// m is the maximum that the exponents refer to, not the latest one: it moves up (and O is multiplied) only when a row's scores
// rise above it by more than 2^8, which leaves every weight at most 256 (times 2^7 in fp16) and the sum in fp32 range. Normally that is
// the first block alone, so O stays in tensor memory untouched.
// Blocks are handed out longest first (causal: the last queries of a prompt have the most keys).
// Bound by the exponentials (16 per clock and multiprocessor) and the tensor core, which are near level, and then by power: 8192
// tokens of 48 heads of 128 in 616 us = 1.34 PFLOP/s in a burst, 724 under sustained load (a large library product: 1.62 and 1.35). Four prompts of 4000
// tokens in all take 86: a block of 256 queries has some 7000 cycles of set-up, first scores and epilogue beside 2900 per key block.
#include "attn_common.cuh"

namespace fb {
namespace {

constexpr int kPfRows = 128;             // queries per tile, keys per block
constexpr int kPfQueries = 2 * kPfRows;  // queries per CTA
constexpr int kPfThreads = 384;          // two softmax warpgroups, one with the copying and the issuing warp
constexpr float kPfSlack = 8.f;          // how far (in powers of two) scores may rise above the maximum in use

template <int D>
struct PfShape {
  static constexpr int kTileBytes = kPfRows * D * 2;
  static constexpr int kHalf = kPfRows * 128;  // a tile is D / 64 parts of 128 rows x 128 bytes
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTileBytes + 1024 + 256;
};

struct PfArgs {
  void* out;
  const int32_t* cu_seqlens;
  uint32_t* status;
  int64_t out_stride;
  float scale_log2;
  int n_seqs, tokens, group;
  int clear;  // tokens outside of all sequences get zeros
};
struct PfMaps {
  CUtensorMap q, k, v;
};

struct PfBars {
  uint64_t q_full[2], s_full[2], s_free[2], p_full[2], o_done[2], full[8], empty[8], cleared, drained;
  uint32_t tmem;
  int aborted;
  int issued;  // copies of keys and values
};
static_assert(sizeof(PfBars) <= 256, "room behind the ring");

template <class T, int D>
__global__ void __launch_bounds__(kPfThreads, 1) attn_prefill_kernel(const PfArgs a, const __grid_constant__ PfMaps maps) {
  using S = PfShape<D>;
  constexpr int kStages = S::kStages, kParts = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_tiles = smem;
  uint8_t* ring = smem + 2 * S::kTileBytes;
  PfBars* bars = reinterpret_cast<PfBars*>(ring + kStages * S::kTileBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 9 * 32) {
    prefetch_map(&maps.q);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  pdl_wait_prior();

  // Which sequence and which 256 queries: item blockIdx.y counts the items of the sequences in order, each from its end.
  // (With `clear` the last blockIdx.y has no item.)
  int start = 0, length = -1, item = -1;
  {
    const int number = a.clear && blockIdx.y + 1 == gridDim.y ? INT32_MAX : int(blockIdx.y);
    int before = 0;
    for (int base = 0; base < a.n_seqs; base += 32) {
      const int s = base + lane;
      int lo = 0, hi = 0;
      if (s < a.n_seqs) {
        lo = a.cu_seqlens[s];
        hi = a.cu_seqlens[s + 1];
        lo = lo < 0 ? 0 : lo > a.tokens ? a.tokens : lo;
        hi = hi < lo ? lo : hi > a.tokens ? a.tokens : hi;
      }
      const int n = (hi - lo + kPfQueries - 1) / kPfQueries;
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += other;
      }
      const int at = number - before;
      const bool mine = n > 0 && at < upto && at >= upto - n;
      const uint32_t who = __ballot_sync(0xffffffffu, mine);
      if (who) {
        const int src = __ffs(who) - 1;
        start = __shfl_sync(0xffffffffu, lo, src);
        length = __shfl_sync(0xffffffffu, hi - lo, src);
        item = __shfl_sync(0xffffffffu, upto - 1 - at, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (item < 0) {  // (block-uniform)
      // With `clear` the blocks without an item, from `idle` on, share the tokens in front of the first and behind the last sequence, each
      // for its head. (`before` is the number of items where the ends do not fall.)
      const int idle = before >= 0 && before < int(gridDim.y) - 1 ? before : int(gridDim.y) - 1;
      if (!a.clear || int(blockIdx.y) < idle) return;
      int least = a.tokens, most = 0;
      for (int i = lane; i < a.n_seqs; i += 32) {
        const int lo = a.cu_seqlens[i] < 0 ? 0 : a.cu_seqlens[i], hi = a.cu_seqlens[i + 1] < a.tokens ? a.cu_seqlens[i + 1] : a.tokens;
        if (lo < hi) {
          least = lo < least ? lo : least;
          most = hi > most ? hi : most;
        }
      }
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
      most = most < least ? least : most;
      constexpr int kChunks = D / 8, kRows = kPfThreads / kChunks;
      const int64_t rest = int64_t(least) + a.tokens - most, step = int64_t(int(gridDim.y) - idle) * kRows;
      for (int64_t i = int64_t(int(blockIdx.y) - idle) * kRows + tid / kChunks; i < rest; i += step) {
        const int64_t row = i < least ? i : most + (i - least);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.out_stride + int64_t(blockIdx.x) * D + tid % kChunks * 8) = make_uint4(0, 0, 0, 0);
      }
      return;
    }
  }
  const int head = blockIdx.x, kv_head = head / a.group;
  const int row0 = item * kPfQueries;
  const int blocks0 = 2 * item + 1, blocks1 = row0 + kPfRows < length ? 2 * item + 2 : 0;
  const int blocks = blocks1 ? blocks1 : blocks0;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // (the copying thread makes the barriers and begins, while the others are on their way)
  constexpr int kCopier = 9 * 32, kEarly = 3;  // copies of keys and values before the barrier
  auto copy = [&](uint8_t* dst, const CUtensorMap* map, int h, int row, uint64_t* bar) {
    mbar_expect_tx(bar, S::kTileBytes);
    for (int p = 0; p < kParts; ++p) tma_load_3d(smem_u32(dst) + p * S::kHalf, map, p * 64, h, row, bar);
  };
  auto copy_block = [&](int i) {  // K_0 V_0 K_1 V_1 ...
    const int slot = i % kStages;
    copy(ring + slot * S::kTileBytes, i & 1 ? &maps.v : &maps.k, kv_head, start + (i >> 1) * kPfRows, &bars->full[slot]);
    bars->issued = i + 1;
  };
  if (tid == kCopier) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->s_free[i], kPfRows);
      mbar_init(&bars->p_full[i], kPfRows);
      mbar_init(&bars->o_done[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->cleared, 1);
    mbar_init(&bars->drained, 2);
    bars->aborted = 0;
    bars->issued = 0;
    mbar_fence_init();
    copy(q_tiles, &maps.q, head, start + row0, &bars->q_full[0]);
    copy_block(0);
    if (blocks1) copy(q_tiles + S::kTileBytes, &maps.q, head, start + row0 + kPfRows, &bars->q_full[1]);
    for (int i = 1; i < kEarly && i < 2 * blocks; ++i) copy_block(i);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (not before the allocation: a block of the next kernel that took tensor memory and then waited for this one would hold it up)
  pdl_launch_dependents();
  // All 512 columns: their address is 0, and every address in tensor memory a constant.
  if (bars->tmem != 0 && tid == 0 && a.status) atomicMax(a.status, uint32_t(FB_STATUS_BAD_WORK));
  constexpr uint32_t kS = 0, kP = 128, kO = 256;  // S; tile i: P in columns 128 + 64 i, O in 256 + 128 i

  // 256 threads x 208 and 128 x 88 registers are the 384 x 168 of the launch.
  if (warp >= 8) {
    regs_down<88>();
    if (warp == 9) {
      // ------------------------------------------------------------------ copies
      if (lane == 0) {
        for (int i = kEarly; i < 2 * blocks; ++i) {
          if (i >= kStages && !bounded_wait(&bars->aborted, a.status, &bars->empty[i % kStages], uint32_t(i / kStages - 1) & 1)) break;
          copy_block(i);
        }
      }
      __syncwarp();
      // Rows of the next sequence in the last block: their weights are zero, but they need not be finite. (The barrier is in the phase of
      // this last copy: its slot was free before.)
      const int i = 2 * blocks - 1, slot = i % kStages, there = length - (blocks - 1) * kPfRows;
      if (there < kPfRows && bounded_wait_warp(&bars->aborted, a.status, &bars->full[slot], uint32_t(i / kStages) & 1)) {
        for (int c = lane; c < (kPfRows - there) * (D / 8); c += 32) {
          const int row = there + c / (D / 8), chunk = c % (D / 8);
          *reinterpret_cast<uint4*>(ring + slot * S::kTileBytes + (chunk / 8) * S::kHalf + row * 128 + (chunk % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->cleared);
      }
    } else if (warp != 11) {
      // ------------------------------------------------------------------ products: a thread for the scores, one for the outputs
      // (The scores must not wait behind outputs whose weights are not there yet. One thread for all products: 4000 cycles per block of
      // keys, one for each tile 3650.)
      constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t kIdesc = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kPfRows >> 4) << 24);
      constexpr uint32_t kIdescQk = kIdesc | (uint32_t(kPfRows >> 3) << 17);
      constexpr uint32_t kIdescPv = kIdesc | (uint32_t(D >> 3) << 17) | (1u << 16);  // V runs along N
      if (elect_one()) {
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && bounded_spin(&bars->aborted, a.status, bar, parity); };
        if (warp == 8) {
          int held_by = -1, held_at = 0;  // whose scores S holds
          for (int j = 0; j < blocks && ok; ++j) {
            const int slot = (2 * j) % kStages;
            wait(&bars->full[slot], uint32_t(2 * j / kStages) & 1);
            const uint32_t kd = umma_desc_lo(smem_u32(ring + slot * S::kTileBytes), 1);
#pragma unroll 1
            for (int t = j < blocks0 ? 0 : 1; t < (j < blocks1 ? 2 : 1); ++t) {
              if (j == 0) wait(&bars->q_full[t], 0);
              if (held_by >= 0) wait(&bars->s_free[held_by], uint32_t(held_at) & 1);
              if (!ok) break;
              held_by = t;
              held_at = j;
              tc_fence_after();
              const uint32_t qd = umma_desc_lo(smem_u32(q_tiles + t * S::kTileBytes), 1);
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t at = (k / 4) * (S::kHalf >> 4) + (k % 4) * 2;
                umma_ss<kIdescQk>(kS, qd + at, kd + at, k > 0);
              }
              umma_commit(&bars->s_full[t]);
            }
            if (ok) umma_commit(&bars->empty[slot]);
          }
        } else {
          for (int j = 0; j < blocks && ok; ++j) {
            const int slot = (2 * j + 1) % kStages;
            wait(&bars->full[slot], uint32_t((2 * j + 1) / kStages) & 1);
            if (length - j * kPfRows < kPfRows) wait(&bars->cleared, 0);
            const uint32_t vd = umma_desc_lo(smem_u32(ring + slot * S::kTileBytes), S::kHalf >> 4);
#pragma unroll 1
            for (int t = j < blocks0 ? 0 : 1; t < (j < blocks1 ? 2 : 1); ++t) {
              wait(&bars->p_full[t], uint32_t(j) & 1);
              if (!ok) break;
              tc_fence_after();
              const uint32_t d = kO + 128 * t, p = kP + 64 * t;
              umma_ts<kIdescPv>(d, p, vd, j > 0);
#pragma unroll
              for (int k = 1; k < kPfRows / 16; ++k) umma_ts<kIdescPv>(d, p + 8 * k, vd + k * (2048 >> 4), true);
              umma_commit(&bars->o_done[t]);
            }
            if (ok) umma_commit(&bars->empty[slot]);
          }
        }
        // Nothing issued here is still running when the tensor memory is given back.
        umma_commit(&bars->drained);
      }
      __syncwarp();
      for (uint32_t i = 0; i < (1u << 16) && !__all_sync(0xffffffffu, mbar_try_wait_hint(&bars->drained, 0)); ++i) {}
    }
  } else {
    regs_up<208>();
    // ------------------------------------------------------------------ softmax
    const int t = warp >> 2, row = tid & 127;
    const int n = t ? blocks1 : blocks0;
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // (32 (warp % 4)) << 16
    const uint32_t s_at = lanes + kS, p_at = lanes + kP + 64 * t, o_at = lanes + kO + 128 * t;
    const bool real = row0 + t * kPfRows + row < length;
    const uint64_t scale = pair_of(a.scale_log2, a.scale_log2);
    float top = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = ok && bounded_wait_warp(&bars->aborted, a.status, &bars->s_full[t], uint32_t(j) & 1);
      if (!ok) break;
      tc_fence_after();
      float s[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(s_at + 32 * i, s[i]);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_landed(s[i]);
      tc_fence_before();
      mbar_arrive(&bars->s_free[t]);
      if (j == n - 1) {  // the diagonal
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (32 * i + c > row) s[i][c] = -INFINITY;
      }
      float latest = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) latest = scores_max(s[i], latest);
      // (always in the first block; from a score that is NaN on, with the maximum, the sum and the outputs NaN; rows behind the sequence
      // are nobody's and decide nothing)
      const bool rises = real && !((latest - top) * a.scale_log2 <= kPfSlack);
      // P and O are free: the block before's product is done.
      if (j > 0) ok = bounded_wait_warp(&bars->aborted, a.status, &bars->o_done[t], uint32_t(j - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (__any_sync(0xffffffffu, rises)) {
        const float up = max3(latest, top, top);
        const float fade = exp2_approx((top - up) * a.scale_log2);
        top = up;
        sum *= fade;
        if (j > 0) {
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
      const float base = top * a.scale_log2 - kLift<T>;
      const uint64_t minus = pair_of(-base, -base);
      uint64_t part[2] = {0, 0};
      if (j == n - 1) {  // (masked scores stay with the exponential unit: exactly zero)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
          scores_exp<T, false>(s[i], scale, minus, p, part);
          tmem_st16(p_at + 16 * i, p);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
          scores_exp<T, true>(s[i], scale, minus, p, part);
          tmem_st16(p_at + 16 * i, p);
        }
      }
      sum += pairs_sum(part);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_full[t]);
    }
    if (n > 0 && ok) ok = bounded_wait_warp(&bars->aborted, a.status, &bars->o_done[t], uint32_t(n - 1) & 1);
    if (n > 0 && ok) {
      tc_fence_after();
      // Through the query tile's memory, which nothing reads any more, to whole rows of 16-byte stores.
      const float inv = 1.f / sum;
      uint8_t* stage = q_tiles + t * S::kTileBytes + (warp & 3) * (32 * D * 2);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float o[32];
        tmem_ld32(o_at + 32 * i, o);
        tmem_ld_wait();
        tmem_landed(o);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint4 v;
          v.x = pack2<T>(o[8 * c] * inv, o[8 * c + 1] * inv);
          v.y = pack2<T>(o[8 * c + 2] * inv, o[8 * c + 3] * inv);
          v.z = pack2<T>(o[8 * c + 4] * inv, o[8 * c + 5] * inv);
          v.w = pack2<T>(o[8 * c + 6] * inv, o[8 * c + 7] * inv);
          *reinterpret_cast<uint4*>(stage + lane * (D * 2) + (((4 * i + c) ^ (lane & 7)) << 4)) = v;
        }
      }
      __syncwarp();
      constexpr int kChunks = D / 8, kRows = 32 / kChunks;
      const int chunk = lane % kChunks;
#pragma unroll 4
      for (int i = 0; i < 32 / kRows; ++i) {
        const int r = i * kRows + lane / kChunks, q = row0 + t * kPfRows + (warp & 3) * 32 + r;
        if (q < length) {
          const uint4 v = *reinterpret_cast<const uint4*>(stage + r * (D * 2) + ((chunk ^ (r & 7)) << 4));
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + int64_t(start + q) * a.out_stride + head * D + chunk * 8) = v;
        }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  tc_fence_after();
  if (bars->aborted && tid == 0) {  // copies that nobody waited for
    const int issued = bars->issued;
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
      for (uint32_t n = 0; n < (1u << 16) && !mbar_try_wait_hint(&bars->full[i % kStages], uint32_t(i / kStages) & 1); ++n) {}
    for (int i = 0; i < (blocks1 ? 2 : 1); ++i)
      for (uint32_t n = 0; n < (1u << 16) && !mbar_try_wait_hint(&bars->q_full[i], 0); ++n) {}
  }
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(bars->tmem), "r"(512) : "memory");
}

// [tokens][heads][dim] in boxes of 128 tokens x 64 values of one head; tokens behind the last one read as zeros.
bool pf_map(CUtensorMap* map, const void* base, bool bf16, int dim, int heads, int tokens, int64_t stride) {
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(dim) * 2, cuuint64_t(stride) * 2};
  const cuuint32_t box[3] = {64, 1, kPfRows}, elem[3] = {1, 1, 1};
  return encode_tiled_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D>
cudaError_t launch_pf(const PfArgs& a, const PfMaps& maps, dim3 grid, cudaStream_t s) {
  static PerDeviceOnce once;
  const cudaError_t e = per_device_once(once, [] { return opt_in_smem(attn_prefill_kernel<T, D>, PfShape<D>::kSmem); });
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_prefill_kernel<T, D>, grid, dim3(kPfThreads), size_t(PfShape<D>::kSmem), s, a, maps);
}

// The call; clear: tokens outside of all sequences get zeros.
int32_t attn_prefill(const fb_qkv* in, int32_t tokens, const int32_t* cu_seqlens, int32_t n_seqs, float scale, void* out, int64_t out_stride,
                     uint32_t* status, void* stream, bool clear) {
  if (!in) return invalid("attn_prefill: null argument");
  const int dim = in->head_dim;
  if (in->dtype != FB_DT_BF16 && in->dtype != FB_DT_F16) return invalid("attn_prefill: bf16 or fp16");
  if (dim != 64 && dim != 128) return invalid("attn_prefill: head_dim 64 or 128");
  if (in->kv_heads < 1 || in->heads < in->kv_heads || in->heads % in->kv_heads || in->heads > 1024)
    return invalid("attn_prefill: heads is a multiple of kv_heads, up to 1024");
  if (tokens < 0 || n_seqs < 0) return invalid("attn_prefill: tokens or n_seqs is negative");
  if (!tokens || (!n_seqs && !clear)) return 0;
  if (!in->q || !in->k || !in->v || !out || !cu_seqlens) return invalid("attn_prefill: null argument");
  if (in->q_stride < int64_t(in->heads) * dim || in->k_stride < int64_t(in->kv_heads) * dim ||
      in->v_stride < int64_t(in->kv_heads) * dim || out_stride < int64_t(in->heads) * dim)
    return invalid("attn_prefill: a stride is smaller than a token's heads");
  if ((in->q_stride | in->k_stride | in->v_stride) >= int64_t(1) << 38) return invalid("attn_prefill: a stride is too large");
  if ((reinterpret_cast<uintptr_t>(in->q) | reinterpret_cast<uintptr_t>(in->k) | reinterpret_cast<uintptr_t>(in->v) |
       reinterpret_cast<uintptr_t>(out)) & 15 || (in->q_stride | in->k_stride | in->v_stride | out_stride) % 8)
    return invalid("attn_prefill: tensors start on 16 bytes and tokens lie a multiple of 8 elements apart");
  if ((reinterpret_cast<uintptr_t>(cu_seqlens) | reinterpret_cast<uintptr_t>(status)) & 3)
    return invalid("attn_prefill: cu_seqlens or status is not aligned");
  if (!(scale > 0.f && scale <= 1.0e30f)) return invalid("attn_prefill: scale is not positive and finite");
  const int64_t items = tokens / kPfQueries + int64_t(n_seqs < tokens ? n_seqs : tokens);
  if (items + clear > 65535) return invalid("attn_prefill: more than 65535 blocks of 256 queries");
  if (!encode_tiled_fn()) {
    set_error("attn_prefill: cuTensorMapEncodeTiled is not available");
    return int32_t(cudaErrorNotSupported);
  }
  const bool bf = in->dtype == FB_DT_BF16;
  PfMaps maps;
  if (!pf_map(&maps.q, in->q, bf, dim, in->heads, tokens, in->q_stride) ||
      !pf_map(&maps.k, in->k, bf, dim, in->kv_heads, tokens, in->k_stride) ||
      !pf_map(&maps.v, in->v, bf, dim, in->kv_heads, tokens, in->v_stride))
    return invalid("attn_prefill: cuTensorMapEncodeTiled failed");
  PfArgs a;
  a.out = out;
  a.cu_seqlens = cu_seqlens;
  a.status = status;
  a.out_stride = out_stride;
  a.scale_log2 = scale * 1.4426950408889634f;  // scores are kept in powers of two
  a.n_seqs = n_seqs;
  a.tokens = tokens;
  a.group = in->heads / in->kv_heads;
  a.clear = clear;
  const dim3 grid(unsigned(in->heads), unsigned(items + clear));
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = dim == 64 ? (bf ? launch_pf<__nv_bfloat16, 64>(a, maps, grid, s) : launch_pf<__half, 64>(a, maps, grid, s))
                                  : (bf ? launch_pf<__nv_bfloat16, 128>(a, maps, grid, s) : launch_pf<__half, 128>(a, maps, grid, s));
  const int32_t st = check_launch("attn_prefill");
  return st ? st : int32_t(e);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

int32_t fb_attn_prefill(const fb_qkv* in, int32_t tokens, const int32_t* cu_seqlens, int32_t n_seqs, float scale, void* out,
                        int64_t out_stride, uint32_t* status, void* stream) {
  return attn_prefill(in, tokens, cu_seqlens, n_seqs, scale, out, out_stride, status, stream, false);
}

int32_t fb_attn_prefill_padded(const fb_qkv* in, int32_t tokens, const int32_t* cu_seqlens, int32_t n_seqs, float scale, void* out,
                               int64_t out_stride, uint32_t* status, void* stream) {
  return attn_prefill(in, tokens, cu_seqlens, n_seqs, scale, out, out_stride, status, stream, true);
}

}  // extern "C"
