// Norms of queries and keys per head and their rotation, in one pass over a projection's output; keys and values go to
// where the attention reads them.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                                   per head of q and k
//   (a, b) -> (a cos p - b sin p, b cos p + a sin p),  p = position[axis(j)] * inv_freq[j]     frequency j's pair
//
// Bound by memory: every value is read once and written once. A block takes a token (or a share of its heads) after the other; D / 8
// lanes hold a head, 16 bytes each, and the next token's values are on their way while this one's are worked on. The angles of a
// token are made once per block: the product of position and frequency in 64 bits, reduced to a part of a turn there
// (a position of a million leaves fp32 no more than four correct digits of the angle), the sine and cosine of the rest in fp32.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace fb {
namespace {

constexpr int kQkThreads = 256;
constexpr int kQkRows = 4;    // heads a thread works on at a time, and as many are in flight behind them
constexpr int kQkBlocks = 2;  // per multiprocessor

struct QkArgs {
  const void* in[3];     // q, k, v
  void* out[3];
  int64_t in_stride[3];  // elements between tokens
  int64_t out_stride[3];
  const void* weight[2];
  const float* inv_freq;
  const int32_t* positions;
  int64_t axis_stride;
  const int64_t* slots;
  int64_t n_slots;
  float eps;
  int weight_dtype, heads, kv_heads, half, adjacent;
  int rows;              // heads of all tensors
  int tokens;
  int first[3];          // first row of q, k, v
  int section_end[4];
};

template <class T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == FB_DT_F32) return static_cast<const float*>(w)[i];
  if (dtype == FB_DT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

template <class T, int D>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const QkArgs a) {
  constexpr int kLanes = D / 8;                    // lanes of a head
  constexpr int kPerPass = kQkThreads / kLanes;    // heads of a block per row of a thread
  __shared__ float cs[2][2][D / 2];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int l = threadIdx.x % kLanes, e0 = 8 * l, slot_row = threadIdx.x / kLanes;
  const int step = kPerPass * gridDim.y, first_row = blockIdx.y * kPerPass + slot_row;
  auto which = [&](int row) { return row >= a.first[2] ? 2 : row >= a.first[1] ? 1 : 0; };
  // Every thread stays for the shuffles; a row behind the last one is not loaded and not stored.
  auto load = [&](int64_t token, int row0, uint4 (&raw)[kQkRows]) {
#pragma unroll
    for (int i = 0; i < kQkRows; ++i) {
      const int row = row0 + i * step;
      if (row < a.rows) {
        const int w = which(row);
        raw[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.in[w]) + token * a.in_stride[w] + (row - a.first[w]) * D + e0);
      } else {
        raw[i] = make_uint4(0, 0, 0, 0);
      }
    }
  };
  int64_t token = blockIdx.x;
  int row0 = first_row;
  uint4 raw[kQkRows];
  load(token, row0, raw);
  // Thread j makes frequency j's sine and cosine.
  const int j = threadIdx.x;
  const bool turns_one = j < a.half;
  const int32_t* positions = nullptr;
  double turns_per = 0.0;
  int position = 0;
  if (turns_one) {
    const int axis = (j >= a.section_end[0]) + (j >= a.section_end[1]) + (j >= a.section_end[2]);
    positions = a.positions + axis * a.axis_stride;
    position = positions[token];
    turns_per = double(a.inv_freq[j]) * 0.15915494309189533577;  // 1 / (2 pi)
  }
  int64_t slot = a.slots ? a.slots[token] : token;
  float wt[2][8];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) wt[w][i] = a.weight[w] ? weight_at(a.weight[w], a.weight_dtype, e0 + i) : 1.f;
  const bool turned = e0 < 2 * a.half;
  // The lane that holds the partners of an element pair (i, i + rot / 2), in this head's lanes.
  const int lane = threadIdx.x & 31;
  const int partner = !turned || a.adjacent ? lane : e0 < a.half ? lane + a.half / 8 : lane - a.half / 8;
  float co[8], si[8];
  int buffer = 0;
  bool fresh = true;
  for (;;) {
    if (fresh) {
      // This lane's cosines and sines, one per element: the sine carries the sign of the partner's product.
      if (turns_one) {
        const double turns = double(position) * turns_per;
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        cs[buffer][0][j] = c;
        cs[buffer][1][j] = s;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        co[i] = 1.f;
        si[i] = 0.f;
        if (turned) {
          const int e = e0 + i, f = a.adjacent ? e >> 1 : e < a.half ? e : e - a.half;
          const bool low = a.adjacent ? !(e & 1) : e < a.half;
          co[i] = cs[buffer][0][f];
          si[i] = low ? -cs[buffer][1][f] : cs[buffer][1][f];
        }
      }
      buffer ^= 1;
    }
    // What comes after these rows is asked for before they are worked on.
    int64_t next_token = token, next_slot = slot;
    int next_row = row0 + kQkRows * step;
    fresh = next_row - slot_row >= a.rows;  // (block-uniform)
    if (fresh) {
      next_token += gridDim.x;
      next_row = first_row;
    }
    const bool more = next_token < a.tokens;
    uint4 next_raw[kQkRows];
    if (more) {
      load(next_token, next_row, next_raw);
      if (fresh) {
        if (turns_one) position = positions[next_token];
        next_slot = a.slots ? a.slots[next_token] : next_token;
      }
    }
#pragma unroll
    for (int i = 0; i < kQkRows; ++i) {
      const int row = row0 + i * step;
      if (row - slot_row >= a.rows) break;  // (block-uniform)
      const int w = row < a.rows ? which(row) : 2;
      float x[8];
      unpack8<T>(raw[i], x);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      const bool norm = w < 2 && a.weight[w];
      const float r = norm ? rsqrtf(sum * (1.f / D) + a.eps) : 1.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * (w == 1 ? wt[1][e] : wt[0][e]);
      float y[8];
      if (a.adjacent) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], co[e], x[e ^ 1] * si[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __shfl_sync(0xffffffffu, x[e], partner);
          y[e] = fmaf(x[e], co[e], turned ? p * si[e] : 0.f);
        }
      }
      if (row < a.rows) {
        const uint4 v = w == 2 ? raw[i] : pack8<T>(y);
        // (a slot outside of the cache is not stored)
        const int64_t to = w == 0 ? token : !a.slots || (slot >= 0 && slot < a.n_slots) ? slot : -1;
        if (to >= 0)
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out[w]) + to * a.out_stride[w] + (row - a.first[w]) * D + e0) = v;
      }
    }
    if (!more) break;
#pragma unroll
    for (int i = 0; i < kQkRows; ++i) raw[i] = next_raw[i];
    token = next_token;
    slot = next_slot;
    row0 = next_row;
  }
}

template <class T>
cudaError_t launch_qk(const QkArgs& a, int dim, dim3 grid, cudaStream_t s) {
  if (dim == 64) return launch_pdl(qk_norm_rope_kernel<T, 64>, grid, dim3(kQkThreads), 0, s, a);
  if (dim == 128) return launch_pdl(qk_norm_rope_kernel<T, 128>, grid, dim3(kQkThreads), 0, s, a);
  return launch_pdl(qk_norm_rope_kernel<T, 256>, grid, dim3(kQkThreads), 0, s, a);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

int32_t fb_qk_norm_rope(const fb_qkv* in, int32_t tokens, const fb_qk_norm* norm, const fb_rope* rope, const fb_qkv_out* out,
                        void* stream) {
  if (!in || !out) return invalid("qk_norm_rope: null argument");
  if (tokens < 0) return invalid("qk_norm_rope: tokens is negative");
  const int dim = in->head_dim;
  if (dim != 64 && dim != 128 && dim != 256) return invalid("qk_norm_rope: head_dim 64, 128 or 256");
  if (in->dtype != FB_DT_BF16 && in->dtype != FB_DT_F16) return invalid("qk_norm_rope: bf16 or fp16");
  if (in->heads < 0 || in->kv_heads < 0 || in->heads > 1024 || in->kv_heads > 1024)
    return invalid("qk_norm_rope: 0..1024 heads");
  if (!tokens) return 0;
  const void* from[3] = {in->q, in->k, in->v};
  void* to[3] = {out->q, out->k, out->v};
  const int64_t from_stride[3] = {in->q_stride, in->k_stride, in->v_stride};
  const int64_t to_stride[3] = {out->q_stride, out->k_stride, out->v_stride};
  QkArgs a;
  a.rows = 0;
  for (int i = 0; i < 3; ++i) {
    const int h = i ? in->kv_heads : in->heads;
    if (!from[i] != !to[i]) return invalid("qk_norm_rope: an input and its output are given together, or neither");
    a.in[i] = from[i];
    a.out[i] = to[i];
    a.in_stride[i] = from_stride[i];
    a.out_stride[i] = to_stride[i];
    a.first[i] = a.rows;
    if (!from[i]) continue;
    if (h <= 0) return invalid("qk_norm_rope: a tensor without heads");
    if ((reinterpret_cast<uintptr_t>(from[i]) | reinterpret_cast<uintptr_t>(to[i])) & 15 || from_stride[i] % 8 || to_stride[i] % 8)
      return invalid("qk_norm_rope: tensors start on 16 bytes and their tokens lie a multiple of 8 elements apart");
    if (from_stride[i] < int64_t(h) * dim || to_stride[i] < int64_t(h) * dim)
      return invalid("qk_norm_rope: a stride is smaller than a token's heads");
    a.rows += h;
  }
  if (!a.rows) return invalid("qk_norm_rope: nothing to do");
  a.weight[0] = norm ? norm->q_weight : nullptr;
  a.weight[1] = norm ? norm->k_weight : nullptr;
  a.weight_dtype = norm ? norm->weight_dtype : FB_DT_F32;
  a.eps = norm ? norm->eps : 0.f;
  if (norm) {
    if (a.weight_dtype != FB_DT_F32 && a.weight_dtype != FB_DT_BF16 && a.weight_dtype != FB_DT_F16)
      return invalid("qk_norm_rope: weights are fp32, bf16 or fp16");
    if (!(norm->eps >= 0.f)) return invalid("qk_norm_rope: eps is negative");
    if ((reinterpret_cast<uintptr_t>(a.weight[0]) | reinterpret_cast<uintptr_t>(a.weight[1])) & (a.weight_dtype == FB_DT_F32 ? 3 : 1))
      return invalid("qk_norm_rope: weights are not aligned to their elements");
  }
  a.half = 0;
  a.adjacent = 0;
  a.inv_freq = nullptr;
  a.positions = nullptr;
  a.axis_stride = 0;
  for (int& e : a.section_end) e = 0;
  if (rope) {
    if (rope->rot_dim <= 0 || rope->rot_dim % 16 || rope->rot_dim > dim)
      return invalid("qk_norm_rope: rot_dim is a multiple of 16 up to head_dim");
    if (rope->axes < 1 || rope->axes > 4) return invalid("qk_norm_rope: 1..4 axes");
    if (!rope->inv_freq || !rope->positions) return invalid("qk_norm_rope: rope without frequencies or positions");
    if ((reinterpret_cast<uintptr_t>(rope->inv_freq) | reinterpret_cast<uintptr_t>(rope->positions)) & 3)
      return invalid("qk_norm_rope: frequencies and positions are not aligned to their elements");
    a.half = rope->rot_dim / 2;
    int end = 0;
    for (int i = 0; i < 4; ++i) {
      const int n = rope->axes == 1 ? (i ? 0 : a.half) : i < rope->axes ? rope->sections[i] : 0;
      if (n < 0 || n > a.half) return invalid("qk_norm_rope: a section is negative or too long");
      a.section_end[i] = end += n;
    }
    if (end != a.half) return invalid("qk_norm_rope: the sections do not add up to rot_dim / 2");
    if (rope->axes > 1 && rope->axis_stride < tokens) return invalid("qk_norm_rope: axis_stride is smaller than tokens");
    // (axes behind the last one are never reached: a frequency is below the last section's end)
    a.adjacent = rope->adjacent != 0;
    a.inv_freq = rope->inv_freq;
    a.positions = rope->positions;
    a.axis_stride = rope->axis_stride;
  }
  a.slots = out->slots;
  a.n_slots = out->n_slots;
  if (a.slots && (reinterpret_cast<uintptr_t>(a.slots) & 7)) return invalid("qk_norm_rope: slots are not aligned");
  if (a.slots && a.n_slots <= 0) return invalid("qk_norm_rope: slots without n_slots");
  a.heads = in->heads;
  a.kv_heads = in->kv_heads;
  a.tokens = tokens;
  // A block per token with up to kQkRows heads per thread and pass, kQkBlocks of them per multiprocessor, each with every so many of
  // the tokens; few tokens share their heads among more blocks.
  const int per_pass = kQkThreads / (dim / 8), passes = (a.rows + per_pass - 1) / per_pass, most = kQkBlocks * sm_count();
  int share = 1;
  while (share < passes && tokens * share < sm_count()) share *= 2;
  const dim3 grid(unsigned(tokens < most ? tokens : most), unsigned(share < passes ? share : passes));
  const cudaError_t e = in->dtype == FB_DT_BF16 ? launch_qk<__nv_bfloat16>(a, dim, grid, as_stream(stream))
                                                : launch_qk<__half>(a, dim, grid, as_stream(stream));
  const int32_t st = check_launch("qk_norm_rope");
  return st ? st : int32_t(e);
}

}  // extern "C"
