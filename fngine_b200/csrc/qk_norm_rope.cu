// Norms of queries and keys per head and their rotation, in one pass over a projection's output; keys and values go to
// where the attention reads them.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                                   per head of q and k
//   (a, b) -> (a cos p - b sin p, b cos p + a sin p),  p = position[axis(j)] * inv_freq[j]     frequency j's pair
//
// Bound by memory latency: every value is read once and written once, 8192 tokens of 48 heads of 128 in 54 us = 3.7 TB/s (a copy: 6.5). A block takes a token (or a share of its heads) after the other; D / 8
// lanes hold a head, 16 bytes each, and the next token's values are on their way while this one's are worked on. The angles of a
// token are made once per block: the product of position and frequency in 64 bits, reduced to a part of a turn there
// (a position of a million leaves fp32 no more than four correct digits of the angle), the sine and cosine of the rest in fp32.
#include "attn_common.cuh"

namespace fb {
namespace {

constexpr int kQkThreads = 256;
constexpr int kQkRows = 4;    // heads a thread works on at a time, and as many are in flight behind them
constexpr int kQkBlocks = 3;  // per multiprocessor
constexpr int kQkTile = 4;    // tokens whose angles are made together

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
  int tokens, tile;
  int first[3];          // first row of q, k, v
  int section_end[4];
};

// Eight values as pairs of fp32, and back with one rounding each.
template <class T>
__device__ __forceinline__ void unpack8(const uint4& v, uint64_t (&f)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __nv_bfloat16>::value) {
      f[i] = pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pair_of(p.x, p.y);
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpair(f[i], a, b);
    w[i] = pack2<T>(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == FB_DT_F32) return static_cast<const float*>(w)[i];
  if (dtype == FB_DT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// Norm weight and rotation of a value are two factors, of itself and of its partner in the pair, the same for all heads of a token:
//   y[e] = r (x[e] own[e] + x[partner(e)] other[e]),   r = rsqrt(mean(x^2) + eps)
// A block keeps them for the tokens of a tile, in the order in which a warp's lanes read them: 16-byte pieces side by side.
template <int D>
struct QkFactors {
  ulonglong2 piece[4][D / 8];  // own 0-3, own 4-7, other 0-3, other 4-7 of each lane's eight values
  __device__ __forceinline__ void set(int e, float own, float other) {
    reinterpret_cast<float*>(&piece[(e >> 2) & 1][e >> 3])[e & 3] = own;
    reinterpret_cast<float*>(&piece[2 + ((e >> 2) & 1)][e >> 3])[e & 3] = other;
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kQkThreads, kQkBlocks) qk_norm_rope_kernel(const QkArgs a) {
  constexpr int kLanes = D / 8;                    // lanes of a head
  constexpr int kPerPass = kQkThreads / kLanes;    // heads of a block per row of a thread
  constexpr int kAngles = (kQkTile * (D / 2) + kQkThreads - 1) / kQkThreads;  // per thread and tile
  __shared__ QkFactors<D> factors[2][kQkTile][2];  // of q and k; the next tile's are made while this one's are in use
  __shared__ float weights[2][D];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int l = threadIdx.x % kLanes, e0 = 8 * l, slot_row = threadIdx.x / kLanes;
  const int tile = a.tile;
  // This thread's rows, the same of every token. Every thread stays for the shuffles; a row behind the last one is not loaded and not
  // stored.
  int kind[kQkRows], off[kQkRows];  // 0 q, 1 k, 2 v, 3 none; values from the token's first
  uint32_t used = 0, turns = 0;     // bit i: the block has rows there; this warp has rows of q or k there
#pragma unroll
  for (int i = 0; i < kQkRows; ++i) {
    const int row = (i * gridDim.y + blockIdx.y) * kPerPass + slot_row;
    kind[i] = row >= a.rows ? 3 : row >= a.first[2] ? 2 : row >= a.first[1] ? 1 : 0;
    off[i] = (row - (kind[i] == 0 ? a.first[0] : kind[i] == 1 ? a.first[1] : a.first[2])) * D + e0;
    if ((i * int(gridDim.y) + int(blockIdx.y)) * kPerPass < a.rows) used |= 1u << i;
    if (__any_sync(0xffffffffu, kind[i] < 2)) turns |= 1u << i;
  }
  auto load = [&](int64_t token, uint4 (&raw)[kQkRows]) {
    const T* q = static_cast<const T*>(a.in[0]) + token * a.in_stride[0];
    const T* k = static_cast<const T*>(a.in[1]) + token * a.in_stride[1];
    const T* v = static_cast<const T*>(a.in[2]) + token * a.in_stride[2];
#pragma unroll
    for (int i = 0; i < kQkRows; ++i)
      raw[i] = kind[i] < 3 ? *reinterpret_cast<const uint4*>((kind[i] == 0 ? q : kind[i] == 1 ? k : v) + off[i]) : make_uint4(0, 0, 0, 0);
  };
  int64_t token0 = int64_t(blockIdx.x) * tile;
  uint4 raw[kQkRows];
  load(token0, raw);
  int64_t next_slot = a.slots ? a.slots[token0] : 0;
  // Thread and index i take an angle of the tile: (token, frequency), the positions asked for a tile ahead.
  int position[kAngles];
  auto ask = [&](int64_t first) {
#pragma unroll
    for (int i = 0; i < kAngles; ++i) {
      const int id = threadIdx.x + i * kQkThreads, t = a.half ? id / a.half : tile, f = id - t * a.half;
      position[i] = 0;
      if (t < tile && first + t < a.tokens) {
        const int axis = (f >= a.section_end[0]) + (f >= a.section_end[1]) + (f >= a.section_end[2]);
        position[i] = a.positions[axis * a.axis_stride + first + t];
      }
    }
  };
  ask(token0);
  for (int e = threadIdx.x; e < 2 * D; e += kQkThreads) {
    const int w = e / D;
    weights[w][e % D] = a.weight[w] ? weight_at(a.weight[w], a.weight_dtype, e % D) : 1.f;
  }
  __syncthreads();
  for (int id = threadIdx.x; id < 2 * kQkTile * 2 * D; id += kQkThreads) {  // values that are not turned: once for all
    const int e = id % D, w = id / D % 2, t = id / (2 * D) % kQkTile;
    if (e >= 2 * a.half) factors[id / (2 * D * kQkTile)][t][w].set(e, weights[w][e], 0.f);
  }
  const bool normed[2] = {a.weight[0] != nullptr, a.weight[1] != nullptr};
  const bool turned = e0 < 2 * a.half;
  // The lane that holds the partners of an element pair (i, i + rot / 2), in this head's lanes.
  const int lane = threadIdx.x & 31;
  const int partner = !turned || a.adjacent ? lane : e0 < a.half ? lane + a.half / 8 : lane - a.half / 8;
  int buffer = 0;
  for (; token0 < a.tokens; token0 += int64_t(gridDim.x) * tile, buffer ^= 1) {
#pragma unroll
    for (int i = 0; i < kAngles; ++i) {
      const int id = threadIdx.x + i * kQkThreads, t = a.half ? id / a.half : tile, f = id - t * a.half;
      if (t < tile) {
        const double turns = double(position[i]) * (double(a.inv_freq[f]) * 0.15915494309189533577);  // 1 / (2 pi)
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        const int lo = a.adjacent ? 2 * f : f, hi = a.adjacent ? 2 * f + 1 : f + a.half;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float wl = weights[w][lo], wh = weights[w][hi];
          factors[buffer][t][w].set(lo, wl * c, -wh * s);
          factors[buffer][t][w].set(hi, wh * c, wl * s);
        }
      }
    }
    ask(token0 + int64_t(gridDim.x) * tile);
    __syncthreads();
    const int here = a.tokens - token0 < tile ? int(a.tokens - token0) : tile;
    for (int t = 0; t < here; ++t) {
      const int64_t token = token0 + t, next = t + 1 < here ? token + 1 : token0 + int64_t(gridDim.x) * tile;
      uint4 next_raw[kQkRows];
      const int64_t slot = a.slots ? next_slot : token;
      const bool kept = !a.slots || (slot >= 0 && slot < a.n_slots);
      if (next < a.tokens) {
        load(next, next_raw);
        if (a.slots) next_slot = a.slots[next];
      }
      T* q = static_cast<T*>(a.out[0]) + token * a.out_stride[0];
      T* k = static_cast<T*>(a.out[1]) + slot * a.out_stride[1];
      T* v = static_cast<T*>(a.out[2]) + slot * a.out_stride[2];
#pragma unroll
      for (int i = 0; i < kQkRows; ++i) {
        if (!((used >> i) & 1)) break;
        uint4 result = raw[i];
        if ((turns >> i) & 1) {
          const QkFactors<D>& f = factors[buffer][t][kind[i] == 1];
          uint64_t x[4], p[4];
          unpack8<T>(raw[i], x);
          uint64_t sum2 = fma2(x[1], x[1], fma2(x[0], x[0], 0));
          sum2 = add2(sum2, fma2(x[3], x[3], fma2(x[2], x[2], 0)));
          float sum, high;
          unpair(sum2, sum, high);
          sum += high;
#pragma unroll
          for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          const float r = normed[kind[i] == 1] ? rsqrtf(fmaf(sum, 1.f / D, a.eps)) : 1.f;
          if (a.adjacent) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              unpair(x[e], lo, hi);
              p[e] = pair_of(hi, lo);
            }
          } else {
            uint4 other;
            other.x = __shfl_sync(0xffffffffu, raw[i].x, partner);
            other.y = __shfl_sync(0xffffffffu, raw[i].y, partner);
            other.z = __shfl_sync(0xffffffffu, raw[i].z, partner);
            other.w = __shfl_sync(0xffffffffu, raw[i].w, partner);
            unpack8<T>(other, p);
          }
          const ulonglong2 o0 = f.piece[0][l], o1 = f.piece[1][l];
          const uint64_t rr = pair_of(r, r);
          uint64_t y[4] = {fma2(x[0], o0.x, 0), fma2(x[1], o0.y, 0), fma2(x[2], o1.x, 0), fma2(x[3], o1.y, 0)};
          if (turned) {
            const ulonglong2 t0 = f.piece[2][l], t1 = f.piece[3][l];
            y[0] = fma2(p[0], t0.x, y[0]);
            y[1] = fma2(p[1], t0.y, y[1]);
            y[2] = fma2(p[2], t1.x, y[2]);
            y[3] = fma2(p[3], t1.y, y[3]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fma2(y[e], rr, 0);
          if (kind[i] < 2) result = pack8<T>(y);
        }
        if (kind[i] == 0 || (kind[i] < 3 && kept))
          *reinterpret_cast<uint4*>((kind[i] == 0 ? q : kind[i] == 1 ? k : v) + off[i]) = result;
      }
#pragma unroll
      for (int i = 0; i < kQkRows; ++i) raw[i] = next_raw[i];
    }
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
    if (rope->axes > 1 && rope->axis_stride && rope->axis_stride < tokens) return invalid("qk_norm_rope: axis_stride is smaller than tokens");
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
  // Up to kQkRows heads per thread, the others to more blocks; few tokens share their heads among blocks, many go to a block in tiles.
  const int per_pass = kQkThreads / (dim / 8), passes = (a.rows + per_pass - 1) / per_pass, room = kQkBlocks * sm_count();
  int share = (passes + kQkRows - 1) / kQkRows;
  while (share < passes && int64_t(tokens) * share < sm_count()) share = 2 * share < passes ? 2 * share : passes;
  a.tokens = tokens;
  // (tiles of four tokens where every block gets two of them: 8192 tokens of 48 heads took 61 us in tiles of four or two, 67 one by one; since the pair arithmetic 54 in tiles of four)
  a.tile = int64_t(tokens) * share >= 2 * int64_t(kQkTile) * room ? kQkTile : 1;
  const int across = room / share > 0 ? room / share : 1;
  const int tiles = (tokens + a.tile - 1) / a.tile;
  const dim3 grid(unsigned(tiles < across ? tiles : across), unsigned(share));
  const cudaError_t e = in->dtype == FB_DT_BF16 ? launch_qk<__nv_bfloat16>(a, dim, grid, as_stream(stream))
                                                : launch_qk<__half>(a, dim, grid, as_stream(stream));
  const int32_t st = check_launch("qk_norm_rope");
  return st ? st : int32_t(e);
}

}  // extern "C"
