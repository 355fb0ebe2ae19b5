// Norms of queries and keys per head and their rotation, in one pass over a projection's output; keys and values go to
// where the attention reads them.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                                   per head of q and k
//   (a, b) -> (a cos p - b sin p, b cos p + a sin p),  p = position[axis(j)] * inv_freq[j]     frequency j's pair
//
// Every value is read once and written once: 8192 tokens of 48 heads of 128 in 40 us = 5.1 TB/s (a copy: 6.5), 4093 of 64 heads in 30. The
// issue slots are the next limit (at 54 us, 77 % of them): so a thread takes one head of a tile's tokens after the other, with its
// addresses made once for the tile, and the next step's 16-byte pieces are on their way while this one's are worked on; D / 8 lanes hold a
// head. (A token's heads one after the other: 54 us; its values by cp.async two or three tokens ahead: 55 to 63; each block's tokens side by
// side in memory instead of a tile of every round: 56.) The angles of a tile are made once per block: the product of position and
// frequency in 64 bits, reduced to a part of a turn there (a position of a million leaves fp32 no more than four correct digits of the
// angle), the sine and cosine of the rest in fp32.
#include "attn_common.cuh"

namespace fb {
namespace {

constexpr int kQkThreads = 256;
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
  int weight_dtype, half, adjacent;
  int rows;              // heads of all tensors
  int tiles, shortest, longer;  // tiles of `shortest` tokens, the first `longer` of them with one more
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
  constexpr int kPerPass = kQkThreads / kLanes;    // heads of a block at a time
  constexpr int kAngles = (kQkTile * (D / 2) + kQkThreads - 1) / kQkThreads;  // per thread and tile
  __shared__ QkFactors<D> factors[2][kQkTile][2];  // of q and k; the next tile's are made while this one's are in use
  __shared__ float weights[2][D];
  __shared__ int64_t slots[2][kQkTile];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int l = threadIdx.x % kLanes, e0 = 8 * l, mine = threadIdx.x / kLanes, lane = threadIdx.x & 31;
  const int passes = (a.rows + kPerPass - 1) / kPerPass;
  // Every gridDim.x-th tile; the first `longer` tiles have one token more than the others.
  int at = blockIdx.x, token0 = at * a.shortest + (at < a.longer ? at : a.longer), here = a.shortest + (at < a.longer);
  // A step: one head (of q, k or v: kind 0, 1, 2, or none: 3) of the tile's tokens, one after the other.
  auto row_of = [&](int pass, int& kind, int& off) {
    const int row = pass * kPerPass + mine;
    kind = row >= a.rows ? 3 : row >= a.first[2] ? 2 : row >= a.first[1] ? 1 : 0;
    off = (row - (kind == 0 ? a.first[0] : kind == 1 ? a.first[1] : a.first[2])) * D + e0;
  };
  auto load = [&](int token, int there, int kind, int off, uint4 (&raw)[kQkTile]) {
    const int64_t stride = kind == 0 ? a.in_stride[0] : kind == 1 ? a.in_stride[1] : a.in_stride[2];
    const T* from = static_cast<const T*>(kind == 0 ? a.in[0] : kind == 1 ? a.in[1] : a.in[2]) + token * stride + off;
#pragma unroll
    for (int t = 0; t < kQkTile; ++t) {
      if (kind < 3 && t < there) raw[t] = *reinterpret_cast<const uint4*>(from);
      from += stride;
    }
  };
  uint4 raw[kQkTile] = {};
  int kind, off;
  row_of(blockIdx.y, kind, off);
  load(token0, here, kind, off, raw);
  // Thread and index i make an angle of the tile, (token, frequency), from positions that are asked for a tile ahead; the first threads
  // bring the slots.
  int angle_t[kAngles], angle_f[kAngles], position[kAngles];
  int64_t slot = 0;
  double turns_of[kAngles];  // per position
  auto ask = [&](int first, int there) {
#pragma unroll
    for (int i = 0; i < kAngles; ++i) {
      const int f = angle_f[i], axis = (f >= a.section_end[0]) + (f >= a.section_end[1]) + (f >= a.section_end[2]);
      position[i] = angle_t[i] < there ? a.positions[axis * a.axis_stride + first + angle_t[i]] : 0;
    }
    if (a.slots && int(threadIdx.x) < there) slot = a.slots[first + threadIdx.x];
  };
#pragma unroll
  for (int i = 0; i < kAngles; ++i) {
    const int id = threadIdx.x + i * kQkThreads;
    angle_t[i] = a.half ? id / a.half : kQkTile;
    angle_f[i] = a.half ? id % a.half : 0;
    turns_of[i] = angle_t[i] < kQkTile ? double(a.inv_freq[angle_f[i]]) * 0.15915494309189533577 : 0.;  // 1 / (2 pi)
  }
  ask(token0, here);
  for (int e = threadIdx.x; e < 2 * D; e += kQkThreads) {
    const int w = e / D;
    weights[w][e % D] = a.weight[w] ? weight_at(a.weight[w], a.weight_dtype, e % D) : 1.f;
  }
  __syncthreads();
  for (int id = threadIdx.x; id < 2 * kQkTile * 2 * D; id += kQkThreads) {  // values that are not turned: once for all
    const int e = id % D, w = id / D % 2, t = id / (2 * D) % kQkTile;
    if (e >= 2 * a.half) factors[id / (2 * D * kQkTile)][t][w].set(e, weights[w][e], 0.f);
  }
  const bool turned = e0 < 2 * a.half;
  // The lane that holds the partners of an element pair (i, i + rot / 2), in this head's lanes.
  const int partner = !turned || a.adjacent ? lane : e0 < a.half ? lane + a.half / 8 : lane - a.half / 8;
  for (int buffer = 0; here > 0; buffer ^= 1) {
#pragma unroll
    for (int i = 0; i < kAngles; ++i) {
      if (angle_t[i] < here) {
        const double turns = double(position[i]) * turns_of[i];
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        const int f = angle_f[i], lo = a.adjacent ? 2 * f : f, hi = a.adjacent ? 2 * f + 1 : f + a.half;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float wl = weights[w][lo], wh = weights[w][hi];
          factors[buffer][angle_t[i]][w].set(lo, wl * c, -wh * s);
          factors[buffer][angle_t[i]][w].set(hi, wh * c, wl * s);
        }
      }
    }
    if (threadIdx.x < kQkTile) slots[buffer][threadIdx.x] = slot;
    at += gridDim.x;
    const int next_here = at < a.tiles ? a.shortest + (at < a.longer) : 0;
    const int next0 = next_here ? at * a.shortest + (at < a.longer ? at : a.longer) : 0;
    ask(next0, next_here);
    __syncthreads();
    for (int pass = blockIdx.y; pass < passes; pass += gridDim.y) {
      // The next step's values are on their way while this one's are worked on.
      uint4 next_raw[kQkTile] = {};
      int next_kind, next_off;
      const bool last = pass + int(gridDim.y) >= passes;
      row_of(last ? int(blockIdx.y) : pass + int(gridDim.y), next_kind, next_off);
      load(last ? next0 : token0, last ? next_here : here, next_kind, next_off, next_raw);
      // Every thread stays for the shuffles; a head behind the last one is not stored.
      const bool works = __any_sync(0xffffffffu, kind < 2), normed = (kind == 1 ? a.weight[1] : a.weight[0]) != nullptr;
      const bool slotted = a.slots && kind != 0;
      const int64_t stride = kind == 0 ? a.out_stride[0] : kind == 1 ? a.out_stride[1] : a.out_stride[2];
      T* to = static_cast<T*>(kind == 0 ? a.out[0] : kind == 1 ? a.out[1] : a.out[2]) + off;
      if (!slotted) to += token0 * stride;
#pragma unroll
      for (int t = 0; t < kQkTile; ++t) {
        if (t >= here) break;
        uint4 result = raw[t];
        if (works) {
          const QkFactors<D>& f = factors[buffer][t][kind == 1];
          uint64_t x[4], p[4];
          unpack8<T>(raw[t], x);
          uint64_t sum2 = fma2(x[1], x[1], fma2(x[0], x[0], 0));
          sum2 = add2(sum2, fma2(x[3], x[3], fma2(x[2], x[2], 0)));
          float sum, high;
          unpair(sum2, sum, high);
          sum += high;
#pragma unroll
          for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          const float r = normed ? rsqrtf(fmaf(sum, 1.f / D, a.eps)) : 1.f;
          if (a.adjacent) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              unpair(x[e], lo, hi);
              p[e] = pair_of(hi, lo);
            }
          } else {
            uint4 other;
            other.x = __shfl_sync(0xffffffffu, raw[t].x, partner);
            other.y = __shfl_sync(0xffffffffu, raw[t].y, partner);
            other.z = __shfl_sync(0xffffffffu, raw[t].z, partner);
            other.w = __shfl_sync(0xffffffffu, raw[t].w, partner);
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
          if (kind < 2) result = pack8<T>(y);
        }
        if (slotted) {
          const int64_t row = slots[buffer][t];
          if (kind < 3 && row >= 0 && row < a.n_slots) *reinterpret_cast<uint4*>(to + row * stride) = result;
        } else {
          if (kind < 3) *reinterpret_cast<uint4*>(to) = result;
          to += stride;
        }
      }
#pragma unroll
      for (int t = 0; t < kQkTile; ++t) raw[t] = next_raw[t];
      kind = next_kind;
      off = next_off;
    }
    token0 = next0;
    here = next_here;
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
  // Tiles of up to kQkTile tokens where every block gets a step of one; the passes over a token's heads go to as many blocks as it takes to
  // give each multiprocessor's blocks two tiles (the angles are made once more in each). Tiles as even as they come: all blocks end together.
  const int per_pass = kQkThreads / (dim / 8), passes = (a.rows + per_pass - 1) / per_pass, room = kQkBlocks * sm_count();
  const int longest = (tokens + kQkTile - 1LL) / kQkTile * passes >= room ? kQkTile : 1;
  const int least = int((tokens + longest - 1LL) / longest);
  int share = 1;
  while (share < passes && int64_t(least) * share < 2 * room) share = 2 * share < passes ? 2 * share : passes;
  const int across = room / share > 0 ? room / share : 1, grid_x = least < across ? least : across;
  const int64_t even = (least + grid_x - 1LL) / grid_x * grid_x;  // as many for each block
  a.tiles = int(even < tokens ? even : tokens);
  a.shortest = tokens / a.tiles;
  a.longer = tokens % a.tiles;
  const dim3 grid{unsigned(grid_x), unsigned(share)};
  const cudaError_t e = in->dtype == FB_DT_BF16 ? launch_qk<__nv_bfloat16>(a, dim, grid, as_stream(stream))
                                                : launch_qk<__half>(a, dim, grid, as_stream(stream));
  const int32_t st = check_launch("qk_norm_rope");
  return st ? st : int32_t(e);
}

}  // extern "C"
