// What the attention kernels share: tcgen05 and TMA wrappers, bounded waits, exponentials to base two, tensor maps.
#pragma once

#include "common.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace fb {

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two floats to a pair of T, the first in the low half; one rounding each.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  else
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  return r;
}

// ------------------------------------------------------------------------------ a row's scores, 32 at a time
// (NaN wins over numbers)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Weights are 2^kLift times the formula's (their sum too, so it falls out): fp16 numbers end at 2^-24, and many keys whose weights are below
// that, one by one nothing, may be a good part of a row in sum. 2^7 and the 2^8 that scores may rise above the maximum in use are 2^15.
template <class T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
// The larger of m and 32 scores.
__device__ __forceinline__ float scores_max(const float (&s)[32], float m) {
  float a = max3(m, s[0], s[1]), b = max3(s[2], s[3], s[4]), c = max3(s[5], s[6], s[7]);
#pragma unroll
  for (int i = 8; i < 32; i += 6) {
    a = max3(a, s[i], s[i + 1]);
    b = max3(b, s[i + 2], s[i + 3]);
    c = max3(c, s[i + 4], s[i + 5]);
  }
  return max3(a, b, c);
}
// 2^x of a pair on the multiply-add pipe: x = n + f with n whole and |f| <= 1/2 (adding 1.5 * 2^23 rounds to whole numbers and leaves
// n in the low bits), a polynomial of degree four for 2^f (minimax by Remez exchange, relative error 2.7e-6), n into the exponent.
// Below -126 it stays at 2^-126, so not for scores that are masked (and a score of minus infinity keeps that weight). NaN does not stay NaN: the row's maximum has to show it.
__device__ __forceinline__ void exp2_poly(uint64_t x2, float& x, float& y) {
  float a, b;
  unpair(x2, a, b);
  a = fmaxf(a, -126.f);
  b = fmaxf(b, -126.f);
  x2 = pair_of(a, b);
  constexpr float kRound = 12582912.f;
  const uint64_t t = add2(x2, pair_of(kRound, kRound));
  const uint64_t f = fma2(add2(t, pair_of(-kRound, -kRound)), pair_of(-1.f, -1.f), x2);
  uint64_t p = fma2(f, pair_of(0.009570102207362652f, 0.009570102207362652f), pair_of(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, pair_of(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
  float n0, n1;
  unpair(t, n0, n1);
  unpair(p, a, b);
  x = __uint_as_float(__float_as_uint(a) + (__float_as_uint(n0) << 23));
  y = __uint_as_float(__float_as_uint(b) + (__float_as_uint(n1) << 23));
}
// 32 weights 2^(scale s - base) as pairs of T and, before the rounding to it, added to `sum` (a pair of partial sums). The products take weights
// of v's type: half a step of each, which costs an output of values with mean zero about as much as its own rounding does (bf16, rms against
// 64 bits: 0.0016 with weights in 32 bits, 0.0020 for 8192 tokens). MIXED: two of sixteen pairs by exp2_poly, which takes work off the exponential
// unit (eight cycles per warp and instruction, 2048 of some 2600 cycles that two softmax warps of a scheduler have for a block of keys)
// at nine instructions a pair: 8192 tokens 624 us with none, 616 with two, 619 with four, 653 with six.
template <class T, bool MIXED>
__device__ __forceinline__ void scores_exp(const float (&s)[32], uint64_t scale, uint64_t minus_base, uint32_t (&p)[16], uint64_t (&sum)[2]) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    float x, y;
    const uint64_t x2 = fma2(pair_of(s[2 * c], s[2 * c + 1]), scale, minus_base);
    if (MIXED && c % 8 == 4) {
      exp2_poly(x2, x, y);
    } else {
      unpair(x2, x, y);
      x = exp2_approx(x);
      y = exp2_approx(y);
    }
    sum[c & 1] = add2(sum[c & 1], pair_of(x, y));
    p[c] = pack2<T>(x, y);
  }
}
__device__ __forceinline__ float pairs_sum(const uint64_t (&sum)[2]) {
  float a, b;
  unpair(add2(sum[0], sum[1]), a, b);
  return a + b;
}

// Moves a warpgroup's registers per thread up or down; the shares have to add up to what the block was launched with.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ------------------------------------------------------------------------------ copies and products
// Brings a tensor map (a kernel parameter) to where copies look for it.
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                   dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared-memory operand descriptors (128-byte swizzle, 8-row groups 1024 bytes apart, descriptor version 1) are given by their low
// words: address / 16, and in the high half `lead`: for a tile whose rows run along K (Q, K) not used (1); for V, whose rows run along
// N, the distance of its two 64-value parts / 16. The lane that issues steps through a tile with 32-bit adds, everything else is a
// constant: an instruction whose operands have to be put together first took 125 cycles beside two busy softmax warps, 1000 for the
// eight of a tile, against the 528 that the tensor core works on them.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t umma_desc_lo(uint32_t addr, uint32_t lead) { return ((addr & 0x3FFFFu) >> 4) | (lead << 16); }
// D[tmem] (+)= A[smem] B[smem] and A[tmem] B[smem], 16 of K.
template <uint32_t IDESC>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "n"(IDESC), "r"(uint32_t(accumulate)), "n"(kDescHi)
      : "memory");
}
template <uint32_t IDESC>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "n"(IDESC), "r"(uint32_t(accumulate)), "n"(kDescHi)
      : "memory");
}
// 32 columns of the warp's 32 lanes; the values are there after tmem_ld_wait and tmem_landed.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&f)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
        "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]),
        "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]),
        "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// No instruction: uses of the values stay behind the wait.
__device__ __forceinline__ void tmem_landed(float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(f[i]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Bounded wait. A wait that ran out is recorded, and every later one ends at once.
__device__ __forceinline__ bool bounded_wait(int* aborted, uint32_t* status, uint64_t* bar, uint32_t parity) {
  // (a plain probe first: a try that may suspend takes some 200 cycles longer even when the phase is complete)
  if (mbar_test_wait(bar, parity)) return true;
  for (uint32_t i = 0; i < (1u << 21); ++i) {
    if (mbar_try_wait_hint(bar, parity)) return true;
    if ((i & 31u) == 0u && *static_cast<volatile int*>(aborted)) return false;
  }
  *static_cast<volatile int*>(aborted) = 1;
  if (status) atomicMax(status, uint32_t(FB_STATUS_PIPELINE_TIMEOUT));
  return false;
}

// For a single thread that issues products: it polls, since waking up from a try takes longer than a product's share of the time.
__device__ __forceinline__ bool bounded_spin(int* aborted, uint32_t* status, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 26); ++i) {
    if (mbar_test_wait(bar, parity)) return true;
    if ((i & 1023u) == 1023u && *static_cast<volatile int*>(aborted)) return false;
  }
  *static_cast<volatile int*>(aborted) = 1;
  if (status) atomicMax(status, uint32_t(FB_STATUS_PIPELINE_TIMEOUT));
  return false;
}
// bounded_wait for a whole warp: one answer for all lanes. What stands behind a wait (barriers, tensor memory, elections) needs the
// warp converged, and lanes that left a polling loop one by one are not.
__device__ __forceinline__ bool bounded_wait_warp(int* aborted, uint32_t* status, uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  const bool ok = __all_sync(0xffffffffu, bounded_wait(aborted, status, bar, parity));
  __syncwarp();
  return ok;
}
// A named barrier of whole warps, each converged first.
__device__ __forceinline__ void warps_sync(int id, int threads) {
  __syncwarp();
  named_bar_sync(id, threads);
}

// ------------------------------------------------------------------------------ host: tensor maps
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

}  // namespace fb
