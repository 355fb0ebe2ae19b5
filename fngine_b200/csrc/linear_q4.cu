// Projections with 4-bit weights and group scales at decode width (T <= 16).
//
//   acc[t][r] = sum over groups g of  s[r][g] * sum_{i in g} (c[r][i] - z[r][g]) * x[t][i],   then the epilogue.
//
// The code bits are the tensor core's operand as they stand: bits 0-7 of a bf16 number whose other bits are zero count in steps of
// 2^-133 (the subnormal numbers and the first normal ones have the same spacing), so a code in bits 0-3 is c 2^-133 and one in bits
// 4-7 is 16 c 2^-133, both exact, and eight codes cost one shift and four ANDs. (As whole bf16 numbers, by an exponent under the bits
// and a subtraction of 128 + z, they cost eleven instructions, and their issue bound the kernel: 110 us for 248320 x 2560 at 16 tokens.)
// The activations bring the scale back: they are multiplied by 2^64, those of the codes in bits 4-7 by 2^60, exactly; or by 1 and 1/16
// in a token that has one of 2^63 or more. Products are exact, the tensor core adds them in fp32 and keeps subnormal sums, so the smallest
// step of a sum is 2^-149 here and 2^-80 (2^-16 in such a token) in the activations' own scale: what is far below it is lost. What a zero
// point takes off, z sum(x) of a group, comes from sums of the activations that are made once, with the same smallest step:
//   acc += s (P - z X),   P = sum of c x 2^-69 over the group, X = sum of x 2^-69.
// (P and X of an infinite activation are infinite, or P is NaN: their difference is NaN for every weight of that token.)
// Nothing is rounded but sums.
//
// Bound by the weights' bytes at few tokens and instruction issue at sixteen: 248320 x 2560 in 69 us for one token (4.8 TB/s), 99 for
// sixteen. The weights are the only large operand, so the kernel is built around their stream. A warp takes 16 MT rows (the M
// side of mma.sync m16n8k16, the tokens are the N side) through K in steps of 128: its own ring of cp.async stages in
// shared memory, no barrier between warps. ldmatrix gives lane (g, t) of a quad eight consecutive codes of row g. The activations lie
// in shared memory in the order (0 4 1 5 2 6 3 7) that the masked codes come in. S warps share
// the K steps of a row tile and add their tiles in shared memory in warp order, so results do not depend on timing.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fb {
namespace {

constexpr int kQ4Warps = 16;
constexpr int kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4Step = 128;    // K values per step of a warp: 64 bytes of a row
constexpr int kQ4MaxTok = 16;
constexpr int kQ4SmemLimit = 226 * 1024;  // (beside the static part)

struct Q4Args {
  const __nv_bfloat16* x;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  void* out;
  const float* inj;
  const float* gate_logit;
  int n, k, tokens, kind, gate_stride;
  int scale_f16;   // 16-bit scales: fp16 instead of bf16
  int units;       // row tiles
  int split;       // warps per row tile
  int chunk;       // K steps whose activations are in shared memory at a time
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Code 0..15 as fp32, without the conversion unit.
__device__ __forceinline__ float code_to_float(uint32_t c) { return __uint_as_float(0x4b000000u | c) - 8388608.f; }

// Stages of a warp's ring. One more costs 16 or 32 KB of the activations' room.
template <int MT>
constexpr int kQ4Stages = MT == 1 ? 6 : 3;
template <int MT>
constexpr int kQ4RowPitch = 16 * MT + 4;  // floats between tokens of a partial tile: lanes of a fragment in 32 banks
template <int MT, int NT>
constexpr int q4_fixed_smem() {
  return kQ4Warps * (kQ4Stages<MT> * MT * 1024 + 8 * NT * kQ4RowPitch<MT> * 4);
}

template <int MT, int NT, int GROUP, bool SF32>
__global__ void __launch_bounds__(kQ4Threads, 1) q4_kernel(const Q4Args a) {
  constexpr int kStages = kQ4Stages<MT>;
  constexpr int kGroups = kQ4Step / GROUP;                           // groups per step
  constexpr int kScaleWords = SF32 ? kGroups : (kGroups + 1) / 2;    // 32-bit words of a row's scales per step
  constexpr int kPitch = kQ4RowPitch<MT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t large_tokens;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) large_tokens = 0;
  uint8_t* ring = smem + warp * (kStages * MT * 1024);
  float* tile = reinterpret_cast<float*>(smem + kQ4Warps * kStages * MT * 1024) + warp * (8 * NT * kPitch);
  float* group_sums = reinterpret_cast<float*>(smem + q4_fixed_smem<MT, NT>());  // [groups of a chunk][8 NT]
  uint8_t* xs = reinterpret_cast<uint8_t*>(group_sums + a.chunk * (kGroups * 8 * NT));
  const int split = a.split, per_cta = kQ4Warps / split;
  const int wk = warp % split, wu = warp / split;
  const int ksteps = a.k / kQ4Step;
  const int half = a.n >> 1;
  const bool swiglu = a.kind == FB_EPI_SWIGLU;
  const int first = blockIdx.x * per_cta + wu, stride = gridDim.x * per_cta;
  const size_t row_bytes = size_t(a.k) >> 1;
  const int row_groups = a.k / GROUP;

  // Row r of a row tile; rows behind the last one repeat it and are not stored. SwiGlu: 16 gate rows, then their up rows.
  auto row_of = [&](int unit, int r) {
    if (swiglu) {
      const int j = unit * 16 + (r & 15);
      return (j < half ? j : half - 1) + (r >> 4) * half;
    }
    const int j = unit * (16 * MT) + r;
    return j < a.n ? j : a.n - 1;
  };

  // Cursor of the code copies: kStages - 1 steps ahead of the products.
  int pu = first, ps = wk;
  const uint8_t* src[2 * MT];
  auto seek = [&] {
    if (pu < a.units) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) src[i] = a.codes + size_t(row_of(pu, 8 * i + g)) * row_bytes + ps * 64 + t * 16;
    }
  };
  const uint32_t ring_addr = smem_u32(ring);
  // 16-byte chunk c of row r lies at r * 64 + (c ^ (r / 2 % 4)) * 16: eight rows of a chunk in eight bank groups.
  const uint32_t put0 = ring_addr + uint32_t(g * 64 + ((t ^ ((g >> 1) & 3)) << 4)), ring_end = put0 + kStages * MT * 1024;
  uint32_t put = put0;
  auto copy_step = [&] {
    if (pu < a.units) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        cp_async16(put + i * 512, src[i]);
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) src[i] += split * 64;
      ps += split;
      if (ps >= ksteps) {
        ps = wk;
        pu += stride;
        seek();
      }
    }
    cp_async_commit();
    put += MT * 1024;
    if (put == ring_end) put = put0;
  };

  // Scales and zero points of the step after the current one.
  uint32_t s_raw[2 * MT][kScaleWords], z_raw[2 * MT];
  int su = first, ss = wk;
  uint32_t s_at[2 * MT];  // group of the step in each row
  auto seek_scales = [&] {
    if (su < a.units) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) s_at[i] = uint32_t(row_of(su, 8 * i + g)) * uint32_t(row_groups) + uint32_t(ss * kGroups);
    }
  };
  auto load_scales = [&] {
    if (su >= a.units) return;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      if (SF32) {
        const float* p = static_cast<const float*>(a.scales) + s_at[i];
        if (kGroups == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          s_raw[i][0] = v.x, s_raw[i][1 % kScaleWords] = v.y, s_raw[i][2 % kScaleWords] = v.z, s_raw[i][3 % kScaleWords] = v.w;
        } else if (kGroups == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          s_raw[i][0] = v.x, s_raw[i][1 % kScaleWords] = v.y;
        } else {
          s_raw[i][0] = __float_as_uint(*p);
        }
      } else {
        const uint16_t* p = static_cast<const uint16_t*>(a.scales) + s_at[i];
        if (kGroups == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          s_raw[i][0] = v.x, s_raw[i][1 % kScaleWords] = v.y;
        } else if (kGroups == 2) {
          s_raw[i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
          s_raw[i][0] = *p;
        }
      }
      if (a.zeros) {
        const uint8_t* z = a.zeros + s_at[i];
        z_raw[i] = kGroups == 1 ? *z : kGroups == 2 ? *reinterpret_cast<const uint16_t*>(z) : *reinterpret_cast<const uint32_t*>(z);
      }
      s_at[i] += split * kGroups;
    }
    ss += split;
    if (ss >= ksteps) {
      ss = wk;
      su += stride;
      seek_scales();
    }
  };

  seek();
  seek_scales();
  pdl_wait_prior();
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) z_raw[i] = 0x08080808u;
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) copy_step();
  load_scales();

  const int x_pitch = a.chunk * (kQ4Step * 2) + 64;  // 64 modulo 128: two tokens' 64-byte blocks in different banks
  const uint32_t xs_addr = smem_u32(xs);
  uint32_t x_row[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {  // token columns behind the last one read its values and are not stored
    const int tok = nt * 8 + g;
    x_row[nt] = xs_addr + uint32_t((tok < a.tokens ? tok : a.tokens - 1) * x_pitch + t * 16);
  }
  // ldmatrix row addresses: lanes 0-7 rows 0-7 of a chunk, 8-15 rows 8-15, 16-31 the same of the next chunk.
  const int lr = (lane & 7) + ((lane >> 3) & 1) * 8, lc = lane >> 4;
  // Chunk pairs (0, 1) and (2, 3) of a row: where this lane's lies in a stage.
  const uint32_t get_x = uint32_t((lr >> 1) & 3), get0 = ring_addr + uint32_t(lr * 64), get_end = get0 + kStages * MT * 1024;
  const uint32_t chunk[2] = {(uint32_t(lc) ^ get_x) << 4, (uint32_t(2 + lc) ^ get_x) << 4};
  uint32_t get = get0;

  float acc[MT][NT][4];
  uint32_t large = 0;  // tokens whose activations are not multiplied by 2^64, and their sums smaller by it
  bool loaded = false;
  for (int base = blockIdx.x * per_cta; base < a.units; base += stride) {
    const int unit = base + wu;
    int step = unit < a.units ? wk : ksteps;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][nt][i] = 0.f;

    for (int c0 = 0; c0 < ksteps; c0 += a.chunk) {
      const int c1 = c0 + a.chunk < ksteps ? c0 + a.chunk : ksteps;
      if (!loaded || a.chunk < ksteps) {  // (block-uniform)
        __syncthreads();
        const int per_row = (c1 - c0) * (kQ4Step / 8);
        auto stage_x = [&] {
          // Four pieces of a thread on their way at a time where there are many (16 tokens of 6144 are 24 per thread: 2560 x 6144 in 23.6 us with
          // one at a time, 20.9 with four; at 2199 x 9984 and eleven tokens 27.9 and 24.8).
          constexpr int kAhead = NT == 2 ? 4 : 1;
          const int all = per_row * a.tokens;
          for (int i0 = threadIdx.x; i0 < all; i0 += kAhead * kQ4Threads) {
            uint4 raw[kAhead];
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
              const int i = i0 + p * kQ4Threads, tok = i / per_row, j = i - tok * per_row;
              if (i < all) raw[p] = *reinterpret_cast<const uint4*>(a.x + size_t(tok) * a.k + size_t(c0) * kQ4Step + j * 8);
            }
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
              const int i = i0 + p * kQ4Threads;
              if (i >= all) break;
              const int tok = i / per_row, j = i - tok * per_row;
              const bool plain = (large >> tok) & 1;
              const uint32_t up = plain ? 0x3f803f80u : 0x5f805f80u, up16 = plain ? 0x3d803d80u : 0x5d805d80u;  // 1, 2^64; 1/16, 2^60
              const uint4 v = raw[p];
              const uint32_t in[4] = {v.x, v.y, v.z, v.w};
              bool found = false;
              float sum = 0.f;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t lo = in[e] & 0x7fffu, hi = (in[e] >> 16) & 0x7fffu;
                found |= (lo >= 0x5f00u && lo < 0x7f80u) || (hi >= 0x5f00u && hi < 0x7f80u);  // 2^63 and more, and finite
                sum += __uint_as_float(in[e] << 16) * 0x1p-69f + __uint_as_float(in[e] & 0xffff0000u) * 0x1p-69f;
              }
              if (found) atomicOr(&large_tokens, 1u << tok);
#pragma unroll
              for (int m = GROUP / 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffu << (lane & 16), sum, m);  // (16 lanes have 128 values)
              if (j % (GROUP / 8) == 0) group_sums[j / (GROUP / 8) * (8 * NT) + tok] = plain ? sum * 0x1p-64f : sum;
              uint4 w;
              w.x = mul_bf16x2(__byte_perm(v.x, v.z, 0x5410), up);
              w.y = mul_bf16x2(__byte_perm(v.x, v.z, 0x7632), up16);
              w.z = mul_bf16x2(__byte_perm(v.y, v.w, 0x5410), up);
              w.w = mul_bf16x2(__byte_perm(v.y, v.w, 0x7632), up16);
              *reinterpret_cast<uint4*>(xs + tok * x_pitch + j * 16) = w;
            }
          }
          __syncthreads();
        };
        // A token that turns out to have large activations: its sums so far are made smaller, and everything is staged once more. (The code
        // for the second time in a copy of its own for up to eight tokens, 68 us for one token of 248320 x 2560 instead of 70; in a
        // loop for more, where the copy costs registers: 98 us instead of 111 for sixteen.)
        auto found_more = [&] {
          const uint32_t more = large_tokens & ~large;  // (the same for all)
          if (!more) return false;
          __syncthreads();
          large |= more;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if ((more >> (nt * 8 + 2 * t + (i & 1))) & 1) acc[m][nt][i] *= 0x1p-64f;
          return true;
        };
        if (NT == 1) {
          stage_x();
          if (found_more()) stage_x();
        } else {
          do stage_x();
          while (found_more());
        }
        loaded = true;
      }
      for (; step < c1; step += split) {
        uint32_t s_now[2 * MT][kScaleWords], z_now[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
#pragma unroll
          for (int j = 0; j < kScaleWords; ++j) s_now[i][j] = s_raw[i][j];
          z_now[i] = z_raw[i];
        }
        load_scales();
        cp_async_wait<kStages - 2>();
        __syncwarp();
        copy_step();  // into the stage that the step before has read
        const uint32_t stage = get;
        get += MT * 1024;
        if (get == get_end) get = get0;
        const uint32_t x_step = uint32_t((step - c0) * (kQ4Step * 2));
        float part[MT][NT][4];
#pragma unroll
        for (int b2 = 0; b2 < 2; ++b2) {
          uint32_t w[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) ldmatrix_x4(w[m], stage + chunk[b2] + m * 1024);
#pragma unroll
          for (int ci = 0; ci < 2; ++ci) {
            constexpr int kBlocks = GROUP / 32;  // blocks of 32 values per group
            const int b = 2 * b2 + ci, group = b / kBlocks;
            if (b % kBlocks == 0) {
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int i = 0; i < 4; ++i) part[m][nt][i] = 0.f;
            }
            uint4 xv[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(xv[nt].x), "=r"(xv[nt].y), "=r"(xv[nt].z), "=r"(xv[nt].w)
                           : "r"(x_row[nt] + x_step + b * 64)
                           : "memory");
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint32_t wa = w[m][2 * ci], wb = w[m][2 * ci + 1], va = wa >> 8, vb = wb >> 8;
              const uint32_t a0 = wa & 0x000f000fu, a1 = wb & 0x000f000fu, a2 = wa & 0x00f000f0u, a3 = wb & 0x00f000f0u;
              const uint32_t a4 = va & 0x000f000fu, a5 = vb & 0x000f000fu, a6 = va & 0x00f000f0u, a7 = vb & 0x00f000f0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_bf16(part[m][nt], a0, a1, a2, a3, xv[nt].x, xv[nt].y);
                mma_bf16(part[m][nt], a4, a5, a6, a7, xv[nt].z, xv[nt].w);
              }
            }
            if (b % kBlocks == kBlocks - 1) {
              float2 xsum[NT];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                xsum[nt] = *reinterpret_cast<const float2*>(group_sums + ((step - c0) * kGroups + group) * (8 * NT) + nt * 8 + 2 * t);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                float sc[2], z[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  if (SF32) {
                    sc[i] = __uint_as_float(s_now[2 * m + i][group]);
                  } else {
                    const uint32_t h = (s_now[2 * m + i][group / 2] >> (16 * (group % 2))) & 0xffffu;
                    sc[i] = a.scale_f16 ? __half2float(__ushort_as_half(uint16_t(h))) : __uint_as_float(h << 16);
                  }
                  z[i] = code_to_float((z_now[2 * m + i] >> (8 * group)) & 15u);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    float v = fmaf(-z[i >> 1], i & 1 ? xsum[nt].y : xsum[nt].x, part[m][nt][i]);
                    acc[m][nt][i] = fmaf(sc[i >> 1], v, acc[m][nt][i]);
                  }
              }
            }
          }
        }
      }
    }

    // The warps of a row tile meet in shared memory; their threads share the outputs.
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tile[(nt * 8 + 2 * t + (i & 1)) * kPitch + m * 16 + g + (i >> 1) * 8] =
              acc[m][nt][i] * 0x1p69f * ((large >> (nt * 8 + 2 * t + (i & 1))) & 1 ? 0x1p64f : 1.f);
    __syncwarp();
    if (split > 1) named_bar_sync(1 + wu, 32 * split);
    if (unit < a.units) {
      const float* tiles = tile - wk * (8 * NT * kPitch);
      // Four rows of a token per thread and step.
      const int quads = swiglu ? 4 : 4 * MT, shift = quads == 4 ? 2 : 3;
      const int row_end = swiglu ? half : a.n;
      for (int i = wk * 32 + lane; i < quads * a.tokens; i += 32 * split) {
        const int r = 4 * (i & (quads - 1)), tok = i >> shift, row = unit * (4 * quads) + r;
        if (row >= row_end) continue;
        const float* p = tiles + tok * kPitch + r;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < split; ++w) {
          const float4 f = *reinterpret_cast<const float4*>(p + w * (8 * NT * kPitch));
          v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
        if (swiglu) {
          float u[4] = {0.f, 0.f, 0.f, 0.f};
          for (int w = 0; w < split; ++w) {
            const float4 f = *reinterpret_cast<const float4*>(p + w * (8 * NT * kPitch) + 16);
            u[0] += f.x, u[1] += f.y, u[2] += f.z, u[3] += f.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = v[e] / (1.f + expf(-v[e])) * u[e];
        } else if (a.kind == FB_EPI_SHARED_SCALE) {
          const float gate = 1.f + expf(-a.gate_logit[size_t(tok) * a.gate_stride]);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] /= gate;
        }
        const int here = row_end - row < 4 ? row_end - row : 4;
        const size_t at = size_t(tok) * row_end + row;
        if (a.kind == FB_EPI_GR_WRITE) {  // four residual streams
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            float* X = static_cast<float*>(a.out) + (size_t(tok) * 4 + s) * a.n + row;
            const float inj = a.inj[tok * 4 + s];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < here) X[e] += inj * v[e];
          }
        } else if (a.kind == FB_EPI_STORE_BF16 || swiglu) {
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + at;
          if (here == 4 && !(reinterpret_cast<uintptr_t>(out) & 7)) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < here) out[e] = __float2bfloat16_rn(v[e]);
          }
        } else {
          float* out = static_cast<float*>(a.out) + at;
          if (here == 4 && !(reinterpret_cast<uintptr_t>(out) & 15)) {
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < here) out[e] = v[e];
          }
        }
      }
    }
    __syncwarp();
    if (split > 1) named_bar_sync(1 + wu, 32 * split);
  }
  cp_async_wait<0>();
}

template <int MT, int NT, int GROUP, bool SF32>
cudaError_t launch_q4(const Q4Args& a, int grid, size_t smem, cudaStream_t stream) {
  static PerDeviceOnce once;
  const cudaError_t e = per_device_once(once, [] { return opt_in_smem(q4_kernel<MT, NT, GROUP, SF32>, kQ4SmemLimit); });
  if (e != cudaSuccess) return e;
  return launch_pdl(q4_kernel<MT, NT, GROUP, SF32>, dim3(unsigned(grid)), dim3(kQ4Threads), smem, stream, a);
}
template <int MT, int NT>
cudaError_t launch_q4_group(const Q4Args& a, int group, bool f32, int grid, size_t smem, cudaStream_t s) {
  if (group == 32) return f32 ? launch_q4<MT, NT, 32, true>(a, grid, smem, s) : launch_q4<MT, NT, 32, false>(a, grid, smem, s);
  if (group == 64) return f32 ? launch_q4<MT, NT, 64, true>(a, grid, smem, s) : launch_q4<MT, NT, 64, false>(a, grid, smem, s);
  return f32 ? launch_q4<MT, NT, 128, true>(a, grid, smem, s) : launch_q4<MT, NT, 128, false>(a, grid, smem, s);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

int32_t fb_linear_q4_decode(const void* x_bf16, int32_t tokens, const fb_q4_weight* weight,
                            const fb_linear_epilogue* epilogue, void* stream) {
  if (!x_bf16 || !weight || !weight->codes || !weight->scales || !epilogue || !epilogue->out)
    return invalid("linear_q4_decode: null argument");
  if (tokens <= 0 || tokens > kQ4MaxTok) return invalid("linear_q4_decode: tokens must be 1..16");
  const int n = weight->n, k = weight->k, group = weight->group, kind = epilogue->kind;
  if (n <= 0 || k <= 0 || k % kQ4Step) return invalid("linear_q4_decode: unsupported shape (k %% 128)");
  if (group != 32 && group != 64 && group != 128) return invalid("linear_q4_decode: groups of 32, 64 or 128 values");
  if (int64_t(n) * (k / group) > INT32_MAX) return invalid("linear_q4_decode: more than 2^31 - 1 groups");
  if (weight->scales_dtype != FB_DT_F32 && weight->scales_dtype != FB_DT_BF16 && weight->scales_dtype != FB_DT_F16)
    return invalid("linear_q4_decode: scales are fp32, bf16 or fp16");
  if (kind < FB_EPI_STORE_BF16 || kind > FB_EPI_SHARED_SCALE) return invalid("linear_q4_decode: unknown epilogue");
  if (kind == FB_EPI_GR_WRITE && !epilogue->inj) return invalid("linear_q4_decode: GrWrite needs inj fp32 [tokens][4]");
  if (kind == FB_EPI_SHARED_SCALE && !epilogue->gate_logit)
    return invalid("linear_q4_decode: SharedScale needs gate_logit");
  if (kind == FB_EPI_SWIGLU && n % 2) return invalid("linear_q4_decode: SwiGlu needs n %% 2 == 0");
  if ((reinterpret_cast<uintptr_t>(weight->codes) | reinterpret_cast<uintptr_t>(x_bf16) |
       reinterpret_cast<uintptr_t>(weight->scales) | reinterpret_cast<uintptr_t>(weight->zeros)) & 15)
    return invalid("linear_q4_decode: x, weight codes, scales and zeros must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(epilogue->out) & (kind == FB_EPI_STORE_BF16 || kind == FB_EPI_SWIGLU ? 1 : 3))
    return invalid("linear_q4_decode: out is not aligned to its elements");
  if ((reinterpret_cast<uintptr_t>(kind == FB_EPI_GR_WRITE ? epilogue->inj : nullptr) |
       reinterpret_cast<uintptr_t>(kind == FB_EPI_SHARED_SCALE ? epilogue->gate_logit : nullptr)) & 3)
    return invalid("linear_q4_decode: inj or gate_logit is not aligned to its elements");
  const size_t out_values = size_t(tokens) * size_t(n);
  const size_t out_bytes = kind == FB_EPI_GR_WRITE ? 16 * out_values : kind == FB_EPI_STORE_BF16 ? 2 * out_values
                           : kind == FB_EPI_SWIGLU ? out_values : 4 * out_values;
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(x_bf16), out0 = reinterpret_cast<uintptr_t>(epilogue->out);
  if (out0 < x0 + size_t(tokens) * size_t(k) * 2 && x0 < out0 + out_bytes)
    return invalid("linear_q4_decode: out lies in the memory of x");

  Q4Args a;
  a.x = static_cast<const __nv_bfloat16*>(x_bf16);
  a.codes = weight->codes;
  a.scales = weight->scales;
  a.zeros = weight->zeros;
  a.out = epilogue->out;
  a.inj = epilogue->inj;
  a.gate_logit = epilogue->gate_logit;
  a.n = n;
  a.k = k;
  a.tokens = tokens;
  a.kind = kind;
  a.gate_stride = epilogue->gate_stride;
  a.scale_f16 = weight->scales_dtype == FB_DT_F16;

  const int sms = sm_count(), ksteps = k / kQ4Step, nt = tokens > 8 ? 2 : 1;
  // Two row tiles of 16 per warp halve the reads of activations and the steps per weight (248320 x 2560, one token: 99 us by 16 rows, 67
  // by 32), where every warp has at least two such steps (2560 x 640: 4.1 us by 16, 5.0 by 32).
  const long long steps32 = (n + 31LL) / 32 * ksteps;
  const int mt = kind == FB_EPI_SWIGLU || nt == 2 || steps32 >= 2LL * kQ4Warps * sms ? 2 : 1;
  const long long units = kind == FB_EPI_SWIGLU ? (n / 2 + 15) / 16 : (n + 16 * mt - 1LL) / (16 * mt);
  // The number of warps per row tile that ends first, by the steps that the busiest warp takes.
  long long best = -1;
  for (int s = 1; s <= kQ4Warps && (s == 1 || s / 2 < ksteps); s *= 2) {
    const long long per_wave = (long long)sms * (kQ4Warps / s);
    const long long cost = (units + per_wave - 1) / per_wave * ((ksteps + s - 1) / s);
    if (s <= ksteps && (best < 0 || cost < best)) {
      best = cost;
      a.split = s;
    }
  }
  a.units = int(units);
  const long long ctas = (units + kQ4Warps / a.split - 1) / (kQ4Warps / a.split);
  const int grid = int(ctas < sms ? ctas : sms);
  const int fixed = mt == 1 ? (nt == 1 ? q4_fixed_smem<1, 1>() : q4_fixed_smem<1, 2>())
                            : (nt == 1 ? q4_fixed_smem<2, 1>() : q4_fixed_smem<2, 2>());
  // Per K step: a token's activations, and the sums of its groups for all token columns.
  const int per_step = tokens * kQ4Step * 2 + (kQ4Step / group) * 8 * nt * 4;
  a.chunk = (kQ4SmemLimit - fixed - tokens * 64) / per_step;
  if (a.chunk > ksteps) a.chunk = ksteps;
  const size_t smem = size_t(fixed) + size_t(tokens) * 64 + size_t(a.chunk) * per_step;
  const bool f32 = weight->scales_dtype == FB_DT_F32;
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = mt == 1 ? launch_q4_group<1, 1>(a, group, f32, grid, smem, s)
                        : nt == 1 ? launch_q4_group<2, 1>(a, group, f32, grid, smem, s)
                                  : launch_q4_group<2, 2>(a, group, f32, grid, smem, s);
  const int32_t st = check_launch("linear_q4_decode");
  return st ? st : int32_t(e);
}

}  // extern "C"
