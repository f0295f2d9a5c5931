// What chunk.cu and sums.cu do with scores alike: their cap, and codes of int8 pages as bf16 operands.
#pragma once

#include <float.h>
#include <math.h>

#include "prefix.cuh"
#include "tensor.cuh"

namespace lkv {

// Do a softmax scale and a cap (0: none) and what the kernels make of them stay within float32? Beyond it 0 times infinity
// would be a score, and a quotient below the normal numbers would be short of bits.
inline bool scores_fit(float scale, float cap) {
  constexpr double kTwoLog2e = 2.0 * 1.4426950408889634;
  if (!(fabsf(scale) <= FLT_MAX) || !(cap >= 0.0f)) return false;
  if (cap == 0.0f) return fabs((double)scale) * kTwoLog2e <= 2.0 * (double)FLT_MAX;
  const double by = fabs((double)scale) / (double)cap;
  return (double)cap * kTwoLog2e <= (double)FLT_MAX && by * kTwoLog2e <= (double)FLT_MAX && (scale == 0.0f || by >= (double)FLT_MIN);
}

// c tanh(s / c) = c (1 - 2 / (1 + 2^(2 s log2(e) / c))): any size, two operations of the exponentials' unit.
__device__ __forceinline__ float capped(float x, float c) {  // x: 2 s log2(e) / c
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + prefix::ex2(x)));
  return fmaf(-2.0f * c, r, c);
}

// The same of N pairs of scores of up to the cap's size, without that unit, which the weights themselves keep busy: tanh(y) is
// y times a polynomial of degree 6 in y^2, fitted on [0, 1] to least relative error (5 x 10^-8; 2^-22.6 in
// float32). y: s / c; replaced by c tanh(y) + add, and `most` by the largest square where that is larger (above 1: not
// good). Step by step for all pairs: one after the other they would wait for their own results.
template <int N>
__device__ __forceinline__ void capped2(uint64_t (&y)[N], float c, const uint64_t (&add)[N], float& most) {
  using namespace tc;
  constexpr float k[7] = {0.9999999403953552f, -0.33332839608192444f, 0.13325203955173492f, -0.05345702916383743f, 0.020289981737732887f, -0.006203379016369581f, 0.0010410224786028266f};
  uint64_t u[N], t[N];
#pragma unroll
  for (int n = 0; n < N; ++n) u[n] = mul2(y[n], y[n]);
#pragma unroll
  for (int n = 0; n < N; ++n) most = fmaxf(fmaxf(most, first_of(u[n])), second_of(u[n]));
#pragma unroll
  for (int n = 0; n < N; ++n) t[n] = fma2(pair(k[6], k[6]), u[n], pair(k[5], k[5]));
#pragma unroll
  for (int i = 4; i >= 0; --i) {
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = fma2(t[n], u[n], pair(k[i], k[i]));
  }
#pragma unroll
  for (int n = 0; n < N; ++n) y[n] = mul2(y[n], pair(c, c));
#pragma unroll
  for (int n = 0; n < N; ++n) y[n] = fma2(y[n], t[n], add[n]);
}

#define LKV_R16(v, i) LKV_R8(v, i), LKV_R8(v, i + 8)
#define LKV_R32(v, i) LKV_R16(v, i), LKV_R16(v, i + 16)

// N columns of a thread's own lane of tensor memory (32 rows to a warp).
template <int N>
struct Lane {
  uint32_t v[N];
};
__device__ __forceinline__ void ld(Lane<32>& f, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : LKV_R32(f.v, 0)
      : "r"(addr));
}
__device__ __forceinline__ void ld(Lane<16>& f, uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : LKV_R16(f.v, 0)
               : "r"(addr));
}
template <int N>
__device__ __forceinline__ void ld_wait(Lane<N>& f) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(f.v[i]));
}

// Four int8 codes as bf16, exactly: 0x4300 | b is 128 + b for b < 128, and 0x4380 is 256.
__device__ __forceinline__ uint2 codes_to_bf16(uint32_t w) {
  const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
  auto code = [](uint32_t x) {
    const uint32_t hi = x & 0xff7fff7fu, lo = x & 0xff80ff80u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&hi), *reinterpret_cast<const __nv_bfloat162*>(&lo));
    return *reinterpret_cast<const uint32_t*>(&d);
  };
  return make_uint2(code(a), code(b));
}

}  // namespace lkv
