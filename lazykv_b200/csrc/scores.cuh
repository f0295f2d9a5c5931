// What chunk.cu and sums.cu do with scores alike: their cap, and codes of int8 pages as bf16 operands.
#pragma once

#include "prefix.cuh"
#include "tensor.cuh"

namespace lkv {

// c tanh(s / c) = c (1 - 2 / (1 + 2^(2 s log2(e) / c))): any size, two operations of the exponentials' unit.
__device__ __forceinline__ float capped(float x, float c) {  // x: 2 s log2(e) / c
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + prefix::ex2(x)));
  return fmaf(-2.0f * c, r, c);
}

// The same of two scores of up to the cap's size, without that unit, which the weights themselves keep busy: tanh(y) is
// y times a polynomial of degree 6 in y^2, fitted on [0, 1] to least relative error (5 x 10^-8; 2^-22.6 in
// float32). y: s / c; returns its squares (above 1: not good) and c tanh(y) + add.
__device__ __forceinline__ uint64_t capped2(uint64_t y, float c, uint64_t add, uint64_t* square) {
  using namespace tc;
  constexpr float k[7] = {0.9999999403953552f, -0.33332839608192444f, 0.13325203955173492f, -0.05345702916383743f, 0.020289981737732887f, -0.006203379016369581f, 0.0010410224786028266f};
  const uint64_t u = mul2(y, y);
  uint64_t t = pair(k[6], k[6]);
#pragma unroll
  for (int i = 5; i >= 0; --i) t = fma2(t, u, pair(k[i], k[i]));
  *square = u;
  return fma2(mul2(y, pair(c, c)), t, add);
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
