// What the kernels of the paged cache have in common: the quantisation of a row, divisions by launch constants,
// and the checks of a cache's geometry.
#pragma once

#include <float.h>

#include "common.cuh"

namespace lkv {
namespace paged {

constexpr float kMaxScale = 0x1.020406p+121f;  // the largest whose 127-fold is finite

// Division by a number that is known when the kernel is launched: n / d for n < 2^31 (d < 2^31) as the high
// half of a product and a shift, with m = floor(2^32 (2^s - d) / d) + 1 and s the least for which 2^s >= d.
struct Divisor {
  uint32_t d, m, s;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};
inline Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

// The scale of a row whose largest magnitude has these bits.
__device__ __forceinline__ float scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fminf(fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), FLT_MIN), kMaxScale);
}

// A lane's codes (4 to a word) of a row with scale s; a NaN scale has codes 0.
template <int C>
__device__ __forceinline__ void quantise(const float* x, float s, uint32_t (&w)[C / 4]) {
  constexpr float kWhole = 12582912.0f;  // 1.5 x 2^23: a sum with it has the whole number in its low bits
  float inv;  // good to a few ulp, which the remainder makes up for
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float half = 0.5f * s;
  float k[C], far = 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    k[i] = fmaf(x[i], inv, kWhole);
    far = fmaxf(far, fabsf(fmaf(kWhole - k[i], s, x[i])));
  }
  if (!(far < half)) {  // next to never, or s is a NaN
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const float r = fmaf(kWhole - k[i], s, x[i]);
      // A remainder of exactly half a step belongs to the even neighbour.
      const bool odd = (__float_as_uint(k[i]) & 1u) != 0;
      if (r > half || (r == half && odd)) k[i] += 1.0f;
      else if (r < -half || (r == -half && odd)) k[i] -= 1.0f;
      if (isnan(s)) k[i] = kWhole;
    }
  }
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const uint32_t lo = __byte_perm(__float_as_uint(k[4 * i]), __float_as_uint(k[4 * i + 1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(k[4 * i + 2]), __float_as_uint(k[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(lo, hi, 0x5410);
  }
}

inline int check_cache(const char* who, int kind, int dtype, int h, int bs, int d, int64_t n_pages, const void* pages, const void* scales) {
  if (!dtype_ok(dtype)) return fail(LKV_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (kind != LKV_CACHE_MODEL && kind != LKV_CACHE_INT8) return fail(LKV_ERR_ARG, "%s: bad cache kind %d", who, kind);
  if (d != 64 && d != 128) return fail(LKV_ERR_ARG, "%s: head_dim %d (64 or 128)", who, d);
  if (bs != 16 && bs != 32 && bs != 64 && bs != 128) return fail(LKV_ERR_ARG, "%s: pages of %d tokens (16, 32, 64 or 128)", who, bs);
  if (h < 1 || n_pages < 0 || n_pages > INT32_MAX) return fail(LKV_ERR_ARG, "%s: bad shape (h %d, pages %lld)", who, h, (long long)n_pages);
  if (pages == nullptr || (kind == LKV_CACHE_INT8 && scales == nullptr)) return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(pages, 16) || !aligned(scales, 4)) return fail(LKV_ERR_PTR, "%s: pages must be 16-byte aligned", who);
  return LKV_OK;
}

inline int shift_of(int bs) { return bs == 16 ? 4 : bs == 32 ? 5 : bs == 64 ? 6 : 7; }

}  // namespace paged
}  // namespace lkv
