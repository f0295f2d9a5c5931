// What the kernels of the shared-prefix attention have in common: the call's parameters, the order of the
// streamed work, the layout of the partials, and small device helpers.
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace lkv {
namespace prefix {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRows = 16;       // rows of an mma.sync tile
constexpr int kMinStages = 2;   // stages of the stream that a warp takes at least
// A unit's start (its queries) and end (its partial) count as this many stages more on the line, or the
// warps that get many short lists would set the time.
constexpr int kUnitStages = 3;

// The streamed work (prefix.cu). A unit is one tile of kRows query rows of one KV head against one list
// of tokens: first the prefix's units (head, row tile of the whole batch), where the prefix is streamed,
// then the sequences' own (sequence, head, row tile). A unit has a stage per 2^stage_shift tokens. All
// units in this order are one line, of which every warp takes an equal piece; a unit is as long on it as
// its stages and kUnitStages, an empty list's has no length.
struct Params {
  const __nv_bfloat16* q;  // [batch, tokens, hq, d], element strides, channels contiguous
  int64_t q_sb, q_st, q_sh;
  const void* pages;  // [n_pages, h, 2, bs, d]
  const float* scales;
  int n_pages, page_shift;
  int batch, tokens, h, group;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* lens;
  const int32_t* prefix_table;
  int prefix_cols;
  int prefix_len;
  float scale_log2;  // the softmax scale times log2(e): scores live in the log2 domain
  int rows;          // batch * tokens * group; row (b * tokens + t) * group + g
  // Tiled prefix (prefix_tile.cu): partials per (split, KV head, row).
  int n_splits;  // 0: no prefix, or a streamed one
  float* tile_o;    // [n_splits][h][rows][d], not yet divided by the sum
  float2* tile_ml;  // [n_splits][h][rows]: (reference in the log2 domain, sum)
  // Streamed work: a partial per (warp, unit) that meet, in slot warp + unit; where one unit fills the four
  // warps of a CTA, one partial for all of them, in its first warp's slot.
  int stage_shift;       // log2 of the tokens per stage
  int prefix_stages;     // stages of a streamed prefix (0: tiled, or none)
  int prefix_row_tiles;  // row tiles of the whole batch, of a streamed prefix
  int own_row_tiles;     // row tiles of a sequence's tokens * group rows
  int n_warps;           // 0: nothing is streamed
  int slot_rows;         // rows a slot holds
  float* slot_o;         // [slots][slot_rows][d]
  float2* slot_ml;       // [slots][slot_rows]
  void* out;             // [batch, tokens, hq, d]
  int out_f32;
  float* lse;            // [batch, tokens, hq]
  int tile_first;        // the stream's launch is behind the tiled prefix's
  // Test hooks of the tiles' waits (lkv_debug_set): how long one may last, and which arrival is withheld (0: none).
  uint64_t max_wait_ns;
  int stall;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x 2^e, e <= 0, also where 2^e alone is too small for a float32 (two references as far apart as value scales may be).
__device__ __forceinline__ float times_ex2(float x, float e) {
  if (e >= -120.0f || e == -INFINITY) return x * ex2(e);
  const float half = ex2(0.5f * e);
  return x * half * half;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
// A weight of bf16 pages in two bf16 terms: its upper half, and the rest and 2^-20 of it more, so that a weight's
// second term is never zero either (0 x infinity would make a NaN of an infinite value). Less than 2^-7 of the
// weight is left to the second term, whose rounding loses 2^-8 of that. Here for two weights at a time.
constexpr float kAndMore = 1.0f + 1.0f / 1048576.0f;
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
__device__ __forceinline__ float rest_of(float x) { return fmaf(x, kAndMore, -__uint_as_float(__float_as_uint(x) & 0xffff0000u)); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 b = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Four int8 codes as f16, exactly: byte b with its sign bit turned is u = code + 128, and 0x6400 | u is
// 1024 + u. `u`: four such bytes.
__device__ __forceinline__ uint2 biased_to_f16(uint32_t u) {
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
__device__ __forceinline__ uint2 codes_to_f16(uint32_t w) { return biased_to_f16(w ^ 0x80808080u); }

// For queries against int8 pages: the power of two 2^-e that brings a row's largest magnitude (its bf16
// bits) to [1, 2), or below 2^16 where that is above 2^113, and 2^e, which its scores have to be multiplied
// with. Both are normal numbers, times a power of two of the factors beside them too; an infinity or a NaN is
// what it is at any scale.
__device__ __forceinline__ float2 row_scales(uint32_t top_bits) {
  int e = (int)(top_bits >> 7) - 127;
  e = e > 112 ? 112 : e < -126 ? -126 : e;
  return make_float2(__int_as_float((127 - e) << 23), __int_as_float((127 + e) << 23));
}

// int8 pages: codes of values are exact in f16, and a weight is rounded to f16 once, as the product with its
// token's value scale: w = 2^(s - m) x scale x 2^-kScaleShift, s the score and m the row's reference. With
// scale < 2^E, m >= max(s + E) - kScaleShift - 7 over the tokens that the row sees makes w < 2^7 when m is set
// (half that for the token that set it, at least) and w < 2^15 until m is set again, and f16's last bit, 2^-24,
// is 2^-30 of the largest w: a token keeps 11 bits however its scale and weight make the product up, and none
// counts by a scale without its weight. The sum of the weights is float32, of 2^(s - m), whose range the shift
// lets scales from 2^-64 (smaller ones count as that, and lose bits below 2^-90) to float32's end share. o and
// the weights' sum l are an ordinary partial as (m + kScaleShift, l x 2^-kScaleShift, o).
constexpr float kScaleShift = 16.0f, kScaleDown = 1.0f / 65536.0f;
__device__ __forceinline__ float weight_room(float scale) {  // E - kScaleShift - 7; a scale that is not finite claims nothing
  const int bits = (__float_as_int(scale) >> 23) & 0xff;
  return (float)(bits == 0xff ? -64 : max(bits - 126, -64)) - (kScaleShift + 7.0f);
}

// Stages of sequence b's own tokens (lens may lie outside [0, the table's reach]).
__device__ __forceinline__ int own_len(const Params& p, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)p.table_cols << p.page_shift);
}
__device__ __forceinline__ int stages_of(const Params& p, int len) { return (own_len(p, len) + (1 << p.stage_shift) - 1) >> p.stage_shift; }
// a / b for 0 <= a, 0 < b (the line is rarely longer than 2^32 stages).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int length_of(int stages) { return stages > 0 ? stages + kUnitStages : 0; }

// Dynamic shared memory above 48 KB, asked for once per kernel and device (`done`: a bit per device).
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

// prefix_tile.cu: the prefix's partials for many rows, and how many splits of the prefix they take.
int tile_splits(int rows, int h, int64_t prefix_len);
int run_tiles(Params p, int d, bool int8, cudaStream_t st);

}  // namespace prefix
}  // namespace lkv
