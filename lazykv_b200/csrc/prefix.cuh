// What the kernels of the shared-prefix attention have in common: the call's parameters, the layout of
// the prefix's partials, and small device helpers.
#pragma once

#include "common.cuh"

namespace lkv {
namespace prefix {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
  // Partials of the prefix, per (split, KV head, row): row r = (b * tokens + t) * group + g.
  int rows;        // batch * tokens * group
  int n_splits;    // 0: no prefix
  float* part_o;   // [n_splits][h][rows][d], not yet divided by the sum
  float2* part_ml; // [n_splits][h][rows]: (running maximum in the log2 domain, sum)
  void* out;       // [batch, tokens, hq, d]
  int out_f32;
  float* lse;      // [batch, tokens, hq]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Two int8 codes as bf16, exactly: bytes 0 and 2 of `w` (the others are ignored). With c = l - 128 f,
// l the low seven bits and f the sign bit, 0x4300 | l is 128 + l and 0x4300 | (f << 7) is 128 + 128 f.
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t w) {
  const uint32_t a = (w & 0x007f007fu) | 0x43004300u, s = (w & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&x);
}

// The page of token pos of a page list, or -1 where it has none.
__device__ __forceinline__ int page_at(const int32_t* table, int cols, int n_pages, int pos, int shift) {
  const int blk = pos >> shift;
  if (blk >= cols) return -1;
  const int id = table[blk];
  return id < n_pages ? id : -1;
}

// prefix_tile.cu: the prefix's partials for many rows, and how many splits of the prefix they take.
int tile_splits(int rows, int h, int64_t prefix_len);
int run_tiles(const Params& p, int d, bool int8, cudaStream_t st);

}  // namespace prefix
}  // namespace lkv
