// The paged cache: tokens written into pages (quantised on the way in) and read back.
//
// One page holds bs tokens of every KV head, keys then values, as the pairs of the tiered store do:
// pages [n_pages, h, 2, bs, d]. The elements are the model's type, or int8 codes with one float32
// scale per (token, head, key or value) row, scales [n_pages, h, 2, bs]. A sequence's token `pos` is
// row pos % bs of page table[b][pos / bs]. Unlike the sealed blocks' records (codec.cu), whose keys
// are quantised per channel over a whole block, a row's scale needs that row only, so a token is
// final as soon as it is written.
//
// The row's code: s = max(max_c |x_c| / 127, FLT_MIN) (at most what keeps 127 s finite), code_c = the whole
// number nearest to x_c / s (halfway: the even one), value code_c * s. The quotient is never rounded before
// the rounding to a whole number: k, x * (1 / s) rounded to one in a fused multiply-add, is within one of
// it, the remainder x - k s is exact in another, and where one reaches s / 2 (next to never) k is put
// right. A row that holds an infinity or a NaN has no scale: it gets s = NaN and codes 0 and reads back as
// NaN throughout.
//
// Every byte moves once. A thread carries 16 bytes of the model's type (8 channels of bf16, 4 of float32) of a
// token's key row and of its value row, so that a warp reads and writes whole runs; with 32 bytes a thread, two
// stores a sector each, a read wrote 4.8 TB/s. Reading, a thread carries several tokens, since its loads wait
// for the page's id and that for the table's row.
//
// Measured (8 heads, d 128, bf16 tokens, int8 pages): 12 x up to 16,000 tokens read back at 6.0 TB/s, 0.94 of a
// plain copy (989 MB, 163 us): memory bounds it. 65,536 tokens of a prompt written at 4.0 TB/s, 0.61 of a copy
// (407 MB, 103 us): quantising bounds it, 74% of the issue slots (model-type pages: 6.6 TB/s). A token of each of 64 sequences written and
// read back: 5.9 us, two launches of three dependent loads each.
#include <float.h>

#include "common.cuh"

namespace lkv {
namespace {

constexpr int kThreads = 256;
constexpr float kMaxScale = 0x1.020406p+121f;  // the largest whose 127-fold is finite

// Division by a number that is known when the kernel is launched: n / d for n < 2^31 (d < 2^31) as the high
// half of a product and a shift, with m = floor(2^32 (2^s - d) / d) + 1 and s the least for which 2^s >= d.
struct Divisor {
  uint32_t d, m, s;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};
Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

struct PagedParams {
  const void* keys;    // write: [b, t, h, d] with these element strides (channels contiguous)
  const void* values;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  void* pages;
  float* scales;
  int64_t n_pages;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* starts;
  const int32_t* lens;  // read: tokens a sequence has (null: as many as its table)
  uint32_t rows;  // batch * tokens * h
  Divisor tokens, h;
  int page_shift;
  void* out_k;  // read: contiguous [b, n, h, d]
  void* out_v;
};

// Channels per thread: 16 bytes of the model's type.
template <typename T>
constexpr int kCh = 16 / (int)sizeof(T);

// A thread's consecutive elements as float; VEC: 16-byte aligned. Plain loads: the read-only path may serve a
// line that the kernel before this one, still running when this one started, has written since.
template <typename T, bool VEC>
__device__ __forceinline__ void load(const T* p, float* x) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < kCh<T>; ++i) x[i] = to_f32<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The page of token `pos` of sequence b, or -1 where it has none (outside the table, a hole, a bad id).
__device__ __forceinline__ int64_t page_of(const PagedParams& p, uint32_t b, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t blk = pos >> p.page_shift;
  if (blk >= p.table_cols) return -1;
  const int64_t id = p.table[(int64_t)b * p.table_ld + blk];
  return id < p.n_pages ? id : -1;
}

// The largest magnitudes of a key row and a value row, C channels per lane of a group of L lanes, as float32
// bits: magnitudes compare as their bits, and infinities and NaN come out above FLT_MAX.
template <typename T, int L, int C>
__device__ __forceinline__ uint2 row_tops(const float* k, const float* v) {
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) a = max(a, __float_as_uint(k[i]) & 0x7fffffffu), b = max(b, __float_as_uint(v[i]) & 0x7fffffffu);
  if constexpr (sizeof(T) == 2) {  // two bf16 travel as one word
    uint32_t both = (a >> 16) | b;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
    return make_uint2(both << 16, both & 0xffff0000u);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o)), b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    return make_uint2(a, b);
  }
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

// Grid: rows of (sequence, token, head), D / kCh threads each.
template <typename T, int D, bool INT8, bool VEC>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(const PagedParams p) {
  constexpr int C = kCh<T>, L = D / C;
  pdl_wait();
  pdl_release();
  const uint32_t row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int c = (threadIdx.x % L) * C;
  const bool live = row < p.rows;
  const uint32_t bt = p.h.of(row), j = row - bt * p.h.d, b = p.tokens.of(bt), t = bt - b * p.tokens.d;
  int64_t page = -1, pos = 0;
  float k[C], v[C];
  if (live) {
    load<T, VEC>(static_cast<const T*>(p.keys) + b * p.k_sb + t * p.k_st + j * p.k_sh + c, k);
    load<T, VEC>(static_cast<const T*>(p.values) + b * p.v_sb + t * p.v_st + j * p.v_sh + c, v);
    pos = (int64_t)p.starts[b] + t;
    page = page_of(p, b, pos);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) k[i] = v[i] = 0.0f;
  }
  const int bs = 1 << p.page_shift, at = (int)(pos & (bs - 1));
  const int64_t kr = ((page * p.h.d + j) * 2) * bs + at, vr = kr + bs;  // rows of the page's keys and values
  if constexpr (INT8) {
    // Even lanes divide for the key's scale, odd ones for the value's.
    const uint2 tops = row_tops<T, L, C>(k, v);
    const int lane = threadIdx.x % 32;
    const float mine = scale_of((lane & 1) ? tops.y : tops.x);
    const float ks = __shfl_sync(0xffffffffu, mine, lane & ~1), vs = __shfl_sync(0xffffffffu, mine, lane | 1);
    uint32_t kq[C / 4], vq[C / 4];
    quantise<C>(k, ks, kq);
    quantise<C>(v, vs, vq);
    if (page < 0) return;
    int8_t* pages = static_cast<int8_t*>(p.pages);
    if constexpr (C == 8) {
      *reinterpret_cast<uint2*>(pages + kr * D + c) = make_uint2(kq[0], kq[1]);
      *reinterpret_cast<uint2*>(pages + vr * D + c) = make_uint2(vq[0], vq[1]);
    } else {
      *reinterpret_cast<uint32_t*>(pages + kr * D + c) = kq[0];
      *reinterpret_cast<uint32_t*>(pages + vr * D + c) = vq[0];
    }
    if (c == 0) {
      p.scales[kr] = ks;
      p.scales[vr] = vs;
    }
  } else {
    if (page < 0) return;
    store<T>(static_cast<T*>(p.pages) + kr * D + c, k);
    store<T>(static_cast<T*>(p.pages) + vr * D + c, v);
  }
}

// Grid: as for the write, kReads tokens of the grid's span apart per thread.
template <bool INT8>
constexpr int kReads = INT8 ? 4 : 2;
template <typename T, int D, bool INT8>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const PagedParams p) {
  constexpr int C = kCh<T>, L = D / C, R = kReads<INT8>, kWords = INT8 ? C / 4 : 4;
  pdl_wait();
  pdl_release();
  const uint32_t span = gridDim.x * (kThreads / L), first = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int c = (threadIdx.x % L) * C, bs = 1 << p.page_shift;
  int64_t from[R];  // the key's row of the pages, or -1
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t row = first + i * span;
    const uint32_t bt = p.h.of(row), j = row - bt * p.h.d, b = p.tokens.of(bt), t = bt - b * p.tokens.d;
    int64_t page = -1, pos = 0;
    if (row < p.rows) {
      pos = (int64_t)p.starts[b] + t;
      if (p.lens == nullptr || pos < p.lens[b]) page = page_of(p, b, pos);
    }
    from[i] = page < 0 ? -1 : (page * p.h.d + j) * 2 * bs + (pos & (bs - 1));
  }
  uint32_t w[R][2][kWords];
  float s[R][2];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const int64_t at = from[i] + kv * bs;
      const char* src = static_cast<const char*>(p.pages) + (at * D + c) * (INT8 ? 1 : (int)sizeof(T));
      s[i][kv] = 0.0f;
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[i][kv][k] = 0;
      if (from[i] >= 0) {
        if constexpr (kWords == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(src);
          w[i][kv][0] = x.x, w[i][kv][1] = x.y, w[i][kv][2] = x.z, w[i][kv][3] = x.w;
        } else if constexpr (kWords == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(src);
          w[i][kv][0] = x.x, w[i][kv][1] = x.y;
        } else {
          w[i][kv][0] = *reinterpret_cast<const uint32_t*>(src);
        }
        if (INT8) s[i][kv] = p.scales[at];
      }
    }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t row = first + i * span;
    if (row >= p.rows) return;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* to = static_cast<T*>(kv ? p.out_v : p.out_k) + (int64_t)row * D + c;
      if constexpr (INT8) {
        float x[C];
#pragma unroll
        for (int k = 0; k < C; ++k) x[k] = (float)(int8_t)(w[i][kv][k / 4] >> (8 * (k % 4))) * s[i][kv];
        store<T>(to, x);
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(w[i][kv][0], w[i][kv][1], w[i][kv][2], w[i][kv][3]);
      }
    }
  }
}

int check_cache(const char* who, int kind, int dtype, int h, int bs, int d, int64_t n_pages, const void* pages, const void* scales) {
  if (!dtype_ok(dtype)) return fail(LKV_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (kind != LKV_CACHE_MODEL && kind != LKV_CACHE_INT8) return fail(LKV_ERR_ARG, "%s: bad cache kind %d", who, kind);
  if (d != 64 && d != 128) return fail(LKV_ERR_ARG, "%s: head_dim %d (64 or 128)", who, d);
  if (bs != 16 && bs != 32 && bs != 64 && bs != 128) return fail(LKV_ERR_ARG, "%s: pages of %d tokens (16, 32, 64 or 128)", who, bs);
  if (h < 1 || n_pages < 0 || n_pages > INT32_MAX) return fail(LKV_ERR_ARG, "%s: bad shape (h %d, pages %lld)", who, h, (long long)n_pages);
  if (pages == nullptr || (kind == LKV_CACHE_INT8 && scales == nullptr)) return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(pages, 16) || !aligned(scales, 4)) return fail(LKV_ERR_PTR, "%s: pages must be 16-byte aligned", who);
  return LKV_OK;
}

int shift_of(int bs) { return bs == 16 ? 4 : bs == 32 ? 5 : bs == 64 ? 6 : 7; }

template <typename T, int D>
cudaError_t launch_write(const PagedParams& p, bool int8, bool vec, unsigned grid, cudaStream_t st) {
  if (int8) return vec ? launch_pdl(paged_write_kernel<T, D, true, true>, dim3(grid), dim3(kThreads), 0, st, 0, p)
                       : launch_pdl(paged_write_kernel<T, D, true, false>, dim3(grid), dim3(kThreads), 0, st, 0, p);
  return vec ? launch_pdl(paged_write_kernel<T, D, false, true>, dim3(grid), dim3(kThreads), 0, st, 0, p)
             : launch_pdl(paged_write_kernel<T, D, false, false>, dim3(grid), dim3(kThreads), 0, st, 0, p);
}

template <typename T, int D>
cudaError_t launch_read(const PagedParams& p, bool int8, unsigned grid, cudaStream_t st) {
  return int8 ? launch_pdl(paged_read_kernel<T, D, true>, dim3(grid), dim3(kThreads), 0, st, 0, p)
              : launch_pdl(paged_read_kernel<T, D, false>, dim3(grid), dim3(kThreads), 0, st, 0, p);
}

// What write and read check alike; `rows` gets batch * tokens * h.
int check_call(const char* who, const lkv_paged_args* a, int64_t* rows) {
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (int rc = check_cache(who, a->kind, a->dtype, a->h, a->bs, a->d, a->n_pages, a->pages, a->scales)) return rc;
  if (a->batch < 0 || a->tokens < 0 || a->table_cols < 0 || (a->batch > 1 && a->table_ld < a->table_cols))
    return fail(LKV_ERR_ARG, "%s: bad shape (batch %d, tokens %d, table of %d columns)", who, a->batch, a->tokens, a->table_cols);
  if ((int64_t)a->batch * a->tokens > INT32_MAX || (int64_t)a->batch * a->tokens * a->h > INT32_MAX)
    return fail(LKV_ERR_ARG, "%s: %d x %d x %d rows of one call", who, a->batch, a->tokens, a->h);
  *rows = (int64_t)a->batch * a->tokens * a->h;
  return LKV_OK;
}

PagedParams params_of(const lkv_paged_args* a, int64_t rows) {
  PagedParams p = {};
  p.keys = a->keys;
  p.values = a->values;
  p.k_sb = a->k_sb, p.k_st = a->k_st, p.k_sh = a->k_sh;
  p.v_sb = a->v_sb, p.v_st = a->v_st, p.v_sh = a->v_sh;
  p.pages = a->pages;
  p.scales = a->scales;
  p.n_pages = a->n_pages;
  p.table = a->table;
  p.table_ld = a->table_ld;
  p.table_cols = a->table_cols;
  p.starts = a->starts;
  p.lens = a->lens;
  p.rows = (uint32_t)rows;
  p.tokens = divisor(a->tokens);
  p.h = divisor(a->h);
  p.page_shift = shift_of(a->bs);
  p.out_k = a->out_k;
  p.out_v = a->out_v;
  return p;
}

unsigned grid_of(int64_t rows, int d, int dtype, int per_thread) {
  const unsigned per_cta = kThreads / (d * (unsigned)dtype_size(dtype) / 16) * per_thread;
  return (unsigned)((rows + per_cta - 1) / per_cta);
}

}  // namespace
}  // namespace lkv

using namespace lkv;

extern "C" {

int lkv_paged_write(const lkv_paged_args* a, void* stream) {
  static const char* who = "lkv_paged_write";
  int64_t rows = 0;
  if (int rc = check_call(who, a, &rows)) return rc;
  if (rows == 0 || a->n_pages == 0 || a->table_cols == 0) return LKV_OK;
  if (a->keys == nullptr || a->values == nullptr || a->table == nullptr || a->starts == nullptr) return fail(LKV_ERR_PTR, "%s: null pointer", who);
  const int size = (int)dtype_size(a->dtype), per = 16 / size;
  if (!aligned(a->keys, size) || !aligned(a->values, size)) return fail(LKV_ERR_PTR, "%s: misaligned keys or values", who);
  const bool vec = aligned(a->keys, 16) && aligned(a->values, 16) && a->k_sb % per == 0 && a->k_st % per == 0 && a->k_sh % per == 0 &&
                   a->v_sb % per == 0 && a->v_st % per == 0 && a->v_sh % per == 0;
  const PagedParams p = params_of(a, rows);
  const unsigned grid = grid_of(rows, a->d, a->dtype, 1);
  const bool int8 = a->kind == LKV_CACHE_INT8;
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (a->dtype == LKV_BF16)
    e = a->d == 64 ? launch_write<__nv_bfloat16, 64>(p, int8, vec, grid, st) : launch_write<__nv_bfloat16, 128>(p, int8, vec, grid, st);
  else
    e = a->d == 64 ? launch_write<float, 64>(p, int8, vec, grid, st) : launch_write<float, 128>(p, int8, vec, grid, st);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

int lkv_paged_read(const lkv_paged_args* a, void* stream) {
  static const char* who = "lkv_paged_read";
  int64_t rows = 0;
  if (int rc = check_call(who, a, &rows)) return rc;
  if (rows == 0) return LKV_OK;
  if ((a->table == nullptr && a->table_cols > 0) || a->starts == nullptr || a->out_k == nullptr || a->out_v == nullptr)
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(a->out_k, 16) || !aligned(a->out_v, 16)) return fail(LKV_ERR_PTR, "%s: outputs must be 16-byte aligned", who);
  const PagedParams p = params_of(a, rows);
  const bool int8 = a->kind == LKV_CACHE_INT8;
  const unsigned grid = grid_of(rows, a->d, a->dtype, int8 ? kReads<true> : kReads<false>);
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (a->dtype == LKV_BF16)
    e = a->d == 64 ? launch_read<__nv_bfloat16, 64>(p, int8, grid, st) : launch_read<__nv_bfloat16, 128>(p, int8, grid, st);
  else
    e = a->d == 64 ? launch_read<float, 64>(p, int8, grid, st) : launch_read<float, 128>(p, int8, grid, st);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
