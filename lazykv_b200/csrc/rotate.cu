// A step's queries and keys, normalised per head and rotated to their positions, and the keys and values
// written into their pages, in one pass over the projections' outputs.
//
// A head's row x of d channels becomes y = w x / sqrt(mean(x^2) + eps) where weights are given, and pair p
// of its channels (a, b), for p < pairs, turns by the angle t = position x frequencies[p]:
//   a cos t - b sin t,  b cos t + a sin t.
// Pairs are (p, p + pairs) or, interleaved, (2 p, 2 p + 1); channels from 2 pairs on do not turn. Queries are
// rounded once, to the model's type; keys and values go to model-dtype pages rounded once, or to int8
// codes as paged.cu quantises them, from the float32 values.
//
// What is rounded where: bfloat16 rows are computed in float32, float32 rows in float64, since a code is
// decided by the side of a border that its value lies on. The angle is a float64 product, brought below half
// a turn in float64 before its sine and cosine are taken: at position 10^6 a float32 angle is off by 0.03.
//
// Each row is read once and written once. A group of d / 8 lanes carries a row, a lane four channels of the first
// elements of pairs and the four of their second ones, so that a rotation needs no other lane. A CTA computes the angles
// of its tokens once for all heads.
//
// Measured: 32,768 tokens, 32 query and 8 KV heads, d 128, norms, to int8 pages 174 us (738 MB: 0.65 of a plain copy), the
// issue slots busy for the larger part; 64 tokens 4.8 us, three dependent loads and the angles.
#include "paged.cuh"
#include "tensor.cuh"

namespace lkv {
namespace {

using namespace paged;

constexpr int kThreads = 256;
constexpr int kMostTokens = 8;  // tokens of a CTA of a long call

struct RotateParams {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  void* out;
  int64_t o_st, o_sh;
  int rows, hq, h;
  const int32_t* positions;
  const float* frequencies;
  int pairs, interleaved;
  const void* q_weight;
  const void* k_weight;
  float eps;
  void* pages;
  float* scales;
  int64_t n_pages;
  int page_shift;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* lens;
  const int32_t* offsets;
  int batch;
  int token_shift;  // log2 of the tokens per CTA
};

template <typename T>
struct Wide {
  using type = float;
};
template <>
struct Wide<float> {
  using type = double;
};

// Four consecutive elements.
template <typename T>
struct Four;
template <>
struct Four<__nv_bfloat16> {
  uint2 w;
};
template <>
struct Four<float> {
  float4 w;
};

template <typename T, bool VEC>
__device__ __forceinline__ Four<T> load4(const T* p) {
  Four<T> f;
  if constexpr (VEC) {
    f.w = *reinterpret_cast<const decltype(f.w)*>(p);
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(p);
    f.w = make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
  } else {
    f.w = make_float4(p[0], p[1], p[2], p[3]);
  }
  return f;
}
template <typename W>
__device__ __forceinline__ void widen(const Four<__nv_bfloat16>& f, W* x) {
  x[0] = __uint_as_float(f.w.x << 16), x[1] = __uint_as_float(f.w.x & 0xffff0000u);
  x[2] = __uint_as_float(f.w.y << 16), x[3] = __uint_as_float(f.w.y & 0xffff0000u);
}
template <typename W>
__device__ __forceinline__ void widen(const Four<float>& f, W* x) {
  x[0] = f.w.x, x[1] = f.w.y, x[2] = f.w.z, x[3] = f.w.w;
}
template <bool VEC>
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* x) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
  }
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, const float* x) {
  if constexpr (VEC) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = x[i];
  }
}

// Cosine and sine of position x frequency. 2 pi in two parts: the whole turns' product is exact enough in two
// fused steps for any int32 position.
__device__ __forceinline__ void turn_of(int position, float frequency, float* c, float* s) {
  const double a = (double)position * (double)frequency, n = rint(a * 0.15915494309189535);
  double r = fma(-n, 6.283185307179586, a);
  r = fma(-n, 2.4492935982947064e-16, r);
  sincospif((float)(r * 0.3183098861837907), s, c);
}
__device__ __forceinline__ void turn_of(int position, float frequency, double* c, double* s) {
  const double a = (double)position * (double)frequency, n = rint(a * 0.15915494309189535);
  double r = fma(-n, 6.283185307179586, a);
  r = fma(-n, 2.4492935982947064e-16, r);
  sincospi(r * 0.3183098861837907, s, c);
}
__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }

// What a lane does to its pairs (a, b) of every row of one kind: weights and turn as four factors a pair, so that a
// normalised row is (a ca + b sb, b cb + a sa) / rms.
template <typename W>
struct Turn {
  W ca[4], sa[4], cb[4], sb[4];
  bool norm, turns;
};
__device__ __forceinline__ void apply(const Turn<double>& t, double (&a)[4], double (&b)[4], double inv) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double x = t.turns ? a[i] * t.ca[i] + b[i] * t.sb[i] : a[i] * t.ca[i], y = t.turns ? b[i] * t.cb[i] + a[i] * t.sa[i] : b[i] * t.cb[i];
    a[i] = x * inv, b[i] = y * inv;
  }
}
__device__ __forceinline__ void apply(const Turn<float>& t, float (&a)[4], float (&b)[4], float inv) {
  using namespace tc;
  const uint64_t by = pair(inv, inv);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint64_t x = pair(a[i], a[i + 1]), y = pair(b[i], b[i + 1]);
    uint64_t u = mul2(x, pair(t.ca[i], t.ca[i + 1])), v = mul2(y, pair(t.cb[i], t.cb[i + 1]));
    if (t.turns) {  // (a turn by nothing would still make a NaN of an infinite neighbour)
      u = fma2(y, pair(t.sb[i], t.sb[i + 1]), u);
      v = fma2(x, pair(t.sa[i], t.sa[i + 1]), v);
    }
    if (t.norm) u = mul2(u, by), v = mul2(v, by);
    a[i] = first_of(u), a[i + 1] = second_of(u), b[i] = first_of(v), b[i + 1] = second_of(v);
  }
}
__device__ __forceinline__ float squares(const float (&a)[4], const float (&b)[4]) {
  using namespace tc;
  uint64_t s = mul2(pair(a[0], a[1]), pair(a[0], a[1]));
  s = fma2(pair(a[2], a[3]), pair(a[2], a[3]), s);
  s = fma2(pair(b[0], b[1]), pair(b[0], b[1]), s);
  s = fma2(pair(b[2], b[3]), pair(b[2], b[3]), s);
  return first_of(s) + second_of(s);
}
__device__ __forceinline__ double squares(const double (&a)[4], const double (&b)[4]) {
  double s = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += a[i] * a[i] + b[i] * b[i];
  return s;
}

// INTER: pairs of neighbours. Grid: p.token_shift tokens a CTA.
template <typename T, int D, bool INT8, bool VEC, bool INTER>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 2) rotate_kernel(const RotateParams p) {
  using W = typename Wide<T>::type;
  constexpr int L = D / 8, kGroups = kThreads / L, U = 2;  // rows that a group asks for at once
  __shared__ W turns[2][kMostTokens][D / 2];  // cosines, sines
  __shared__ int64_t where[kMostTokens];      // row 0 of the token's place in its page; -1: no page; -2: no sequence's token
  pdl_wait();
  pdl_release();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, tokens = 1 << p.token_shift, row0 = blockIdx.x << p.token_shift;
  const int bs = 1 << p.page_shift;

  // A group's token, its heads sub, sub + per, .., and a lane's pairs: 4 l .. 4 l + 3, at channels c0 .. and c1 ..
  const int per = kGroups >> p.token_shift, group = tid / L, l = tid % L, t = group / per, sub = group % per, row = row0 + t;
  const uint32_t mask = L == 32 ? 0xffffffffu : ((1u << L) - 1) << (lane / L * L);
  int c0 = 8 * l, c1 = c0 + 4;
  if (!INTER) {
    const int pr = 4 * l;
    c0 = pr < p.pairs ? pr : pr + p.pairs;
    c1 = pr < p.pairs ? pr + p.pairs : pr + D / 2;
  }
  // A group's rows of one kind: sub, sub + per, ..; U of them are asked for at once. Addresses go on by a step a row.
  Four<T> lo[U], hi[U];
  const int to_c1 = c1 - c0;
  auto fetch = [&](const T* at, int64_t step, int j0, int n) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row < p.rows && j0 + u * per < n) lo[u] = load4<T, VEC>(at + u * step), hi[u] = load4<T, VEC>(at + u * step + to_c1);
  };
  auto first_of_kind = [&](const void* rows, int64_t s_token, int64_t s_head) { return static_cast<const T*>(rows) + (int64_t)row * s_token + sub * s_head + c0; };
  const T* q = first_of_kind(p.q, p.q_st, p.q_sh);
  const int64_t q_step = per * p.q_sh;
  fetch(q, q_step, sub, p.hq);

  if (warp >= 8 - tokens) {  // the last warps find the tokens' places
    const int mine = 7 - warp, r = row0 + mine;
    int b = 0;
    for (int i = lane; i < p.batch; i += 32) b += r < p.rows && p.offsets[i + 1] <= r;
    b = __reduce_add_sync(0xffffffffu, b);
    if (lane == 0) {
      int64_t at = -2;
      if (r < p.rows && b < p.batch) {
        const int from = p.offsets[b], end = p.offsets[b + 1];
        if (from <= r && r < end) {
          at = -1;
          const int64_t pos = (int64_t)p.lens[b] - end + r, col = pos >> p.page_shift;
          if (pos >= 0 && col < p.table_cols) {
            const int64_t page = p.table[(int64_t)b * p.table_ld + col];
            if (page >= 0 && page < p.n_pages) at = page * p.h * 2 * bs + (pos & (bs - 1));
          }
        }
      }
      where[mine] = at;
    }
  }
  for (int i = tid; i < tokens * (D / 2); i += kThreads) {
    const int tt = i / (D / 2), pr = i % (D / 2);
    W c = 1, s = 0;
    if (row0 + tt < p.rows && pr < p.pairs) turn_of(p.positions[row0 + tt], p.frequencies[pr], &c, &s);
    turns[0][tt][pr] = c, turns[1][tt][pr] = s;
  }
  __syncthreads();
  const int64_t place = where[t];
  if (place == -2) return;

  auto of = [](const Four<T>& x, const Four<T>& y, W (&a)[4], W (&b)[4]) {  // a lane's channels as its pairs
    W w[8];
    widen(x, w), widen(y, w + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = INTER ? w[2 * i] : w[i], b[i] = INTER ? w[2 * i + 1] : w[4 + i];
  };
  auto turn_with = [&](const void* weight) {
    Turn<W> f;
    f.norm = weight != nullptr, f.turns = 4 * l < p.pairs;
    W a[4] = {1, 1, 1, 1}, b[4] = {1, 1, 1, 1};
    if (f.norm) of(load4<T, VEC>(static_cast<const T*>(weight) + c0), load4<T, VEC>(static_cast<const T*>(weight) + c1), a, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const W c = turns[0][t][4 * l + i], s = turns[1][t][4 * l + i];
      f.ca[i] = a[i] * c, f.sa[i] = a[i] * s, f.cb[i] = b[i] * c, f.sb[i] = -b[i] * s;
    }
    return f;
  };
  auto turned = [&](const Turn<W>& f, W (&a)[4], W (&b)[4]) {
    W inv = 1;
    if (f.norm) {
      W sum = squares(a, b);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
      inv = inverse_root(sum * (W)(1.0 / D) + (W)p.eps);
    }
    apply(f, a, b, inv);
  };
  auto in_order = [](const W (&a)[4], const W (&b)[4], float (&z)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[INTER ? 2 * i : i] = (float)a[i], z[INTER ? 2 * i + 1 : 4 + i] = (float)b[i];
  };
  {
    const Turn<W> f = turn_with(p.q_weight);
    T* out = static_cast<T*>(p.out) + (int64_t)row * p.o_st + sub * p.o_sh + c0;
    const int64_t o_step = per * p.o_sh;
    for (int j0 = sub; j0 < p.hq; j0 += U * per) {
      if (j0 != sub) fetch(q, q_step, j0, p.hq);
      q += U * q_step;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * per;
        if (j >= p.hq) break;
        W a[4], b[4];
        of(lo[u], hi[u], a, b);
        turned(f, a, b);
        float z[8];
        in_order(a, b, z);
        store4<VEC>(out, z);
        store4<VEC>(out + to_c1, z + 4);
        out += o_step;
      }
    }
  }
  if (place < 0) return;
  const int64_t row_step = (int64_t)per * 2 * bs;
  auto put = [&](const float (&z)[8], int64_t to) {  // to: the row of the pages
    if constexpr (INT8) {
      uint32_t top = 0, codes[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
      const float s = scale_of(top);
      quantise<8>(z, s, codes);
      int8_t* dst = static_cast<int8_t*>(p.pages) + to * D;
      *reinterpret_cast<uint32_t*>(dst + c0) = codes[0];
      *reinterpret_cast<uint32_t*>(dst + c1) = codes[1];
      if (l == 0) p.scales[to] = s;
    } else {
      T* dst = static_cast<T*>(p.pages) + to * D;
      store4<true>(dst + c0, z);
      store4<true>(dst + c1, z + 4);
    }
  };
  {
    const Turn<W> f = turn_with(p.k_weight);
    const T* k = first_of_kind(p.k, p.k_st, p.k_sh);
    const int64_t k_step = per * p.k_sh;
    int64_t to = place + (int64_t)sub * 2 * bs;
    for (int j0 = sub; j0 < p.h; j0 += U * per, k += U * k_step) {
      fetch(k, k_step, j0, p.h);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * per;
        if (j >= p.h) break;
        W a[4], b[4];
        of(lo[u], hi[u], a, b);
        turned(f, a, b);
        float z[8];
        in_order(a, b, z);
        put(z, to);
        to += row_step;
      }
    }
  }
  const T* v = first_of_kind(p.v, p.v_st, p.v_sh);
  const int64_t v_step = per * p.v_sh;
  int64_t to = place + ((int64_t)sub * 2 + 1) * bs;
  for (int j0 = sub; j0 < p.h; j0 += U * per, v += U * v_step) {
    fetch(v, v_step, j0, p.h);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * per;
      if (j >= p.h) break;
      W w[8];
      widen(lo[u], w), widen(hi[u], w + 4);
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = (float)w[i];
      put(z, to);
      to += row_step;
    }
  }
}

template <typename T, int D, bool INT8, bool VEC>
cudaError_t launch_as(const RotateParams& p, unsigned grid, cudaStream_t st) {
  return p.interleaved ? launch_pdl(rotate_kernel<T, D, INT8, VEC, true>, dim3(grid), dim3(kThreads), 0, st, 0, p)
                       : launch_pdl(rotate_kernel<T, D, INT8, VEC, false>, dim3(grid), dim3(kThreads), 0, st, 0, p);
}
template <typename T, int D>
cudaError_t launch(const RotateParams& p, bool int8, bool vec, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)p.rows + (1 << p.token_shift) - 1) >> p.token_shift);
  if (int8) return vec ? launch_as<T, D, true, true>(p, grid, st) : launch_as<T, D, true, false>(p, grid, st);
  return vec ? launch_as<T, D, false, true>(p, grid, st) : launch_as<T, D, false, false>(p, grid, st);
}

}  // namespace
}  // namespace lkv

using namespace lkv;

extern "C" int lkv_paged_write_rotated(const lkv_rotate_args* a, void* stream) {
  static const char* who = "lkv_paged_write_rotated";
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (int rc = check_cache(who, a->kind, a->dtype, a->h, a->bs, a->d, a->n_pages, a->pages, a->scales)) return rc;
  if (a->rows < 0 || a->rows > (1 << 30) || a->hq < 0 || a->batch < 0 || a->table_cols < 0 || (a->batch > 1 && a->table_ld < a->table_cols) || a->hq > 65536 || a->h > 65536)
    return fail(LKV_ERR_ARG, "%s: bad shape (rows %d, heads %d and %d, batch %d, table of %d columns)", who, a->rows, a->hq, a->h, a->batch, a->table_cols);
  if (a->pairs < 0 || a->pairs > a->d / 2 || a->pairs % 4 != 0) return fail(LKV_ERR_ARG, "%s: %d rotated pairs of head_dim %d (a multiple of 4)", who, a->pairs, a->d);
  if (!(a->eps >= 0.0f)) return fail(LKV_ERR_ARG, "%s: eps %g", who, (double)a->eps);
  if (a->rows == 0 || a->batch == 0) return LKV_OK;
  if (a->keys == nullptr || a->values == nullptr || a->lens == nullptr || a->offsets == nullptr || (a->table == nullptr && a->table_cols > 0) ||
      (a->hq > 0 && (a->q == nullptr || a->out == nullptr)) || (a->pairs > 0 && (a->positions == nullptr || a->frequencies == nullptr)))
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  const int size = (int)dtype_size(a->dtype);
  const void* all[6] = {a->q, a->keys, a->values, a->out, a->q_weight, a->k_weight};
  bool vec = ((a->q_st | a->q_sh | a->k_st | a->k_sh | a->v_st | a->v_sh | a->o_st | a->o_sh) & 3) == 0;
  for (const void* x : all) {
    if (!aligned(x, size)) return fail(LKV_ERR_PTR, "%s: misaligned rows or weights", who);
    vec = vec && aligned(x, 4 * size);
  }
  RotateParams p = {};
  p.q = a->q, p.k = a->keys, p.v = a->values;
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.k_st = a->k_st, p.k_sh = a->k_sh, p.v_st = a->v_st, p.v_sh = a->v_sh;
  p.out = a->out, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.rows = a->rows, p.hq = a->hq, p.h = a->h;
  p.positions = a->positions, p.frequencies = a->frequencies, p.pairs = a->pairs, p.interleaved = a->interleaved != 0;
  p.q_weight = a->q_weight, p.k_weight = a->k_weight, p.eps = a->eps;
  p.pages = a->pages, p.scales = a->scales, p.n_pages = a->n_pages, p.page_shift = shift_of(a->bs);
  p.table = a->table, p.table_ld = a->table_ld, p.table_cols = a->table_cols, p.lens = a->lens, p.offsets = a->offsets, p.batch = a->batch;
  // As many tokens to a CTA, up to eight, as leave every SM two CTAs (their angles, places and waits are shared: 2%
  // less time with eight than with four for a prompt of 32,768 tokens, 32 and 8 heads, d 128, to int8 pages).
  while (p.token_shift < 3 && a->rows >> (p.token_shift + 1) >= 2 * kNumSMs) ++p.token_shift;
  const bool int8 = a->kind == LKV_CACHE_INT8;
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (a->dtype == LKV_BF16)
    e = a->d == 64 ? launch<__nv_bfloat16, 64>(p, int8, vec, st) : launch<__nv_bfloat16, 128>(p, int8, vec, st);
  else
    e = a->d == 64 ? launch<float, 64>(p, int8, vec, st) : launch<float, 128>(p, int8, vec, st);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}
