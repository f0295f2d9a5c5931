// Attention of a batch that shares a prefix: every query attends the prefix's tokens and its own
// sequence's, and the prefix's pages are read once for the whole batch.
//
// The query rows of KV head j are (b, t, g): sequence, position among the step's tokens, query head of
// the group. Row (b, t, g) sees the prefix [0, prefix_len) and own tokens 0 .. lens[b] - tokens + t.
// Softmaxes over disjoint key sets merge exactly by their references and sums, so the work is cut into
// partials (m, l, o), l = sum 2^(s - m), o = sum 2^(s - m) v, s the scores in the log2 domain:
//   1. prefix_tile_kernel (prefix_tile.cu): the prefix for many rows, on tcgen05;
//   2. stream_kernel: the sequences' own tokens, and the prefix too where the batch has few rows;
//   3. combine_kernel: the partials of every row.
// Each launch starts under the one before it (programmatic dependent launch): the stream's CTAs take the
// SMs that the tiles leave, or never had (32 rows on 32K int8 tokens: 38 us, the other way about 44).
//
// stream_kernel's work is one line of stages (prefix.cuh) that all warps
// of the grid share equally, whatever the sequences' lengths: only the device knows them, and with a CTA
// or a cluster per (sequence, head) the longest sequence set the time. A warp takes a tile of 16 rows
// through its stages with mma.sync.m16n8k16 (float32 accumulators). A lane copies by cp.async exactly the
// bytes that it will hold as mma fragments, into slots of shared memory of its own, so the pipeline needs
// no barrier and has no bank conflicts; the channels are permuted so that a fragment's elements are 16
// contiguous bytes of a row (a dot product does not mind, and the output's permutation ends in contiguous
// runs again).
//
// bf16 pages: a weight goes into the second product as two bf16 terms (prefix.cuh, rest_of: 2^-15 of it is
// lost): twice the products at 0 to 3% of the time, since copies bound it. int8 pages: codes and queries are f16
// (prefix_tile.cu tells how exactly), a key's scale multiplies its column of scores in float32, and a value's scale
// its column of weights, before they are rounded to f16, the only rounding of the second product's operands (prefix.cuh, weight_room: 2^-11 relative,
// and an absolute 2^-31 of the largest weight times scale).
//
// Measured: 6 sequences on 32,768 bf16 tokens, 16 KV heads, d 128: 276 MB in 63 us, 4.4 TB/s; each further
// token moves at 5.8 TB/s, the rest is the start, the last stages and the merge (13 us). int8 pages are bound by
// issue slots instead, some 600 instructions of a warp per 16 tokens and head (codes to f16, products, softmax):
// 64 sequences' own 0 .. 2,000 tokens, 8 KV heads of d 128, take 46 us at 37% of the memory's cycles (bf16: 63 us
// at 52%).
#include "prefix.cuh"

namespace lkv {
namespace prefix {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLag = 8.0f;  // powers of two that a reference may lag behind the maximum

template <bool F16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int N>
__device__ __forceinline__ void copy(uint32_t dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
// N bytes, or N zeros where !there (nothing is read then).
template <int N>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void* src, bool there) {
  const int n = there ? N : 0;
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }

constexpr int stage_shift_of(int d) { return d == 128 ? 4 : 5; }

// Geometry of the stream for one head dimension and cache type.
template <int D, bool INT8>
struct Shape {
  static constexpr int kElt = INT8 ? 1 : 2;
  static constexpr int kTok = 1 << stage_shift_of(D);          // tokens per stage
  static constexpr int kGran = kTok / 16;                      // 16-token granules per stage
  static constexpr int kKLoads = D * kElt / 64;                // 16-byte loads per lane and 8 keys (4 lanes a row)
  static constexpr int kVBytes = D * kElt / 8 >= 16 ? 16 : 8;  // bytes per lane and load of a value row (8 lanes a row)
  static constexpr int kVLoads = D * kElt / 8 / kVBytes;
  static constexpr int kKBytes = 2 * kKLoads * 16;             // per lane and granule
  static constexpr int kVAll = 4 * kVLoads * kVBytes;
  static constexpr int kSBytes = INT8 ? 32 : 0;                // the scales of 4 tokens' keys and values
  static constexpr int kGranBytes = (kKBytes + kVAll + kSBytes) * 32;
  static constexpr int kStageBytes = kGran * kGranBytes;
  static constexpr int kStages = 3;
  static constexpr int kRing = kWarps * kStages * kStageBytes;  // 60 to 96 KB; the warps' states fit too
  static_assert(kRing >= kWarps * kRows * ((D + 4) * 4 + 8), "the merge is done in the ring");
  static constexpr int kCtas = INT8 ? 3 : 2;                    // per SM
  static constexpr int kVCh = kVBytes / kElt;                   // channels per value load
  // The channel of column n of the i-th output tile: kVCh consecutive ones per column and kVCh tiles.
  __device__ static __forceinline__ int channel(int i, int n) { return (i / kVCh) * (8 * kVCh) + n * kVCh + i % kVCh; }
};

// One warp's running softmax over its tokens: lane (r, c) = (lane / 4, lane % 4) holds rows r and r + 8.
template <int D>
struct State {
  float o[D / 8][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
  }
};

// The A fragments of a 16-row tile of queries, channels permuted as the keys' are, and per row what its
// scores have to be multiplied with. Rows without a pointer are zero.
template <int D, bool INT8>
__device__ __forceinline__ void load_queries(uint32_t (&qf)[D / 16][4], float (&scale)[2], const __nv_bfloat16* lo, const __nv_bfloat16* hi, int c,
                                             float scale_log2) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const __nv_bfloat16* row = half ? hi : lo;
    scale[half] = scale_log2;
    if constexpr (INT8) {
      uint4 w[D / 64][2];
      uint32_t top = 0;
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          w[x][y] = row != nullptr ? reinterpret_cast<const uint4*>(row + 64 * x + 16 * c)[y] : make_uint4(0, 0, 0, 0);
          const uint32_t u[4] = {w[x][y].x, w[x][y].y, w[x][y].z, w[x][y].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
        }
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float2 by = row_scales(top);
      scale[half] *= by.y;
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w[x]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // k-step 4 x + i: four channels
          qf[4 * x + i][half] = pack_f16(__uint_as_float(u[2 * i] << 16) * by.x, __uint_as_float(u[2 * i] & 0xffff0000u) * by.x);
          qf[4 * x + i][2 + half] = pack_f16(__uint_as_float(u[2 * i + 1] << 16) * by.x, __uint_as_float(u[2 * i + 1] & 0xffff0000u) * by.x);
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row != nullptr) w = *reinterpret_cast<const uint4*>(row + 32 * x + 8 * c);
        qf[2 * x][half] = w.x, qf[2 * x][2 + half] = w.y;
        qf[2 * x + 1][half] = w.z, qf[2 * x + 1][2 + half] = w.w;
      }
    }
  }
}

// Starts the copies of one stage: tokens first .. first + kTok - 1 of a list that ends at `end`, those at
// or past it and those without a page as zeros. Returns a bit per granule that has a page.
template <int D, bool INT8>
__device__ __forceinline__ uint32_t fill_stage(const Params& p, int j, const int (&id)[Shape<D, INT8>::kGran], int first, int end, uint32_t slot, int lane) {
  using S = Shape<D, INT8>;
  constexpr int kRowBytes = D * S::kElt;
  const int r = lane / 4, c = lane % 4;
  const int bs = 1 << p.page_shift;
  uint32_t have = 0;
#pragma unroll
  for (int g = 0; g < S::kGran; ++g) {
    const int tok = first + 16 * g;
    const bool ok = id[g] >= 0 && id[g] < p.n_pages && tok < end;
    have |= (ok ? 1u : 0u) << g;
    const int64_t krow = (((int64_t)(ok ? id[g] : 0) * p.h + j) * 2) * bs + (tok & (bs - 1));
    const char* kp = static_cast<const char*>(p.pages) + krow * kRowBytes;
    const char* vp = kp + bs * kRowBytes + 2 * c * kRowBytes + r * S::kVBytes;
    kp += r * kRowBytes + 16 * c;
    const uint32_t kd = slot + g * S::kGranBytes + lane * 16, vd = slot + g * S::kGranBytes + S::kKBytes * 32 + lane * S::kVBytes;
    if (ok && tok + 16 <= end) {
#pragma unroll
      for (int i = 0; i < 2 * S::kKLoads; ++i) copy<16>(kd + 512 * i, kp + (i / S::kKLoads) * 8 * kRowBytes + 64 * (i % S::kKLoads));
#pragma unroll
      for (int i = 0; i < 4 * S::kVLoads; ++i)
        copy<S::kVBytes>(vd + S::kVBytes * 32 * i, vp + (((i / S::kVLoads) & 1) + 8 * (i / S::kVLoads >> 1)) * kRowBytes + (i % S::kVLoads) * 8 * S::kVBytes);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * S::kKLoads; ++i)
        copy_or_zero<16>(kd + 512 * i, kp + (i / S::kKLoads) * 8 * kRowBytes + 64 * (i % S::kKLoads), ok && tok + 8 * (i / S::kKLoads) + r < end);
#pragma unroll
      for (int i = 0; i < 4 * S::kVLoads; ++i) {
        const int t = ((i / S::kVLoads) & 1) + 8 * (i / S::kVLoads >> 1);
        copy_or_zero<S::kVBytes>(vd + S::kVBytes * 32 * i, vp + t * kRowBytes + (i % S::kVLoads) * 8 * S::kVBytes, ok && tok + 2 * c + t < end);
      }
    }
    if constexpr (INT8) {
      const uint32_t sd = slot + g * S::kGranBytes + (S::kKBytes + S::kVAll) * 32 + lane * 8;
      const float* sp = p.scales + krow + 2 * c;  // two tokens' key scales, then (bs further) their value scales
      // Past `end` inside a page the scales are read all the same: they exist, and their columns are masked.
#pragma unroll
      for (int i = 0; i < 4; ++i) copy_or_zero<8>(sd + 256 * i, sp + (i >> 1) * bs + 8 * (i & 1), ok);
    }
  }
  copies_done();
  return have;
}

// A granule's P V without mma (see fold_stage), token by token; seen: how many of them rows r and r + 8 see.
template <int D>
__device__ __forceinline__ void fold_values_singly(State<D>& st, const char* values, const float (&s)[2][4], const int (&seen)[2], int lane) {
  using S = Shape<D, false>;
  const int c = lane % 4;
  __syncwarp();  // a lane has waited for its own copies; here it reads other lanes' too
#pragma unroll 1
  for (int t = 0; t < 16; ++t) {
    const int c2 = (t & 7) >> 1, owner = (lane & ~3) | c2;  // the lane that holds this token's weights of rows r, r + 8
    const float x0 = t < 8 ? (t & 1 ? s[0][1] : s[0][0]) : (t & 1 ? s[1][1] : s[1][0]);
    const float x1 = t < 8 ? (t & 1 ? s[0][3] : s[0][2]) : (t & 1 ? s[1][3] : s[1][2]);
    const float p0 = __shfl_sync(0xffffffffu, x0, owner), p1 = __shfl_sync(0xffffffffu, x1, owner);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      // Column n of output tile i is in what lane (n, c2) copied: load t % 2 + 2 (t / 8), and i / kVCh of it.
      const char* src = values + (((t & 1) + 2 * (t >> 3)) * S::kVLoads + i / S::kVCh) * (S::kVBytes * 32) + 2 * (i % S::kVCh);
      const float va = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(src + ((2 * c) * 4 + c2) * S::kVBytes));
      const float vb = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(src + ((2 * c + 1) * 4 + c2) * S::kVBytes));
      if (t < seen[0]) st.o[i][0] += p0 * va, st.o[i][1] += p0 * vb;
      if (t < seen[1]) st.o[i][2] += p1 * va, st.o[i][3] += p1 * vb;
    }
  }
  __syncwarp();  // these slots are other lanes' to fill again
}

// One stage's tokens folded into the warp's state. limit[0/1]: the tokens that rows r and r + 8 see. MASKED:
// some row's sight ends in this stage, or a page is missing.
template <int D, bool INT8, bool MASKED>
__device__ __forceinline__ void fold_stage(State<D>& st, const uint32_t (&qf)[D / 16][4], const float (&scale)[2], const char* slot, int first,
                                           const int (&limit)[2], uint32_t have, int lane) {
  using S = Shape<D, INT8>;
  const int c = lane % 4;
  float s[2 * S::kGran][4];
  float2 vs[2 * S::kGran];  // int8: the value scales of this lane's columns
#pragma unroll
  for (int g = 0; g < S::kGran; ++g) {
    const char* base = slot + g * S::kGranBytes + lane * 16;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      float* x = s[2 * g + nt];
      x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll
      for (int i = 0; i < S::kKLoads; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(base + (nt * S::kKLoads + i) * 512);
        if constexpr (INT8) {
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint2 b = codes_to_f16(u[k]);
            mma16816<true>(x, qf[4 * i + k], b.x, b.y);
          }
        } else {
          mma16816<false>(x, qf[2 * i], w.x, w.y);
          mma16816<false>(x, qf[2 * i + 1], w.z, w.w);
        }
      }
      if constexpr (INT8) {
        const char* sp = slot + g * S::kGranBytes + (S::kKBytes + S::kVAll) * 32 + nt * 256 + lane * 8;
        const float2 ks = *reinterpret_cast<const float2*>(sp);
        vs[2 * g + nt] = *reinterpret_cast<const float2*>(sp + 512);
        // The scales' product first: a key's and a query row's may be as far apart as float32 goes.
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= (e & 1 ? ks.y : ks.x) * scale[e >> 1];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= scale[e >> 1];
      }
    }
  }
  if constexpr (MASKED) {
#pragma unroll
    for (int n = 0; n < 2 * S::kGran; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = first + 8 * n + 2 * c + (e & 1);
        if (tok >= limit[e >> 1] || !((have >> (n / 2)) & 1)) s[n][e] = -INFINITY;
      }
  }
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int n = 0; n < 2 * S::kGran; ++n) {
    // int8: a weight is rounded together with its token's value scale, so the largest product sets the reference,
    // not the largest weight, and what a row does not see (a score of -infinity) has no part in it.
    const float up[2] = {INT8 ? weight_room(vs[n].x) : 0.0f, INT8 ? weight_room(vs[n].y) : 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], INT8 ? s[n][e] + up[e & 1] : s[n][e]);
  }
  // A reference moves where a lane sees it outgrown (or has none yet), for the four lanes of the row alike.
  if (__any_sync(0xffffffffu, top[0] > st.m[0] + kLag || top[1] > st.m[1] + kLag)) {
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float want = top[i];
      want = fmaxf(want, __shfl_xor_sync(0xffffffffu, want, 1));
      want = fmaxf(want, __shfl_xor_sync(0xffffffffu, want, 2));
      f[i] = want > st.m[i] ? ex2(st.m[i] - want) : 1.0f;  // 0 where nothing was seen before
      st.l[i] = INT8 && want > st.m[i] ? times_ex2(st.l[i], st.m[i] - want) : st.l[i] * f[i];
      st.m[i] = fmaxf(st.m[i], want);
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) st.o[i][0] *= f[0], st.o[i][1] *= f[0], st.o[i][2] *= f[1], st.o[i][3] *= f[1];
  }
  // A row that has seen nothing keeps m = -inf: its weights come from a reference of 0, ex2(-inf) = 0.
  const float m0 = st.m[0] == -INFINITY ? 0.0f : st.m[0], m1 = st.m[1] == -INFINITY ? 0.0f : st.m[1];
#pragma unroll
  for (int n = 0; n < 2 * S::kGran; ++n) {
    s[n][0] = ex2(s[n][0] - m0), s[n][1] = ex2(s[n][1] - m0);
    s[n][2] = ex2(s[n][2] - m1), s[n][3] = ex2(s[n][3] - m1);
    st.l[0] += s[n][0] + s[n][1];
    st.l[1] += s[n][2] + s[n][3];
    if constexpr (INT8) {
      const float by2[2] = {vs[n].x * kScaleDown, vs[n].y * kScaleDown};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // What a row does not see is nothing whatever its scale; what it sees counts, a NaN under a weight of zero too.
        const bool unseen = MASKED && (first + 8 * n + 2 * c + (e & 1) >= limit[e >> 1] || !((have >> (n / 2)) & 1));
        s[n][e] = unseen ? 0.0f : s[n][e] * by2[e & 1];
      }
    }
  }
#pragma unroll
  for (int g = 0; g < S::kGran; ++g) {
    const char* values = slot + g * S::kGranBytes + S::kKBytes * 32;
    uint32_t w[S::kVLoads][4][S::kVBytes / 4];
#pragma unroll
    for (int y = 0; y < S::kVLoads; ++y)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const char* src = values + lane * S::kVBytes + (t * S::kVLoads + y) * (S::kVBytes * 32);
        if constexpr (S::kVBytes == 16) {
          const uint4 x = *reinterpret_cast<const uint4*>(src);
          w[y][t][0] = x.x, w[y][t][1] = x.y, w[y][t][2] = x.z, w[y][t][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(src);
          w[y][t][0] = x.x, w[y][t][1] = x.y;
        }
      }
    if constexpr (MASKED && !INT8) {
      // 0 x infinity is NaN: a token that some rows do not see must not reach them through a value that is
      // not finite.
      bool odd = false;
#pragma unroll
      for (int y = 0; y < S::kVLoads; ++y)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < S::kVBytes / 4; ++i) odd = odd || (w[y][t][i] & 0x7f80u) == 0x7f80u || (w[y][t][i] & 0x7f800000u) == 0x7f800000u;
      if (__any_sync(0xffffffffu, odd)) {
        const float weights[2][4] = {{s[2 * g][0], s[2 * g][1], s[2 * g][2], s[2 * g][3]}, {s[2 * g + 1][0], s[2 * g + 1][1], s[2 * g + 1][2], s[2 * g + 1][3]}};
        const bool page = (have >> g) & 1;
        const int seen[2] = {page ? limit[0] - first - 16 * g : 0, page ? limit[1] - first - 16 * g : 0};
        fold_values_singly<D>(st, values, weights, seen, lane);
        continue;
      }
    }
    auto packed = [](float x, float y) { return INT8 ? pack_f16(x, y) : upper_halves(x, y); };
    const uint32_t a[4] = {packed(s[2 * g][0], s[2 * g][1]), packed(s[2 * g][2], s[2 * g][3]), packed(s[2 * g + 1][0], s[2 * g + 1][1]),
                           packed(s[2 * g + 1][2], s[2 * g + 1][3])};
    [[maybe_unused]] uint32_t low[4];  // the second terms
    if constexpr (!INT8) {
      auto rest = [](float x, float y) { return pack_bf16(rest_of(x), rest_of(y)); };
      low[0] = rest(s[2 * g][0], s[2 * g][1]), low[1] = rest(s[2 * g][2], s[2 * g][3]);
      low[2] = rest(s[2 * g + 1][0], s[2 * g + 1][1]), low[3] = rest(s[2 * g + 1][2], s[2 * g + 1][3]);
    }
#pragma unroll
    for (int y = 0; y < S::kVLoads; ++y)
#pragma unroll
      for (int i = 0; i < S::kVBytes / 4; ++i) {
        const uint32_t(&v)[4][S::kVBytes / 4] = w[y];
        if constexpr (INT8) {
          // Bytes of two tokens by turns: (0, 1) of both, then (2, 3).
          const uint2 lo01 = codes_to_f16(__byte_perm(v[0][i], v[1][i], 0x5140)), hi01 = codes_to_f16(__byte_perm(v[0][i], v[1][i], 0x7362));
          const uint2 lo23 = codes_to_f16(__byte_perm(v[2][i], v[3][i], 0x5140)), hi23 = codes_to_f16(__byte_perm(v[2][i], v[3][i], 0x7362));
          float(*o)[4] = &st.o[S::kVCh * y + 4 * i];
          mma16816<true>(o[0], a, lo01.x, lo23.x);
          mma16816<true>(o[1], a, lo01.y, lo23.y);
          mma16816<true>(o[2], a, hi01.x, hi23.x);
          mma16816<true>(o[3], a, hi01.y, hi23.y);
        } else {
          const uint32_t even[2] = {__byte_perm(v[0][i], v[1][i], 0x5410), __byte_perm(v[2][i], v[3][i], 0x5410)};
          const uint32_t odd[2] = {__byte_perm(v[0][i], v[1][i], 0x7632), __byte_perm(v[2][i], v[3][i], 0x7632)};
          mma16816<false>(st.o[S::kVCh * y + 2 * i], a, even[0], even[1]);
          mma16816<false>(st.o[S::kVCh * y + 2 * i + 1], a, odd[0], odd[1]);
          mma16816<false>(st.o[S::kVCh * y + 2 * i], low, even[0], even[1]);
          mma16816<false>(st.o[S::kVCh * y + 2 * i + 1], low, odd[0], odd[1]);
        }
      }
  }
}

// The line, as a warp sees it: a lane has the length on it of the sequences before its slice of sequences
// (of one head's and row tile's units), and the length of all.
struct Line {
  int64_t before, all;
};
__device__ __forceinline__ int slice_of(const Params& p) { return (p.batch + 31) / 32; }

__device__ __forceinline__ Line sum_line(const Params& p, int lane) {
  const int n = slice_of(p);
  int64_t mine = 0;
  for (int b = lane * n; b < min(p.batch, (lane + 1) * n); ++b) mine += length_of(stages_of(p, p.lens[b]));
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  return {upto - mine, __shfl_sync(0xffffffffu, upto, 31)};
}
// Lengths of the prefix's part, of the whole line, and of each warp's piece of it.
__device__ __forceinline__ int64_t prefix_length(const Params& p) { return (int64_t)length_of(p.prefix_stages) * p.h * p.prefix_row_tiles; }
__device__ __forceinline__ int64_t line_length(const Params& p, const Line& line) {
  return prefix_length(p) + line.all * p.h * p.own_row_tiles;
}
__device__ __forceinline__ int64_t piece_length(const Params& p, const Line& line) {
  return max(quotient(line_length(p, line) + p.n_warps - 1, p.n_warps), (int64_t)kMinStages);
}

// A place on the line, `x` further than the warp's first: stage s of the n of unit `unit` of sequence b (-1:
// of the prefix), units of one list counted head by head, row tile by row tile.
struct Place {
  int64_t x;
  int b, unit, s, n, len;
};
// To the first stage of the next unit, which lies `skip` further.
__device__ __forceinline__ void next_unit(const Params& p, Place& at, int skip) {
  at.x += skip;
  at.s = 0;
  if (++at.unit < p.h * (at.b < 0 ? p.prefix_row_tiles : p.own_row_tiles)) return;
  at.unit = 0;
  do {
    if (++at.b >= p.batch) {
      at.x = INT64_MAX;  // the line's end
      return;
    }
    at.len = own_len(p, p.lens[at.b]);
    at.n = stages_of(p, at.len);
  } while (at.n == 0);
}
__device__ __forceinline__ void advance(const Params& p, Place& at) {
  ++at.x;
  if (++at.s == at.n) next_unit(p, at, kUnitStages);
}
// The first stage at or past place x of the line (x inside it).
__device__ __forceinline__ Place place_at(const Params& p, const Line& line, int64_t x) {
  Place at;
  at.x = 0;
  const int64_t prefix = prefix_length(p);
  int64_t rest = x;
  if (x < prefix) {
    at.b = -1, at.n = p.prefix_stages, at.len = p.prefix_len;
  } else {
    x -= prefix;
    const int per = p.h * p.own_row_tiles;
    const int lo = 31 - __clz(__ballot_sync(0xffffffffu, line.before * per <= x));  // the last slice that begins at or before x
    int64_t before = __shfl_sync(0xffffffffu, line.before, lo);
    for (at.b = lo * slice_of(p);; ++at.b) {
      at.len = own_len(p, p.lens[at.b]);
      at.n = stages_of(p, at.len);
      if (x < (before + length_of(at.n)) * per) break;
      before += length_of(at.n);
    }
    rest = x - before * per;
  }
  const int length = length_of(at.n);
  at.unit = (int)quotient(rest, length);
  at.s = (int)(rest - (int64_t)at.unit * length);
  if (at.s >= at.n) next_unit(p, at, length - at.s);
  return at;
}

template <int D, bool INT8>
__device__ __forceinline__ void stream(const Params& p, char* ring) {
  using S = Shape<D, INT8>;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, r = lane / 4, c = lane % 4;
  const Line line = sum_line(p, lane);
  const int w = blockIdx.x * kWarps + warp;
  const int64_t piece = piece_length(p, line), length = line_length(p, line);
  const int64_t x0 = w * piece, n = min(piece, length - x0);  // this warp's places: x0 .. x0 + n - 1
  // One unit's stages may fill the pieces of all four warps: then they are merged here.
  bool whole = false;
  Place at;
  if ((w - warp) * piece < length) {
    at = place_at(p, line, (w - warp) * piece);
    whole = at.x == 0 && at.n - at.s >= kWarps * piece;
    if (whole) at.s += (int)(warp * piece);
    else if (warp > 0 && n > 0) at = place_at(p, line, x0);
  }
  if (!whole && n <= 0) return;
  Place ahead = at;
  const uint32_t slots = (uint32_t)__cvta_generic_to_shared(ring) + warp * (S::kStages * S::kStageBytes);
  const char* slots_p = ring + warp * (S::kStages * S::kStageBytes);
  // Pages are looked up one stage before their copies start.
  int id[S::kGran];
  auto look_up = [&]() {
    const int32_t* table = ahead.b < 0 ? p.prefix_table : p.table + (int64_t)ahead.b * p.table_ld;
    const int cols = ahead.b < 0 ? p.prefix_cols : p.table_cols;
#pragma unroll
    for (int g = 0; g < S::kGran; ++g) {
      const int blk = (ahead.s * S::kTok + 16 * g) >> p.page_shift;
      id[g] = blk < cols ? table[blk] : -1;
    }
  };
  uint32_t have = 0;  // kGran bits per stage in flight, the oldest lowest
  auto fetch = [&](int slot, int place) {
    if (ahead.x >= n) {
      copies_done();
      return;
    }
    const int tiles = ahead.b < 0 ? p.prefix_row_tiles : p.own_row_tiles, j = tiles == 1 ? ahead.unit : ahead.unit / tiles;
    have |= fill_stage<D, INT8>(p, j, id, ahead.s * S::kTok, ahead.len, slots + slot * S::kStageBytes, lane) << (place * S::kGran);
    advance(p, ahead);
    if (ahead.x < n) look_up();
  };
  if (ahead.x < n) look_up();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) fetch(i, i);
  State<D> st;
  uint32_t qf[D / 16][4];
  float scale[2];
  int limit[2], low = 0, n_rows = 0, unit = 0;
  bool fresh = true;
  int slot = 0;
  while (at.x < n) {
    if (fresh) {
      // The unit's rows, and the tokens that each of this lane's two sees.
      const bool pre = at.b < 0;
      const int tiles = pre ? p.prefix_row_tiles : p.own_row_tiles, j = at.unit / tiles, row0 = (at.unit % tiles) * kRows;
      const int rows = pre ? p.rows : p.tokens * p.group;
      n_rows = min(kRows, rows - row0);
      unit = pre ? at.unit : p.h * p.prefix_row_tiles + at.b * p.h * p.own_row_tiles + at.unit;
      // Rows count their sight from the length as given, which may lie past the list's end.
      const int given = pre ? 0 : max(p.lens[at.b], 0);
      const __nv_bfloat16* src[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int x = min(row0 + r + 8 * k, rows - 1), g = x % p.group, bt = x / p.group, t = bt % p.tokens, b = pre ? bt / p.tokens : at.b;
        src[k] = r + 8 * k < n_rows ? p.q + b * p.q_sb + t * p.q_st + (int64_t)(j * p.group + g) * p.q_sh : nullptr;
        limit[k] = pre ? at.len : min(at.len, max(0, given - p.tokens + t + 1));
      }
      low = pre ? at.len : min(at.len, max(0, given - p.tokens + row0 / p.group + 1));
      load_queries<D, INT8>(qf, scale, src[0], src[1], c, p.scale_log2);
      st.clear();
      fresh = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    fetch(slot == 0 ? S::kStages - 1 : slot - 1, S::kStages - 1);
    const uint32_t has = have & ((1u << S::kGran) - 1);
    const int first = at.s * S::kTok;
    if (low < first + S::kTok || has != (1u << S::kGran) - 1)
      fold_stage<D, INT8, true>(st, qf, scale, slots_p + slot * S::kStageBytes, first, limit, has, lane);
    else
      fold_stage<D, INT8, false>(st, qf, scale, slots_p + slot * S::kStageBytes, first, limit, has, lane);
    have >>= S::kGran;
    slot = slot + 1 == S::kStages ? 0 : slot + 1;
    if (at.s + 1 == at.n || at.x + 1 >= n) {
      // The unit, or this warp's part of it, is done.
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        st.l[k] += __shfl_xor_sync(0xffffffffu, st.l[k], 1);
        st.l[k] += __shfl_xor_sync(0xffffffffu, st.l[k], 2);
        if (INT8) st.m[k] += kScaleShift, st.l[k] *= kScaleDown;  // o is in units of 2^(m + kScaleShift)
      }
      if (whole) break;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = r + 8 * k;
        if (row < n_rows) {
          const int64_t to = (int64_t)(w + unit) * p.slot_rows + row;
          if (c == 0) p.slot_ml[to] = make_float2(st.m[k], st.l[k]);
          // Tiles kVCh y .. kVCh y + kVCh - 1 of columns 2 c and 2 c + 1 are 2 kVCh consecutive channels.
#pragma unroll
          for (int x = 0; x < D / 8; x += 4)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float4*>(p.slot_o + to * D + S::channel(x, 2 * c + e)) =
                  make_float4(st.o[x][2 * k + e], st.o[x + 1][2 * k + e], st.o[x + 2][2 * k + e], st.o[x + 3][2 * k + e]);
        }
      }
      fresh = true;
    }
    advance(p, at);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!whole) return;
  // The four warps' states, in the ring, as one partial.
  __syncthreads();
  constexpr int kLd = D + 4;
  float* po = reinterpret_cast<float*>(ring);                          // [kWarps][kRows][kLd]
  float2* pml = reinterpret_cast<float2*>(po + kWarps * kRows * kLd);  // [kWarps][kRows]
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = warp * kRows + r + 8 * k;
    if (c == 0) pml[row] = make_float2(st.m[k], st.l[k]);
#pragma unroll
    for (int x = 0; x < D / 8; x += 4)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float4*>(po + row * kLd + S::channel(x, 2 * c + e)) =
            make_float4(st.o[x][2 * k + e], st.o[x + 1][2 * k + e], st.o[x + 2][2 * k + e], st.o[x + 3][2 * k + e]);
  }
  __syncthreads();
  for (int x = tid; x < n_rows * (D / 4); x += kThreads) {
    const int row = x / (D / 4), ch = x % (D / 4) * 4;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, pml[i * kRows + row].x);
    const float from = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float2 ml = pml[i * kRows + row];
      const float f = ex2(ml.x - from);
      const float4 v = *reinterpret_cast<const float4*>(po + (i * kRows + row) * kLd + ch);
      l += times_ex2(ml.y, ml.x - from);
      o.x += v.x * f, o.y += v.y * f, o.z += v.z * f, o.w += v.w * f;
    }
    const int64_t to = (int64_t)(w - warp + unit) * p.slot_rows + row;
    if (ch == 0) p.slot_ml[to] = make_float2(m, l);
    *reinterpret_cast<float4*>(p.slot_o + to * D + ch) = o;
  }
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kThreads, (Shape<D, INT8>::kCtas)) stream_kernel(const Params p) {
  extern __shared__ __align__(128) char ring[];
  // Behind the tiles' launch, which itself waited for what ran before it and only then let this one start,
  // the inputs are in place; otherwise this one has to wait for them.
  if (!p.tile_first) pdl_wait();
  pdl_release();
  stream<D, INT8>(p, ring);
  if (p.tile_first) pdl_wait();  // what comes after this launch may read the tiles' partials too
}

// A warp's sum over some partials of a row: lane `lane` has channels 4 (lane % (D / 4)) .., and where D is 64
// one of the warp's halves every second partial.
struct Sum {
  float m, l;
  float4 o;
};
__device__ __forceinline__ void fold(Sum& a, float m, float l, float4 o) {
  const float top = fmaxf(a.m, m), from = top == -INFINITY ? 0.0f : top, f = ex2(a.m - from), e = ex2(m - from);
  a.l = times_ex2(a.l, a.m - from) + times_ex2(l, m - from);
  a.m = top;
  a.o.x = a.o.x * f + o.x * e, a.o.y = a.o.y * f + o.y * e, a.o.z = a.o.z * f + o.z * e, a.o.w = a.o.w * f + o.w * e;
}

// The slots of one unit, stages [x, x + n) of the line in pieces of `piece`: a warp each up to the first CTA
// that the unit fills, then a slot per CTA (every kWarps), then a warp each again.
struct Slots {
  int first, heads, ctas, tails;
};
__device__ __forceinline__ Slots slots_of(int64_t x, int n, int64_t piece, int unit) {
  if (n <= 0) return {0, 0, 0, 0};
  const int w0 = (int)quotient(x, piece), w1 = (int)quotient(x + n - 1, piece);
  const int c0 = (int)quotient(x + kWarps * piece - 1, kWarps * piece), c1 = (int)quotient(x + n, kWarps * piece);  // CTAs filled: c0 .. c1 - 1
  if (c1 <= c0) return {w0 + unit, w1 - w0 + 1, 0, 0};
  return {w0 + unit, c0 * kWarps - w0, c1 - c0, w1 + 1 - c1 * kWarps};
}

// The partials of every row: `team` warps (1, 2 or 4) per row of (sequence, KV head), kWarps / team rows a
// CTA. Grid: (rows of a sequence and head by CTAs, head, sequence).
template <int D>
__global__ void __launch_bounds__(kThreads, 4) combine_kernel(const Params p, int team) {
  __shared__ Sum sums[kWarps][32];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int j = blockIdx.y, b = blockIdx.z, unit_rows = p.tokens * p.group;
  const int row = blockIdx.x * (kWarps / team) + warp / team, part = warp % team;
  const bool live = row < unit_rows;
  // The lengths are this call's input, in place since before the launches in front of this one began
  // (where there are none, they have to be waited for).
  const bool alone = p.n_warps == 0 && p.n_splits == 0;
  if (alone) pdl_wait();
  Slots own = {0, 0, 0, 0}, pre = {0, 0, 0, 0};  // the row's own unit, and the prefix's where that is streamed
  if (p.n_warps > 0) {
    const Line line = sum_line(p, lane);
    const int64_t piece = piece_length(p, line);
    const int n = stages_of(p, p.lens[b]), slice = b / slice_of(p);
    int64_t before = __shfl_sync(0xffffffffu, line.before, slice);
    for (int i = slice * slice_of(p); i < b; ++i) before += length_of(stages_of(p, p.lens[i]));
    int unit = j * p.own_row_tiles + row / kRows;
    own = slots_of(prefix_length(p) + before * p.h * p.own_row_tiles + (int64_t)unit * length_of(n), n, piece,
                   p.h * p.prefix_row_tiles + b * p.h * p.own_row_tiles + unit);
    unit = j * p.prefix_row_tiles + (b * unit_rows + row) / kRows;
    pre = slots_of((int64_t)unit * length_of(p.prefix_stages), p.prefix_stages, piece, unit);
  }
  if (!alone) pdl_wait();
  pdl_release();
  // All partials of the row as one list: the tiled prefix's, the own ones, the streamed prefix's. Partial
  // rows are numbered through the workspace, the tiled ones first.
  const int64_t tiled = (int64_t)p.n_splits * p.h * p.rows;
  auto row_of = [&](int i) -> int64_t {
    if (i < p.n_splits) return ((int64_t)i * p.h + j) * p.rows + (int64_t)b * unit_rows + row;
    i -= p.n_splits;
    const int n_own = own.heads + own.ctas + own.tails;
    const bool mine = i < n_own;
    const Slots x = mine ? own : pre;
    if (!mine) i -= n_own;
    if (i >= x.heads) i = i < x.heads + x.ctas ? x.heads + (i - x.heads) * kWarps : i + x.ctas * (kWarps - 1);
    return tiled + (int64_t)(x.first + i) * p.slot_rows + (mine ? row : b * unit_rows + row) % kRows;
  };
  const int n_parts = p.n_splits + own.heads + own.ctas + own.tails + pre.heads + pre.ctas + pre.tails;
  constexpr int kLanes = D / 4, kTogether = 32 / kLanes;  // partials side by side in the warp
  const int ch = 4 * (lane % kLanes), side = lane / kLanes;
  Sum a = {-INFINITY, 0.0f, make_float4(0.f, 0.f, 0.f, 0.f)};
  // 32 at a time: references and sums, one per lane, then the outputs with weights that are known.
  for (int base = part; live && base < n_parts; base += 32 * team) {
    const int mine = base + lane * team;
    const int64_t from_row = row_of(min(mine, n_parts - 1));
    float2 x = make_float2(-INFINITY, 0.0f);
    if (mine < n_parts) x = p.tile_ml[from_row];
    const int count = min(32, (n_parts - base + team - 1) / team);
    float top = x.x;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    top = fmaxf(top, a.m);
    const float from = top == -INFINITY ? 0.0f : top, f = ex2(a.m - from), by = ex2(x.x - from);
    float l = times_ex2(x.y, x.x - from);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    a.l = times_ex2(a.l, a.m - from) + l;
    a.m = top;
    a.o.x *= f, a.o.y *= f, a.o.z *= f, a.o.w *= f;
#pragma unroll 1
    for (int i = 0; i < count; i += 8 * kTogether) {
      float4 v[8];
      float weight[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int which = i + k * kTogether + side;
        const int64_t at = __shfl_sync(0xffffffffu, from_row, which & 31);
        weight[k] = __shfl_sync(0xffffffffu, by, which & 31);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (which < count) v[k] = *reinterpret_cast<const float4*>(p.tile_o + at * D + ch);
        else weight[k] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        a.o.x += v[k].x * weight[k], a.o.y += v[k].y * weight[k], a.o.z += v[k].z * weight[k], a.o.w += v[k].w * weight[k];
    }
  }
  if constexpr (D == 64) {  // the two halves of the warp share m and l and have half of the outputs each
    a.o.x += __shfl_xor_sync(0xffffffffu, a.o.x, 16), a.o.y += __shfl_xor_sync(0xffffffffu, a.o.y, 16);
    a.o.z += __shfl_xor_sync(0xffffffffu, a.o.z, 16), a.o.w += __shfl_xor_sync(0xffffffffu, a.o.w, 16);
  }
  if (team > 1) {
    sums[warp][lane] = a;
    __syncthreads();
    if (part == 0)
      for (int i = 1; i < team; ++i) {
        const Sum x = sums[warp + i][lane];
        fold(a, x.m, x.l, x.o);
      }
  }
  if (!live || part != 0 || lane >= D / 4) return;
  const float inv = a.l > 0.0f ? 1.0f / a.l : a.l == 0.0f ? 0.0f : a.l;  // no key at all: 0; a NaN stays one
  const int64_t at = ((int64_t)b * p.tokens + row / p.group) * (p.h * p.group) + j * p.group + row % p.group;
  const float4 o = make_float4(a.o.x * inv, a.o.y * inv, a.o.z * inv, a.o.w * inv);
  if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at * D + 4 * lane) = o;
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at * D + 4 * lane) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
  if (lane == 0) p.lse[at] = a.l == 0.0f ? -INFINITY : (a.m + log2f(a.l)) * kLn2;
}

template <int D, bool INT8>
cudaError_t launch_stream(const Params& p, cudaStream_t st) {
  using S = Shape<D, INT8>;
  auto k = stream_kernel<D, INT8>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, S::kRing, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(k, dim3(p.n_warps / kWarps), dim3(kThreads), S::kRing, st, 0, p);
}

// Batches of at most kRows rows per KV head stream the prefix: one row tile. Beyond, the stream copies the prefix once
// per row tile, and the tensor cores' tile of 128 rows is empty for the most part below. Both sides, in us, tiles and
// stream, 8 KV heads: bf16, d 128, a prefix of 8,192: 16.7 and 16.1 at 8 rows, 17.0 and 16.9 at 16, 17.6 and 24.0 at 20;
// of 32,768: 36.3 and 37.7 at 16, 36.4 and 62.6 at 20. int8, d 128: 20.0 and 16.7 at 16 rows of 8,192, 21.1 and 20.2 at 20;
// 37.2 and 30.2, 37.7 and 45.6 of 32,768. Prefixes of 1,024 cost 12 and 10 us on either side.
bool streams(int64_t rows) { return rows <= kRows; }

// How a call is cut up: Params' numbers that follow from the shapes alone, and the workspace they take.
struct Plan {
  int n_splits, prefix_stages, prefix_row_tiles, own_row_tiles, n_warps, slot_rows;
  size_t tile_floats, slot_count;
  size_t bytes(int d, int64_t rows, int h) const {
    return (size_t)n_splits * h * rows * ((size_t)d * 4 + 8) + slot_count * slot_rows * ((size_t)d * 4 + 8);
  }
};

Plan plan_of(int batch, int tokens, int hq, int h, int d, int64_t prefix_len, int kind, int64_t own_reach) {
  Plan x = {};
  const int64_t unit = (int64_t)tokens * (hq / h), rows = batch * unit;
  const int shift = stage_shift_of(d);
  const bool stream_prefix = prefix_len > 0 && streams(rows);
  if (prefix_len > 0 && !stream_prefix) x.n_splits = tile_splits((int)rows, h, prefix_len);
  x.own_row_tiles = (int)((unit + kRows - 1) / kRows);
  if (stream_prefix) {
    x.prefix_stages = (int)((prefix_len + (1 << shift) - 1) >> shift);
    x.prefix_row_tiles = (int)((rows + kRows - 1) / kRows);
  }
  // Warps for as many stages as there can be, up to all that the GPU holds at once.
  const int64_t most = (int64_t)x.prefix_stages * h * x.prefix_row_tiles + ((own_reach + (1 << shift) - 1) >> shift) * batch * h * x.own_row_tiles;
  const int64_t room = (int64_t)kNumSMs * (kind == LKV_CACHE_INT8 ? 3 : 2) * kWarps;
  int64_t warps = (most + kMinStages - 1) / kMinStages;
  warps = warps < room ? (warps + kWarps - 1) / kWarps * kWarps : room;
  x.n_warps = (int)warps;
  x.slot_rows = (int)(stream_prefix && rows > unit ? (rows < kRows ? rows : kRows) : (unit < kRows ? unit : kRows));
  x.slot_count = x.n_warps == 0 ? 0 : (size_t)x.n_warps + (size_t)h * x.prefix_row_tiles + (size_t)batch * h * x.own_row_tiles;
  return x;
}

}  // namespace
}  // namespace prefix
}  // namespace lkv

using namespace lkv;
using namespace lkv::prefix;

extern "C" {

size_t lkv_prefix_attention_workspace(int batch, int tokens, int hq, int h, int d, int64_t prefix_len, int kind, int64_t own_reach) {
  if (batch < 1 || tokens < 1 || h < 1 || hq < h || prefix_len < 0 || own_reach < 0 || (d != 64 && d != 128)) return 0;
  return plan_of(batch, tokens, hq, h, d, prefix_len, kind, own_reach).bytes(d, (int64_t)batch * tokens * (hq / h), h);
}

int lkv_prefix_attention(const lkv_prefix_args* a, void* stream) {
  static const char* who = "lkv_prefix_attention";
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (a->kind != LKV_CACHE_MODEL && a->kind != LKV_CACHE_INT8) return fail(LKV_ERR_ARG, "%s: bad cache kind %d", who, a->kind);
  if (a->dtype != LKV_BF16) return fail(LKV_ERR_ARG, "%s: bad dtype %d (queries and model pages are bfloat16)", who, a->dtype);
  if (!dtype_ok(a->out_dtype)) return fail(LKV_ERR_ARG, "%s: bad dtype %d of the output", who, a->out_dtype);
  if (a->d != 64 && a->d != 128) return fail(LKV_ERR_ARG, "%s: head_dim %d (64 or 128)", who, a->d);
  if (a->bs != 16 && a->bs != 32 && a->bs != 64 && a->bs != 128) return fail(LKV_ERR_ARG, "%s: pages of %d tokens (16, 32, 64 or 128)", who, a->bs);
  if (a->h < 1 || a->hq < 1 || a->hq % a->h != 0) return fail(LKV_ERR_ARG, "%s: %d query heads do not group over %d KV heads", who, a->hq, a->h);
  if (a->batch < 0 || a->tokens < 0 || a->table_cols < 0 || a->prefix_cols < 0 || a->n_pages < 0 || a->n_pages > INT32_MAX || a->prefix_len < 0 ||
      (a->batch > 1 && a->table_ld < a->table_cols))
    return fail(LKV_ERR_ARG, "%s: bad shape (batch %d, tokens %d, tables of %d and %d columns, pages %lld, prefix %lld)", who, a->batch, a->tokens,
                a->table_cols, a->prefix_cols, (long long)a->n_pages, (long long)a->prefix_len);
  if (a->prefix_len > (int64_t)a->prefix_cols * a->bs)
    return fail(LKV_ERR_ARG, "%s: a prefix of %lld tokens in %d pages of %d", who, (long long)a->prefix_len, a->prefix_cols, a->bs);
  if (a->prefix_len > (1 << 30) || (int64_t)a->table_cols * a->bs > (1 << 30)) return fail(LKV_ERR_ARG, "%s: more than 2^30 tokens of one list", who);
  if (a->batch == 0 || a->tokens == 0) return LKV_OK;
  const int group = a->hq / a->h;
  const int64_t rows = (int64_t)a->batch * a->tokens * group;
  if (a->batch > 65535 || a->h > 65535 || rows > (1 << 24)) return fail(LKV_ERR_ARG, "%s: a batch of %d with %lld rows per KV head", who, a->batch, (long long)rows);
  const int64_t own_units = (int64_t)a->batch * a->h * (((int64_t)a->tokens * group + kRows - 1) / kRows);
  if (own_units > (1 << 30)) return fail(LKV_ERR_ARG, "%s: a batch of %d with %lld row tiles", who, a->batch, (long long)own_units);
  if (a->q == nullptr || a->out == nullptr || a->lse == nullptr || a->lens == nullptr || a->pages == nullptr ||
      (a->kind == LKV_CACHE_INT8 && a->scales == nullptr) || (a->table_cols > 0 && a->table == nullptr) || (a->prefix_len > 0 && a->prefix_table == nullptr))
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(a->q, 16) || !aligned(a->pages, 16) || !aligned(a->scales, 8) || !aligned(a->out, 16) || a->q_sb % 8 || a->q_st % 8 || a->q_sh % 8)
    return fail(LKV_ERR_PTR, "%s: queries (their strides too), pages and the output must be 16-byte aligned", who);
  Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
  p.pages = a->pages;
  p.scales = a->scales;
  p.n_pages = (int)a->n_pages;
  p.page_shift = a->bs == 16 ? 4 : a->bs == 32 ? 5 : a->bs == 64 ? 6 : 7;
  p.batch = a->batch, p.tokens = a->tokens, p.h = a->h, p.group = group;
  p.table = a->table;
  p.table_ld = a->table_ld;
  p.table_cols = a->table_cols;
  p.lens = a->lens;
  p.prefix_table = a->prefix_table;
  p.prefix_cols = a->prefix_cols;
  p.prefix_len = (int)a->prefix_len;
  p.scale_log2 = a->scale * kLog2e;
  p.rows = (int)rows;
  const int64_t reach = (int64_t)a->table_cols * a->bs;
  const Plan plan = plan_of(a->batch, a->tokens, a->hq, a->h, a->d, a->prefix_len, a->kind, reach);
  p.n_splits = plan.n_splits;
  p.stage_shift = stage_shift_of(a->d);
  p.prefix_stages = plan.prefix_stages;
  p.prefix_row_tiles = plan.prefix_row_tiles;
  p.own_row_tiles = plan.own_row_tiles;
  p.n_warps = plan.n_warps;
  p.slot_rows = plan.slot_rows;
  p.out = a->out;
  p.out_f32 = a->out_dtype == LKV_F32;
  p.lse = a->lse;
  const size_t need = plan.bytes(a->d, rows, a->h);
  if (need > 0) {
    if (a->workspace_bytes < need) return fail(LKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, need);
    if (a->workspace == nullptr || !aligned(a->workspace, 16)) return fail(LKV_ERR_PTR, "%s: workspace must be 16-byte aligned", who);
    const size_t tiled = (size_t)p.n_splits * a->h * rows, slots = plan.slot_count * plan.slot_rows;
    p.tile_o = static_cast<float*>(a->workspace);
    p.slot_o = p.tile_o + tiled * a->d;
    p.tile_ml = reinterpret_cast<float2*>(p.slot_o + slots * a->d);
    p.slot_ml = p.tile_ml + tiled;
  }
  cudaStream_t st = as_stream(stream);
  const bool int8 = a->kind == LKV_CACHE_INT8, wide = a->d == 128;
  cudaError_t e = cudaSuccess;
  if (p.n_splits > 0) {
    if (int rc = run_tiles(p, a->d, int8, st)) return rc;
    p.tile_first = 1;
  }
  if (p.n_warps > 0) {
    e = wide ? (int8 ? launch_stream<128, true>(p, st) : launch_stream<128, false>(p, st))
             : (int8 ? launch_stream<64, true>(p, st) : launch_stream<64, false>(p, st));
    if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s (stream): %s", who, cudaGetErrorString(e));
  }
  // Several warps to a row where it has many partials.
  const int parts = p.n_splits + (p.prefix_stages > 0 ? p.n_warps / (kWarps * a->h) : 0), team = parts > 16 ? 4 : parts > 8 ? 2 : 1;
  const int unit = a->tokens * group, per = kWarps / team;
  const dim3 grid((unit + per - 1) / per, a->h, a->batch);
  e = wide ? launch_pdl(combine_kernel<128>, grid, dim3(kThreads), 0, st, 0, p, team) : launch_pdl(combine_kernel<64>, grid, dim3(kThreads), 0, st, 0, p, team);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s (combine): %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
