// Attention of a batch that shares a prefix: every query attends the prefix's tokens and its own
// sequence's, and the prefix's pages are read once for the whole batch.
//
// The query rows of KV head j are (b, t, g): sequence, position among the step's tokens, query head of
// the group. Row (b, t, g) sees the prefix [0, prefix_len) and own tokens 0 .. lens[b] - tokens + t. Two
// softmaxes over disjoint key sets merge exactly by their maxima and sums, so the work is two launches:
//   1. the prefix: all rows of the batch against chunks of the prefix, a partial (m, l, o) per chunk;
//   2. the sequences' own tokens, one cluster of CTAs per (sequence, KV head, row tile), which then
//      folds the prefix's partials in and writes the output.
// The second launch starts under the first (programmatic dependent launch) and waits for it only before
// it folds.
//
// prefix_tile.cu does the first launch. stream_kernel does the second, and the first where the batch has
// few rows: each warp takes a
// tile of 16 rows through its share of the tokens with mma.sync.m16n8k16 (bf16 operands, float32
// accumulators). A lane copies by cp.async exactly the bytes that it will hold as mma fragments, into
// slots of shared memory of its own, so the pipeline needs no barrier and no bank conflicts arise; the
// channels are permuted so that a fragment's elements are 16 contiguous bytes of a row (a dot product
// does not mind, and the output's permutation ends in contiguous runs again). int8 codes become bf16
// exactly in registers; a key's scale multiplies its column of scores, a value's its column of
// probabilities, both in float32. Probabilities are rounded to bf16 for the second product (2^-9
// relative, unbiased over the keys, and below the rounding of a bf16 output).
#include <cooperative_groups.h>

#include "prefix.cuh"

namespace lkv {
namespace prefix {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;  // rows of an mma tile
constexpr int kMaxCluster = 8;

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Asynchronous copy of N bytes, or N zeros where !there (nothing is read then).
template <int N>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void* src, bool there) {
  const int n = there ? N : 0;
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}

constexpr int stage_tokens(int d) { return d == 128 ? 16 : 32; }

// Geometry of the stream for one head dimension and cache type.
template <int D, bool INT8>
struct Shape {
  static constexpr int kElt = INT8 ? 1 : 2;
  static constexpr int kTok = stage_tokens(D);                 // tokens per stage
  static constexpr int kGran = kTok / 16;                      // 16-token granules per stage
  static constexpr int kKLoads = D * kElt / 64;                // 16-byte loads per lane and 8 keys (4 lanes a row)
  static constexpr int kVBytes = D * kElt / 8 >= 16 ? 16 : 8;  // bytes per lane and load of a value row (8 lanes a row)
  static constexpr int kVLoads = D * kElt / 8 / kVBytes;
  static constexpr int kKBytes = 2 * kKLoads * 16;             // per lane and granule
  static constexpr int kVAll = 4 * kVLoads * kVBytes;
  static constexpr int kSBytes = INT8 ? 32 : 0;                // the scales of 4 tokens' keys and values
  static constexpr int kGranBytes = (kKBytes + kVAll + kSBytes) * 32;
  static constexpr int kStageBytes = kGran * kGranBytes;
  static constexpr int kStages = INT8 ? 4 : 3;                 // 72 to 96 KB of copies per CTA, two CTAs an SM
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kVCh = kVBytes / kElt;                  // channels per value load
  // The channel of column n of the i-th output tile.
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

// The A fragments of a 16-row tile of queries, channels permuted as Shape's keys are. Rows without a
// pointer are zero.
template <int D, bool INT8>
__device__ __forceinline__ void load_queries(uint32_t (&qf)[D / 16][4], const __nv_bfloat16* lo, const __nv_bfloat16* hi, int c) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const __nv_bfloat16* row = half ? hi : lo;
    if constexpr (INT8) {
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (row != nullptr) {
          const uint4* p = reinterpret_cast<const uint4*>(row + 64 * x + 16 * c);
          w[0] = p[0], w[1] = p[1];
        }
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // k-step 4x + i: channels (0, 2) then (1, 3) of four
          qf[4 * x + i][half] = __byte_perm(u[2 * i], u[2 * i + 1], 0x5410);
          qf[4 * x + i][2 + half] = __byte_perm(u[2 * i], u[2 * i + 1], 0x7632);
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

// Starts the copies of one stage: tokens first .. first + kTok - 1 of the list, those at or past `end`
// and those without a page as zeros. `have` gets a bit per granule that has a page.
template <int D, bool INT8>
__device__ __forceinline__ uint32_t fill_stage(const Params& p, int j, const int (&page)[Shape<D, INT8>::kGran], int first, int end, uint32_t slot, int lane) {
  using S = Shape<D, INT8>;
  const int r = lane / 4, c = lane % 4;
  const int bs = 1 << p.page_shift;
  uint32_t have = 0;
#pragma unroll
  for (int g = 0; g < S::kGran; ++g) {
    const int tok = first + 16 * g;
    const bool ok = page[g] >= 0;
    have |= (ok ? 1u : 0u) << g;
    const int64_t krow = (((int64_t)(ok ? page[g] : 0) * p.h + j) * 2) * bs + (tok & (bs - 1));
    const char* kp = static_cast<const char*>(p.pages) + krow * (D * S::kElt);
    const char* vp = kp + (int64_t)bs * (D * S::kElt);
    uint32_t dst = slot + g * S::kGranBytes + lane * 16;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int x = 0; x < S::kKLoads; ++x, dst += 512) {
        const int t = 8 * nt + r;
        copy_or_zero<16>(dst, kp + t * (D * S::kElt) + 64 * x + 16 * c, ok && tok + t < end);
      }
    if constexpr (S::kVBytes == 8) dst = slot + g * S::kGranBytes + S::kKBytes * 32 + lane * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 2 * c + (i & 1) + 8 * (i >> 1);
#pragma unroll
      for (int y = 0; y < S::kVLoads; ++y, dst += S::kVBytes * 32)
        copy_or_zero<S::kVBytes>(dst, vp + t * (D * S::kElt) + (8 * y + r) * S::kVBytes, ok && tok + t < end);
    }
    if constexpr (INT8) {
      dst = slot + g * S::kGranBytes + (S::kKBytes + S::kVAll) * 32 + lane * 8;
      const float* sp = p.scales + krow + 2 * c;  // two tokens' key scales, then (bs further) their value scales
#pragma unroll
      for (int i = 0; i < 4; ++i, dst += 256) {
        // Past `end` inside a page the scales are read all the same: they exist, and their columns are masked.
        copy_or_zero<8>(dst, sp + (i >> 1) * bs + 8 * (i & 1), ok);
      }
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  return have;
}

// One stage's tokens folded into the warp's state. limit[0/1]: the tokens that rows r and r + 8 see.
template <int D, bool INT8>
__device__ __forceinline__ void fold_stage(State<D>& st, const uint32_t (&qf)[D / 16][4], const char* slot, int first, const int (&limit)[2], int low,
                                           uint32_t have, float scale_log2, int lane) {
  using S = Shape<D, INT8>;
  const int c = lane % 4;
  float s[2 * S::kGran][4];
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
          for (int k = 0; k < 4; ++k) mma16816(x, qf[4 * i + k], codes_to_bf16(u[k]), codes_to_bf16(u[k] >> 8));
        } else {
          mma16816(x, qf[2 * i], w.x, w.y);
          mma16816(x, qf[2 * i + 1], w.z, w.w);
        }
      }
      if constexpr (INT8) {
        const float2 ks = *reinterpret_cast<const float2*>(slot + g * S::kGranBytes + (S::kKBytes + S::kVAll) * 32 + nt * 256 + lane * 8);
        x[0] *= ks.x * scale_log2, x[1] *= ks.y * scale_log2;
        x[2] *= ks.x * scale_log2, x[3] *= ks.y * scale_log2;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= scale_log2;
      }
    }
  }
  // The mask, where a row's sight ends inside this stage or a page is missing (the same for the warp).
  const bool masked = low < first + S::kTok || have != (1u << S::kGran) - 1;
  if (masked) {
#pragma unroll
    for (int n = 0; n < 2 * S::kGran; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = first + 8 * n + 2 * c + (e & 1);
        if (tok >= limit[e >> 1] || !((have >> (n / 2)) & 1)) s[n][e] = -INFINITY;
      }
  }
  float top[2] = {st.m[0], st.m[1]};
#pragma unroll
  for (int n = 0; n < 2 * S::kGran; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
  }
  if (__any_sync(0xffffffffu, top[0] > st.m[0] || top[1] > st.m[1])) {
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[i] = top[i] > st.m[i] ? ex2(st.m[i] - top[i]) : 1.0f;  // 0 where nothing was seen before
      st.l[i] *= f[i];
      st.m[i] = top[i];
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) st.o[i][0] *= f[0], st.o[i][1] *= f[0], st.o[i][2] *= f[1], st.o[i][3] *= f[1];
  }
  // A row that has seen nothing keeps m = -inf: its weights come from a maximum of 0, ex2(-inf) = 0.
  const float m0 = st.m[0] == -INFINITY ? 0.0f : st.m[0], m1 = st.m[1] == -INFINITY ? 0.0f : st.m[1];
#pragma unroll
  for (int n = 0; n < 2 * S::kGran; ++n) {
    s[n][0] = ex2(s[n][0] - m0), s[n][1] = ex2(s[n][1] - m0);
    s[n][2] = ex2(s[n][2] - m1), s[n][3] = ex2(s[n][3] - m1);
    st.l[0] += s[n][0] + s[n][1];
    st.l[1] += s[n][2] + s[n][3];
    if constexpr (INT8) {
      const float2 vs = *reinterpret_cast<const float2*>(slot + (n / 2) * S::kGranBytes + (S::kKBytes + S::kVAll) * 32 + (2 + n % 2) * 256 + lane * 8);
      // A weight of zero stays zero whatever the scale (a masked token's may be NaN).
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = s[n][e] == 0.0f ? 0.0f : s[n][e] * ((e & 1) ? vs.y : vs.x);
    }
  }
#pragma unroll
  for (int g = 0; g < S::kGran; ++g) {
    const char* base = slot + g * S::kGranBytes + S::kKBytes * 32 + lane * S::kVBytes;
    const uint32_t a[4] = {pack_bf16(s[2 * g][0], s[2 * g][1]), pack_bf16(s[2 * g][2], s[2 * g][3]), pack_bf16(s[2 * g + 1][0], s[2 * g + 1][1]),
                           pack_bf16(s[2 * g + 1][2], s[2 * g + 1][3])};
#pragma unroll
    for (int y = 0; y < S::kVLoads; ++y) {
      constexpr int kWords = S::kVBytes / 4;
      uint32_t w[4][kWords];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const char* src = base + (t * S::kVLoads + y) * (S::kVBytes * 32);
        if constexpr (kWords == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(src);
          w[t][0] = x.x, w[t][1] = x.y, w[t][2] = x.z, w[t][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(src);
          w[t][0] = x.x, w[t][1] = x.y;
        }
      }
      if constexpr (!INT8) {
        if (masked) {
          // 0 x infinity is NaN: a token that some rows do not see must not reach them through a value
          // that is not finite. Such a stage (the step's own last tokens only) is summed without mma.
          bool odd = false;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < kWords; ++i) odd |= (w[t][i] & 0x7f80u) == 0x7f80u || (w[t][i] & 0x7f800000u) == 0x7f800000u;
          if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
            for (int t = 0; t < 16; ++t) {
              const int e = t & 1, owner = (lane & ~3) | ((t & 7) >> 1);  // the lane that holds this token's weights for rows r, r + 8
              const float x0 = t < 8 ? (e ? s[2 * g][1] : s[2 * g][0]) : (e ? s[2 * g + 1][1] : s[2 * g + 1][0]);
              const float x1 = t < 8 ? (e ? s[2 * g][3] : s[2 * g][2]) : (e ? s[2 * g + 1][3] : s[2 * g + 1][2]);
              const float p0 = bf16_round(__shfl_sync(0xffffffffu, x0, owner)), p1 = bf16_round(__shfl_sync(0xffffffffu, x1, owner));
              const int slot_t = e + 2 * (t >> 3);
#pragma unroll
              for (int i = 0; i < S::kVCh; ++i) {
                // Column n of output tile (y, i) is channel(., n), which lane (n, owner's c) copied.
                const char* src = slot + g * S::kGranBytes + S::kKBytes * 32 + (slot_t * S::kVLoads + y) * (S::kVBytes * 32);
                const int c2 = (t & 7) >> 1;
                const __nv_bfloat16 va = *reinterpret_cast<const __nv_bfloat16*>(src + ((2 * c) * 4 + c2) * S::kVBytes + 2 * i);
                const __nv_bfloat16 vb = *reinterpret_cast<const __nv_bfloat16*>(src + ((2 * c + 1) * 4 + c2) * S::kVBytes + 2 * i);
                float* o = st.o[S::kVCh * y + i];
                if (p0 != 0.0f) o[0] += p0 * __bfloat162float(va), o[1] += p0 * __bfloat162float(vb);
                if (p1 != 0.0f) o[2] += p1 * __bfloat162float(va), o[3] += p1 * __bfloat162float(vb);
              }
            }
            __syncwarp();  // these slots are other lanes' to fill again
            continue;
          }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          mma16816(st.o[S::kVCh * y + 2 * i], a, __byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x5410));
          mma16816(st.o[S::kVCh * y + 2 * i + 1], a, __byte_perm(w[0][i], w[1][i], 0x7632), __byte_perm(w[2][i], w[3][i], 0x7632));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          // Bytes (0, 1) of two tokens, then (2, 3): the even bytes of a word are two tokens' same channel.
          const uint32_t lo01 = __byte_perm(w[0][i], w[1][i], 0x5410), hi01 = __byte_perm(w[0][i], w[1][i], 0x7632);
          const uint32_t lo23 = __byte_perm(w[2][i], w[3][i], 0x5410), hi23 = __byte_perm(w[2][i], w[3][i], 0x7632);
          float(*o)[4] = &st.o[S::kVCh * y + 4 * i];
          mma16816(o[0], a, codes_to_bf16(lo01), codes_to_bf16(lo23));
          mma16816(o[1], a, codes_to_bf16(lo01 >> 8), codes_to_bf16(lo23 >> 8));
          mma16816(o[2], a, codes_to_bf16(hi01), codes_to_bf16(hi23));
          mma16816(o[3], a, codes_to_bf16(hi01 >> 8), codes_to_bf16(hi23 >> 8));
        }
      }
    }
  }
}

// PREFIX: grid (row tile, split, head); the tokens are the prefix's, the rows the whole batch's.
// Otherwise: grid (row tile and, within its cluster of n_ctas, split; head; sequence); own tokens.
template <int D, bool INT8, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 2) stream_kernel(const Params p, int n_ctas) {
  using S = Shape<D, INT8>;
  extern __shared__ __align__(128) char ring[];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, r = lane / 4, c = lane % 4;
  // Launched after the prefix's kernel, which itself waited for what ran before it and only then let
  // this one start, so the inputs are in place; alone, this one has to wait.
  if (PREFIX || p.n_splits == 0) pdl_wait();
  int tile, split, j, b = 0;
  if constexpr (PREFIX) {
    tile = blockIdx.x, split = blockIdx.y, j = blockIdx.z;
    pdl_release();
  } else {
    split = blockIdx.x % n_ctas, tile = blockIdx.x / n_ctas, j = blockIdx.y, b = blockIdx.z;
  }
  const int unit_rows = PREFIX ? p.rows : p.tokens * p.group;
  const int row0 = tile * kRows, n_rows = min(kRows, unit_rows - row0);
  // Tokens of the list that each of this lane's rows sees, the most that any row of the tile sees and the least.
  const int32_t* table = PREFIX ? p.prefix_table : p.table + (int64_t)b * p.table_ld;
  const int cols = PREFIX ? p.prefix_cols : p.table_cols;
  int limit[2], end, low;
  if constexpr (PREFIX) {
    limit[0] = limit[1] = low = end = p.prefix_len;
  } else {
    const int64_t room = (int64_t)p.table_cols << p.page_shift;
    const int len = (int)min((int64_t)max(p.lens[b], 0), room);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = min(row0 + r + 8 * i, unit_rows - 1) / p.group;
      limit[i] = max(0, len - p.tokens + t + 1);
    }
    low = max(0, len - p.tokens + row0 / p.group + 1);
    end = max(0, len - p.tokens + (row0 + n_rows - 1) / p.group + 1);
  }
  // This CTA's stages; its warps take them in turn.
  const int n_stages = (end + S::kTok - 1) / S::kTok;
  const int share = max((n_stages + n_ctas - 1) / n_ctas, kWarps);
  const int s_lo = min(split * share, n_stages), s_hi = min(s_lo + share, n_stages);
  uint32_t qf[D / 16][4];
  {
    const __nv_bfloat16* at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r + 8 * i;
      at[i] = nullptr;
      if (row < n_rows) {
        const int x = row0 + row, g = x % p.group, bt = x / p.group;
        const int t = PREFIX ? bt % p.tokens : bt, bb = PREFIX ? bt / p.tokens : b;
        at[i] = p.q + bb * p.q_sb + t * p.q_st + (int64_t)(j * p.group + g) * p.q_sh;
      }
    }
    load_queries<D, INT8>(qf, at[0], at[1], c);
  }
  State<D> st;
  st.clear();
  {
    const char* mine = ring + warp * (S::kStages * S::kStageBytes);
    const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
    // Pages are looked up one stage before their copies start.
    int page[S::kGran];
    auto look_up = [&](int s) {
#pragma unroll
      for (int g = 0; g < S::kGran; ++g) page[g] = s < s_hi && s * S::kTok + 16 * g < end ? page_at(table, cols, p.n_pages, s * S::kTok + 16 * g, p.page_shift) : -1;
    };
    uint32_t have[S::kStages];
    int s = s_lo + warp;
    look_up(s);
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
      have[i] = 0;
      if (s + i * kWarps < s_hi) have[i] = fill_stage<D, INT8>(p, j, page, (s + i * kWarps) * S::kTok, end, mine_u + i * S::kStageBytes, lane);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      look_up(s + (i + 1) * kWarps);
    }
    have[S::kStages - 1] = 0;
    int slot = 0;
    for (; s < s_hi; s += kWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      const int ahead = s + (S::kStages - 1) * kWarps, to = slot == 0 ? S::kStages - 1 : slot - 1;
      uint32_t got = 0;
      if (ahead < s_hi) got = fill_stage<D, INT8>(p, j, page, ahead * S::kTok, end, mine_u + to * S::kStageBytes, lane);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      look_up(ahead + kWarps);
      fold_stage<D, INT8>(st, qf, mine + slot * S::kStageBytes, s * S::kTok, limit, low, have[0], p.scale_log2, lane);
#pragma unroll
      for (int i = 0; i + 1 < S::kStages - 1; ++i) have[i] = have[i + 1];
      have[S::kStages - 2] = got;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // The warps' states, then one per CTA: rows of D + 4 floats (o), and (m, l).
  __syncthreads();
  constexpr int kLd = D + 4;
  float* po = reinterpret_cast<float*>(ring);                        // [kWarps][16][kLd]
  float2* pml = reinterpret_cast<float2*>(po + kWarps * kRows * kLd);  // [kWarps][16]
  float2* cml = pml + kWarps * kRows;                                 // [16], the CTA's
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
    if (c == 0) pml[warp * kRows + r + 8 * i] = make_float2(st.m[i], st.l[i]);
  }
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) po[(warp * kRows + r + 8 * (e >> 1)) * kLd + S::channel(i, 2 * c + (e & 1))] = st.o[i][e];
  __syncthreads();
  constexpr int kPer = D / 4;  // threads per row, a float4 each
  for (int x = tid; x < n_rows * kPer; x += kThreads) {
    const int row = x / kPer, ch = (x % kPer) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, pml[w * kRows + row].x);
    const float from = m == -INFINITY ? 0.0f : m;  // nothing seen: every weight below is 0 (or NaN, which stays)
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = pml[w * kRows + row];
      const float f = ex2(ml.x - from);
      const float4 v = *reinterpret_cast<const float4*>(po + (w * kRows + row) * kLd + ch);
      l += ml.y * f;
      o.x += v.x * f, o.y += v.y * f, o.z += v.z * f, o.w += v.w * f;
    }
    if constexpr (PREFIX) {
      const int64_t at = ((int64_t)split * p.h + j) * p.rows + row0 + row;
      *reinterpret_cast<float4*>(p.part_o + at * D + ch) = o;
      if (ch == 0) p.part_ml[at] = make_float2(m, l);
    } else {
      *reinterpret_cast<float4*>(po + row * kLd + ch) = o;  // warp 0's place: only this thread reads it
      if (ch == 0) cml[row] = make_float2(m, l);
    }
  }
  if constexpr (!PREFIX) {
    cg::cluster_group cluster = cg::this_cluster();
    if (n_ctas > 1) cluster.sync();
    else __syncthreads();
    if (p.n_splits > 0) pdl_wait();  // the prefix's partials
    pdl_release();
    for (int x = split * kThreads + tid; x < n_rows * kPer; x += n_ctas * kThreads) {
      const int row = x / kPer, ch = (x % kPer) * 4, u = row0 + row;
      float m = -INFINITY, l = 0.0f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      auto fold = [&](float2 ml, float4 v) {
        const float top = fmaxf(m, ml.x), from = top == -INFINITY ? 0.0f : top, f = ex2(m - from), e = ex2(ml.x - from);
        m = top;
        l = l * f + ml.y * e;
        o.x = o.x * f + v.x * e, o.y = o.y * f + v.y * e, o.z = o.z * f + v.z * e, o.w = o.w * f + v.w * e;
      };
      for (int i = 0; i < n_ctas; ++i) {
        const float* src = n_ctas > 1 ? cluster.map_shared_rank(po, i) : po;
        const float2* sml = n_ctas > 1 ? cluster.map_shared_rank(cml, i) : cml;
        fold(sml[row], *reinterpret_cast<const float4*>(src + row * kLd + ch));
      }
      const int64_t prow = (int64_t)b * unit_rows + u, step = (int64_t)p.h * p.rows;
      const float2* ml = p.part_ml + (int64_t)j * p.rows + prow;
      const float* po2 = p.part_o + ((int64_t)j * p.rows + prow) * D + ch;
      int i = 0;
      for (; i + 8 <= p.n_splits; i += 8) {
        float2 a[8];
        float4 v[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) a[y] = ml[(i + y) * step], v[y] = *reinterpret_cast<const float4*>(po2 + (i + y) * step * D);
#pragma unroll
        for (int y = 0; y < 8; ++y) fold(a[y], v[y]);
      }
      for (; i < p.n_splits; ++i) fold(ml[i * step], *reinterpret_cast<const float4*>(po2 + i * step * D));
      const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // no key at all: 0; a NaN stays one
      const int64_t at = ((int64_t)b * p.tokens + u / p.group) * (p.h * p.group) + j * p.group + u % p.group;
      if (p.out_f32)
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at * D + ch) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      else
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at * D + ch) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      if (ch == 0) p.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
    if (n_ctas > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
  }
}

template <int D, bool INT8, bool PREFIX>
cudaError_t launch_stream(const Params& p, dim3 grid, int cluster, int n_ctas, cudaStream_t st) {
  using S = Shape<D, INT8>;
  constexpr int kMerge = kWarps * kRows * (D + 4) * 4 + (kWarps + 1) * kRows * 8;
  constexpr int kSmem = S::kRing > kMerge ? S::kRing : kMerge;
  auto k = stream_kernel<D, INT8, PREFIX>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(k, grid, dim3(kThreads), kSmem, st, cluster, p, n_ctas);
}

// Batches of at most this many rows per KV head take the prefix through stream_kernel, one row tile.
bool streams(int rows) { return rows <= kRows; }

// Splits of the prefix: enough CTAs for two on each SM, no split shorter than two stages per warp.
int prefix_splits(int rows, int h, int64_t prefix_len, int d) {
  if (prefix_len <= 0) return 0;
  if (!streams(rows)) return tile_splits(rows, h, prefix_len);
  const int tok = stage_tokens(d);
  const int64_t tiles = (rows + kRows - 1) / kRows, most = (prefix_len + 2 * kWarps * tok - 1) / (2 * kWarps * tok);
  int64_t n = (2 * kNumSMs) / (tiles * h);
  if (n < 1) n = 1;
  if (n > most) n = most;
  return (int)n;
}

}  // namespace
}  // namespace prefix
}  // namespace lkv

using namespace lkv;
using namespace lkv::prefix;

extern "C" {

size_t lkv_prefix_attention_workspace(int batch, int tokens, int hq, int h, int d, int64_t prefix_len) {
  if (batch < 1 || tokens < 1 || h < 1 || hq < h || prefix_len < 1) return 0;
  const int64_t rows = (int64_t)batch * tokens * (hq / h);
  return (size_t)prefix_splits((int)rows, h, prefix_len, d) * h * rows * ((size_t)d * 4 + 8);
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
  p.n_splits = prefix_splits(p.rows, a->h, a->prefix_len, a->d);
  p.out = a->out;
  p.out_f32 = a->out_dtype == LKV_F32;
  p.lse = a->lse;
  if (p.n_splits > 0) {
    const size_t need = lkv_prefix_attention_workspace(a->batch, a->tokens, a->hq, a->h, a->d, a->prefix_len);
    if (a->workspace_bytes < need) return fail(LKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, need);
    if (a->workspace == nullptr || !aligned(a->workspace, 16)) return fail(LKV_ERR_PTR, "%s: workspace must be 16-byte aligned", who);
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)p.n_splits * a->h * rows * a->d);
  }
  cudaStream_t st = as_stream(stream);
  const bool int8 = a->kind == LKV_CACHE_INT8, wide = a->d == 128;
  cudaError_t e = cudaSuccess;
  if (p.n_splits > 0 && !streams(p.rows)) {
    if (int rc = run_tiles(p, a->d, int8, st)) return rc;
  } else if (p.n_splits > 0) {
    const int tiles = (p.rows + kRows - 1) / kRows;
    if (p.n_splits > 65535) return fail(LKV_ERR_ARG, "%s: prefix too long", who);
    const dim3 grid(tiles, p.n_splits, a->h);
    e = wide ? (int8 ? launch_stream<128, true, true>(p, grid, 0, p.n_splits, st) : launch_stream<128, false, true>(p, grid, 0, p.n_splits, st))
             : (int8 ? launch_stream<64, true, true>(p, grid, 0, p.n_splits, st) : launch_stream<64, false, true>(p, grid, 0, p.n_splits, st));
    if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s (prefix): %s", who, cudaGetErrorString(e));
  }
  const int unit = a->tokens * group, tiles = (unit + kRows - 1) / kRows;
  // Own tokens: more CTAs per (sequence, head, row tile) while they all stay resident and the tables
  // could hold at least 512 tokens for each; how many tokens there are only the device knows.
  int c = 1;
  while (c < kMaxCluster && (int64_t)a->batch * a->h * tiles * c * 2 <= 2 * kNumSMs && (int64_t)a->table_cols * a->bs >= 512 * 2 * c) c *= 2;
  const dim3 grid(tiles * c, a->h, a->batch);
  e = wide ? (int8 ? launch_stream<128, true, false>(p, grid, c > 1 ? c : 0, c, st) : launch_stream<128, false, false>(p, grid, c > 1 ? c : 0, c, st))
           : (int8 ? launch_stream<64, true, false>(p, grid, c > 1 ? c : 0, c, st) : launch_stream<64, false, false>(p, grid, c > 1 ? c : 0, c, st));
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
