// How much weight every cached token got from the queries of new chunks: sums[s] += sum over query rows r that
// see token s of 2^(score(r, s) - lse(r)), the attention's own weights, whose lse the attention left.
//
// The scores are computed again, keys first: S' = K Q^T on the 5th-generation tensor cores has a token to a lane of
// tensor memory and a query row to a column, so that a thread sums the weights of one token in its registers, over all
// rows, in their order: no atomics, the same result every time. 256 tokens (two tiles of 128 keys, a warpgroup
// each) are taken against chunks of up to 128 query rows of their KV head. The chunks' scores are double-buffered in
// tensor memory: the products run ahead of the exponentials.
//
// The keys are read once; nothing is read of the values. A batch that decodes (a few rows a head) is bound by the
// keys' bytes, long chunks by the exponentials. Every sequence's 256-token tiles, weighted by their chunks of rows,
// are one line that the CTAs share equally. Warps 0-3 and 4-7 sum, 8 issues the products, 9 copies keys, 10 and 11
// write what no tile covers, 12-15 bring the queries; with int8 pages 16-23 turn codes into bf16 operands.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "prefix.cuh"
#include "scores.cuh"
#include "tensor.cuh"

namespace lkv {
namespace {

using namespace tc;
using namespace paged;
using prefix::ex2;
using prefix::kLog2e;

constexpr int kPair = 2 * kTile;  // tokens of a step
constexpr int kMostBatch = 8192;
constexpr int kQStages = 2;
// Tiles whose scales and page bits are kept. A tile's copies begin when the keys at most three tiles before it have been
// multiplied, and those are not before the scores two steps (four tiles) back are read.
constexpr int kInfo = 16;

struct SumsParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const float* lse;  // [rows, hq]
  const void* pages;
  const float* scales;
  int n_pages, page_shift;
  int rows, batch, h, group;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* lens;
  const int32_t* offsets;
  int last;        // query tokens of a chunk that count
  const float* sums;  // [batch, h, cap], or null: zeros
  float* out;
  int cap;
  float scale, cap_log2;  // scores x scale are in the log2 domain (capped: divided by the cap)
  uint64_t max_wait_ns;
};

template <int D, bool INT8>
struct Geometry {
  static constexpr int kHalves = D / 64, kHalfBytes = kTile * 128, kBytes = kHalves * kHalfBytes;
  static constexpr int kStages = INT8 ? 3 : 4;  // tiles of keys
  static constexpr int kRawBytes = INT8 ? kTile * D : 0, kRaw = INT8 ? 3 : 0;
  static constexpr int kThreads = INT8 ? 768 : 512;
  // Registers per thread: the warpgroups that sum take what the others leave of the launch's.
  static constexpr int kMany = INT8 ? 128 : 168, kFew = INT8 ? 56 : 80;
  static_assert(256 * kMany + (kThreads - 256) * kFew <= kThreads * (INT8 ? 80 : 128), "the register split is the launch's own");
  static constexpr int kSmemTiles = (kStages + kQStages) * kBytes + kRaw * kRawBytes + (INT8 ? kInfo * kTile * 4 : 0);
  static constexpr int kSmem = (kSmemTiles > kMostBatch * 8 ? kSmemTiles : kMostBatch * 8) + 1024;
};

struct Barriers {
  uint64_t k_full[4], k_empty[4], raw_full[3], raw_empty[3], q_full[kQStages], q_empty[kQStages], s_full[2][2], s_empty[2][2], info[kInfo], drain;
  alignas(16) float minus[kQStages][kTile];  // (read four at a time) -lse in the log2 domain; minus infinity: the row does not count
  alignas(16) int limit[kQStages][kTile];    // tokens that the row sees
  uint32_t have[kInfo];          // bit g: tokens 16 g .. 16 g + 15 of the tile have a page
  int64_t pos, end;              // this CTA's piece of the line: where its first step begins, and where it ends
  int b, k;                      // that step
  uint64_t max_wait_ns;
  uint32_t tmem;
  int quit;
};

struct Sequence {
  int q0, n_rows;   // first packed row and query rows per KV head that count
  int limit;        // tokens that the first of them sees
  int old;          // tokens in front of the chunk: their sums go on
  int seen;         // tokens there are
  int steps;        // of kPair tokens, per KV head
  int chunks;       // of query rows
};
__device__ __forceinline__ Sequence sequence_of(const SumsParams& p, int b) {
  Sequence s;
  const int from = max(0, p.offsets[b]), end = min(p.rows, p.offsets[b + 1]), n = max(0, end - from), used = min(n, p.last);
  const int len = p.lens[b];
  s.q0 = from + n - used;
  s.n_rows = used * p.group;
  s.old = (int)max((int64_t)0, (int64_t)len - n);
  s.limit = (int)max((int64_t)INT32_MIN / 2, min((int64_t)len - used + 1, (int64_t)INT32_MAX / 2));
  s.seen = (int)max((int64_t)0, min(min((int64_t)len, (int64_t)p.cap), (int64_t)p.table_cols << p.page_shift));
  s.steps = s.n_rows > 0 ? (s.seen + kPair - 1) / kPair : 0;
  s.chunks = (s.n_rows + kTile - 1) / kTile;
  return s;
}

// The steps of this CTA, in order; every role walks along.
struct Walk {
  Sequence q;
  int64_t pos, end;
  int b, k, j, step, from;  // from: the first chunk with a row that sees a token of the step
  bool first, last;         // of the CTA's steps of this sequence and head
  __device__ __forceinline__ Walk(const SumsParams& p, const Barriers& s) : pos(s.pos), end(s.end), b(s.b), k(s.k), first(true) {
    if (pos < end) q = sequence_of(p, b), place(p);
  }
  __device__ __forceinline__ bool more() const { return pos < end; }
  __device__ __forceinline__ void place(const SumsParams& p) {
    j = k / q.steps, step = k - j * q.steps;
    last = step == q.steps - 1 || pos + q.chunks >= end;
    // Row r sees tokens up to limit + r / group: the chunk's last row decides.
    const int64_t row = (int64_t)(step * kPair - q.limit + 1) * p.group;  // the first row that sees the step's first token
    from = row <= 0 ? 0 : (int)min((int64_t)(q.chunks - 1), row / kTile);
  }
  __device__ __forceinline__ void next(const SumsParams& p) {
    pos += q.chunks;
    first = last;
    if (!more()) return;
    if (++k == p.h * q.steps) {
      k = 0;
      do q = sequence_of(p, ++b);
      while (q.steps == 0 && b + 1 < p.batch);
      if (q.steps == 0) {
        pos = end;
        return;
      }
    }
    place(p);
  }
};

// 16 columns of a thread's own lane of tensor memory.
struct Lane {
  uint32_t v[16];
};
__device__ __forceinline__ void ld(Lane& f, uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : LKV_R8(f.v, 0), LKV_R8(f.v, 8)
               : "r"(addr));
}
__device__ __forceinline__ void ld_wait(Lane& f) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(f.v[i]));
}

template <int D, bool INT8, bool CAP>
__global__ void __launch_bounds__(Geometry<D, INT8>::kThreads, 1) sums_kernel(const SumsParams p, const __grid_constant__ CUtensorMap pages_map) {
  using G = Geometry<D, INT8>;
  constexpr int kStages = G::kStages;
  extern __shared__ char raw_smem[];
  __shared__ Barriers s;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  char* q_stages = smem;
  char* stages = q_stages + kQStages * G::kBytes;
  char* raws = stages + kStages * G::kBytes;
  float* scale_ring = reinterpret_cast<float*>(raws + G::kRaw * G::kRawBytes);  // [kInfo][kTile]: the keys'
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, bs = 1 << p.page_shift;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.k_full[i], INT8 ? 4 : 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < G::kRaw; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_empty[i], 4);
    }
    for (int i = 0; i < kQStages; ++i) {
      mbar_init(&s.q_full[i], 4);
      mbar_init(&s.q_empty[i], 9);  // the products' and the sums' warps
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s.s_full[i / 2][i % 2], 1);
      mbar_init(&s.s_empty[i / 2][i % 2], 4);
    }
    for (int i = 0; i < kInfo; ++i) mbar_init(&s.info[i], 1);
    mbar_init(&s.drain, 1);
    s.max_wait_ns = p.max_wait_ns;
    s.quit = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s.tmem;  // columns: scores of the two tiles, two buffers of 128 each
  pdl_wait();
  pdl_release();

  // Every sequence's length on the line, into shared memory that no copy uses yet; then this CTA's piece.
  int64_t* lengths = reinterpret_cast<int64_t*>(smem);
  for (int b = tid; b < p.batch; b += G::kThreads) {
    const Sequence q = sequence_of(p, b);
    lengths[b] = (int64_t)q.steps * q.chunks * p.h;
  }
  __syncthreads();
  if (warp == 0) {
    int64_t all = 0;
    for (int b = lane; b < p.batch; b += 32) all += lengths[b];
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const int64_t n = gridDim.x, c = blockIdx.x;
    const int64_t lo = all / n * c + all % n * c / n, hi = all / n * (c + 1) + all % n * (c + 1) / n;
    // The first step that begins at or behind lo.
    int64_t before = 0;
    int found = -1;
    int64_t k = 0, pos = hi;
    for (int b0 = 0; b0 < p.batch && found < 0 && lo < hi; b0 += 32) {
      const int b = b0 + lane;
      int64_t upto = b < p.batch ? lengths[b] : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, before + upto > lo);
      if (behind != 0) {
        const int l = __ffs(behind) - 1;
        if (l > 0) before += __shfl_sync(0xffffffffu, upto, l - 1);
        found = b0 + l;
      } else {
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (found >= 0) {
      const Sequence q = sequence_of(p, found);
      k = (max(lo - before, (int64_t)0) + q.chunks - 1) / q.chunks;
      pos = before + k * q.chunks;
      while (pos < hi && k >= (int64_t)sequence_of(p, found).steps * p.h) {  // behind this sequence's last step: the next one's first
        do ++found;
        while (found + 1 < p.batch && lengths[found] == 0);
        k = 0;
      }
    }
    if (lane == 0) s.pos = pos, s.end = hi, s.b = max(found, 0), s.k = (int)k;
  }
  fence_async();
  __syncthreads();

  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kMany));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kFew));
  if (warp < 8) {
    // ---- sums: a thread has a token -------------------------------------------------------------------
    const int u = warp / 4, i = tid % kTile;
    const uint32_t ts = tmem + ((uint32_t)(warp % 4) << 21) + u * 2 * kTile;
    int q_count = 0, job = 0, tile = u;
    bool ok = true;
    for (Walk w(p, s); w.more() && ok; w.next(p), tile += 2) {
      const int token = w.step * kPair + u * kTile + i, info = tile % kInfo;
      const int64_t at = ((int64_t)w.b * p.h + w.j) * p.cap + token;
      float old = 0.0f;
      if (p.sums != nullptr && token < min(w.q.old, w.q.seen)) old = p.sums[at];
      ok = wait_for(s, &s.info[info], (tile / kInfo) & 1);
      if (!ok) break;
      const bool there = token < w.q.seen && (s.have[info] >> (i / 16) & 1);
      const float factor = INT8 && there ? p.scale * scale_ring[info * kTile + i] : p.scale;
      const uint64_t factor2 = pair(factor, factor);
      uint64_t sum[2] = {0, 0};
      bool wide_step = false;  // capped scores above their cap's size
      for (int c = w.from; c < w.q.chunks; ++c, ++job) {
        const int buf = job & 1, stage = q_count % kQStages;
        ok = wait_for(s, &s.q_full[stage], (q_count / kQStages) & 1) && wait_for(s, &s.s_full[u][buf], (job >> 1) & 1);
        if (!ok) break;
        tc_after();
        const int n_cols = min(kTile, w.q.n_rows - c * kTile);
        const bool masked = n_cols % 16 != 0 || s.limit[stage][0] < w.step * kPair + u * kTile + kTile;
        const float4* minus = reinterpret_cast<const float4*>(s.minus[stage]);
        const int4* limit = reinterpret_cast<const int4*>(s.limit[stage]);
        // MASK: some row does not see the tile whole. WIDE: scores may be above their cap's size; false where one is and WIDE
        // is not.
        auto all = [&](auto mask, [[maybe_unused]] auto any_size) {
          constexpr bool MASK = decltype(mask)::value, WIDE = decltype(any_size)::value;
          uint64_t more[2] = {sum[0], sum[1]};
          float most = 0.0f;
          auto add = [&](const Lane& f, int n) {
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
              const float4 m = minus[(16 * n + x) / 4];
              [[maybe_unused]] int4 upto;
              if constexpr (MASK) upto = limit[(16 * n + x) / 4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint64_t z = pair(__uint_as_float(f.v[x + 2 * e]), __uint_as_float(f.v[x + 2 * e + 1]));
                const uint64_t by = e == 0 ? pair(m.x, m.y) : pair(m.z, m.w);
                if constexpr (!CAP) {
                  z = fma2(z, factor2, by);
                } else if constexpr (WIDE) {
                  z = mul2(z, pair(2.0f * kLog2e * factor, 2.0f * kLog2e * factor));
                  z = add2(pair(capped(first_of(z), p.cap_log2), capped(second_of(z), p.cap_log2)), by);
                } else {
                  uint64_t square;
                  z = capped2(mul2(z, factor2), p.cap_log2, by, &square);
                  most = fmaxf(fmaxf(most, first_of(square)), second_of(square));
                }
                z = pair(ex2(first_of(z)), ex2(second_of(z)));
                if constexpr (MASK) z = pair(token < (e == 0 ? upto.x : upto.z) ? first_of(z) : 0.0f, token < (e == 0 ? upto.y : upto.w) ? second_of(z) : 0.0f);
                more[e] = add2(more[e], z);
              }
            }
          };
          Lane f[2];
          const int n = (n_cols + 15) / 16;
          ld(f[0], ts + buf * kTile);
          ld_wait(f[0]);
#pragma unroll 1
          for (int x = 0; x < n; x += 2) {
            if (x + 1 < n) ld(f[1], ts + buf * kTile + 16 * (x + 1));
            add(f[0], x);
            if (x + 1 < n) ld_wait(f[1]);
            if (x + 2 < n) ld(f[0], ts + buf * kTile + 16 * (x + 2));
            if (x + 1 < n) add(f[1], x + 1);
            if (x + 2 < n) ld_wait(f[0]);
          }
          if constexpr (CAP && !WIDE) {
            if (__any_sync(0xffffffffu, most > 1.0f)) return false;
          }
          sum[0] = more[0], sum[1] = more[1];
          return true;
        };
        const std::true_type yes;
        const std::false_type no;
        if (CAP && wide_step) {
          if (masked) all(yes, yes);
          else all(no, yes);
        } else if (!(masked ? all(yes, no) : all(no, no))) {
          wide_step = true;
          if (masked) all(yes, yes);
          else all(no, yes);
        }
        tc_before();
        warp_arrive(&s.s_empty[u][buf], lane);
        // (One chunk a sequence and head stays for all of its steps.)
        if (w.q.chunks > 1 || w.last) {
          warp_arrive(&s.q_empty[stage], lane);
          ++q_count;
        }
      }
      const float got = (first_of(sum[0]) + second_of(sum[0])) + (first_of(sum[1]) + second_of(sum[1]));
      if (token < p.cap) p.out[at] = old + (!ok ? __uint_as_float(0x7fc00000u) : there ? got : 0.0f);
    }
  } else if (warp == 8) {
    // ---- matrix products ------------------------------------------------------------------------------
    const uint32_t q_u = smem_u32(q_stages), k_u = smem_u32(stages), mine = elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
    int q_count = 0, job = 0, tiles = 0;
    bool ok = true;
    for (Walk w(p, s); w.more() && ok; w.next(p), tiles += 2) {
      for (int c = w.from; ok && c < w.q.chunks; ++c, ++job) {
        const int buf = job & 1, stage = q_count % kQStages;
        ok = wait_for(s, &s.q_full[stage], (q_count / kQStages) & 1);
        const uint32_t inst = instruction<false>((min(kTile, w.q.n_rows - c * kTile) + 15) / 16 * 16, false);
        for (int u = 0; ok && u < 2; ++u) {
          const int slot = (tiles + u) % kStages;
          if (c == w.from) ok = wait_for(s, &s.k_full[slot], ((tiles + u) / kStages) & 1);
          if (ok && job >= 2) ok = wait_for(s, &s.s_empty[u][buf], ((job >> 1) - 1) & 1);
          if (!ok) break;
          tc_after();
          const uint64_t a = desc_of(k_u + slot * G::kBytes, 16), b = desc_of(q_u + stage * G::kBytes, 16);
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint64_t off = ((x / 4) * G::kHalfBytes + (x % 4) * 32) / 16;
            mma_ss(tm + u * 2 * kTile + buf * kTile, a + off, b + off, inst, x > 0, mine);
          }
          commit(&s.s_full[u][buf], mine);
          if (c == w.q.chunks - 1) commit(&s.k_empty[slot], mine);
        }
        if (!ok) break;
        if (w.q.chunks > 1 || w.last) {
          commit(&s.q_empty[stage], mine);
          ++q_count;
        }
      }
      if (!ok) break;
    }
    commit(&s.drain, mine);
    mbar_wait(&s.drain, 0);
    __syncwarp();
  } else if (warp == 9) {
    // ---- copies of keys: the pages of 128 tokens at a time ----------------------------------------------
    const int per = kTile >> p.page_shift;
    int filled = 0;
    bool ok = true;
    constexpr int kSlots = INT8 ? G::kRaw : kStages;
    // Lane i has page i of each tile, looked up a step ahead (their ids, checked where they are used).
    int ahead[2] = {-1, -1};
    auto look_up = [&](const Walk& w) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int token = w.step * kPair + u * kTile + lane * bs;
        ahead[u] = w.more() && lane < per && token < w.q.seen ? p.table[w.b * p.table_ld + (token >> p.page_shift)] : -1;
      }
    };
    Walk next(p, s);
    look_up(next);
    while (next.more() && ok) {
      const Walk w = next;
      const int pages[2] = {ahead[0], ahead[1]};
      next.next(p);
      look_up(next);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int slot = filled % kSlots, page = pages[u] < p.n_pages ? pages[u] : -1;
        uint64_t* full = INT8 ? &s.raw_full[slot % 3] : &s.k_full[slot];
        if (filled >= kSlots) ok = ok && wait_for(s, INT8 ? &s.raw_empty[slot % 3] : &s.k_empty[slot], (filled / kSlots - 1) & 1);
        if (!ok) break;
        const int info = filled % kInfo;
        const uint32_t granules = page >= 0 ? ((1u << (bs / 16)) - 1) << (lane * (bs / 16)) : 0u;
        const uint32_t have = __reduce_or_sync(0xffffffffu, granules);
        if (lane == 0) {
          s.have[info] = have;
          if (INT8) mbar_arrive_expect_tx(&s.info[info], __popc(have) * 64);  // 16 scales of each 16 tokens
          else mbar_arrive(&s.info[info]);
        }
        if constexpr (!INT8) {
          if (lane == 0) mbar_arrive_expect_tx(full, G::kBytes);
          __syncwarp();
          if (lane < per) {
            const int rows = p.n_pages * 2 * p.h * bs;  // one past the last: zeros
            const int y = page >= 0 ? ((page * p.h + w.j) * 2) * bs : rows;
            const uint32_t dst = smem_u32(stages) + slot * G::kBytes + lane * bs * 128;
#pragma unroll
            for (int h2 = 0; h2 < G::kHalves; ++h2) tma_2d(dst + h2 * G::kHalfBytes, &pages_map, 64 * h2, y, full);
          }
        } else {
          const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, page >= 0));
          if (lane == 0) mbar_arrive_expect_tx(full, n_copies * bs * D);
          __syncwarp();
          if (page >= 0) {
            tma_load_1d(scale_ring + info * kTile + lane * bs, p.scales + ((int64_t)page * p.h + w.j) * 2 * bs, bs * 4, &s.info[info]);
            tma_load_1d(raws + slot * G::kRawBytes + lane * bs * D, static_cast<const char*>(p.pages) + (((int64_t)page * p.h + w.j) * 2) * ((int64_t)bs * D), bs * D, full);
          }
        }
        ++filled;
      }
    }
    for (int n = max(0, filled - kInfo); n < filled; ++n) mbar_wait(&s.info[n % kInfo], (n / kInfo) & 1);
    for (int n = max(0, filled - kSlots); n < filled; ++n) mbar_wait(INT8 ? &s.raw_full[n % 3] : &s.k_full[n % kSlots], (n / kSlots) & 1);
    __syncwarp();
  } else if (warp < 12) {
    // ---- slots that no step covers: what was there goes on, new and missing tokens have nothing -----------
    const int64_t n = (int64_t)p.batch * p.h;
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
      const Sequence q = sequence_of(p, (int)(row / p.h));
      const int go_on = min(q.old, q.seen);
      for (int64_t i = (int64_t)q.steps * kPair + tid - 10 * 32; i < p.cap; i += 64) {
        p.out[row * p.cap + i] = p.sums != nullptr && i < go_on ? p.sums[row * p.cap + i] : 0.0f;
      }
    }
  } else if (warp < 16) {
    // ---- queries: a thread has a row of the chunk ------------------------------------------------------
    const int r = tid % kTile;
    int q_count = 0;
    bool ok = true;
    for (Walk w(p, s); w.more() && ok; w.next(p)) {
      if (w.q.chunks == 1 && !w.first) continue;
      for (int c = w.from; c < w.q.chunks; ++c, ++q_count) {
        const int stage = q_count % kQStages, row = c * kTile + r;
        if (q_count >= kQStages) ok = wait_for(s, &s.q_empty[stage], (q_count / kQStages - 1) & 1);
        if (!ok) break;
        const bool live = row < w.q.n_rows;
        const int t = live ? row / p.group : 0, head = live ? w.j * p.group + row - t * p.group : 0;
        const __nv_bfloat16* src = p.q + (int64_t)(w.q.q0 + t) * p.q_st + (int64_t)head * p.q_sh;
        char* dst = q_stages + stage * G::kBytes + r * 128;
        if (row < w.q.n_rows + 16) {  // (rows of the product past the last one: zeros)
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + (i / 8) * (kTile * 128) + (((i % 8) ^ (r & 7)) << 4))), "l"(src + 8 * i),
                         "r"(live ? 16 : 0)
                         : "memory");
        }
        const float lse = live ? p.lse[(int64_t)(w.q.q0 + t) * (p.h * p.group) + head] : -INFINITY;
        s.minus[stage][r] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
        s.limit[stage][r] = live && lse != -INFINITY ? w.q.limit + t : 0;
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        fence_async();
        warp_arrive(&s.q_full[stage], lane);
      }
    }
  } else if constexpr (INT8) {
    // ---- codes to bf16 operands: warps 16-19 the first tile's, 20-23 the second's -----------------------
    const int i = tid % kTile, u = (tid - 16 * 32) / kTile;
    // As chunk.cu: pieces of 16 codes, one channel range of every kStep-th token, without bank conflicts.
    constexpr int kPer = D / 16, kStep = kTile / kPer;
    const int odd = (i >> 2) & 1, half = odd ^ ((i >> 3) & 1);
    const int tok0 = kPer == 8 ? (i >> 4) * 2 + odd : i / kPer, c = kPer == 8 ? half * 4 + (i & 3) : i % kPer;
    const int from = (tok0 * kPer + c) * 16, row = (c / 4) * G::kHalfBytes + tok0 * 128, at = (c % 4) * 2;
    const int to0 = row + ((at ^ (tok0 & 7)) << 4), to1 = row + (((at + 1) ^ (tok0 & 7)) << 4);
    bool ok = true;
    int n = u;
    for (Walk w(p, s); w.more() && ok; w.next(p), n += 2) {
      const int raw = n % G::kRaw, slot = n % kStages;
      ok = wait_for(s, &s.raw_full[raw], (n / G::kRaw) & 1);
      if (ok && n >= kStages) ok = wait_for(s, &s.k_empty[slot], (n / kStages - 1) & 1);
      if (!ok) break;
      const char* src = raws + raw * G::kRawBytes + from;
      char* dst = stages + slot * G::kBytes;
#pragma unroll
      for (int x0 = 0; x0 < kPer; x0 += 4) {
        uint4 v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = *reinterpret_cast<const uint4*>(src + (x0 + x) * (kStep * kPer * 16));
        if (x0 + 4 >= kPer) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.raw_empty[raw]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint2 a = codes_to_bf16(v[x].x), b = codes_to_bf16(v[x].y), d = codes_to_bf16(v[x].z), e = codes_to_bf16(v[x].w);
          *reinterpret_cast<uint4*>(dst + to0 + kStep * (x0 + x) * 128) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(dst + to1 + kStep * (x0 + x) * 128) = make_uint4(d.x, d.y, e.x, e.y);
        }
      }
      fence_async();
      warp_arrive(&s.k_full[slot], lane);
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int D, bool INT8, bool CAP>
cudaError_t launch(const SumsParams& p, const CUtensorMap& map, int grid, cudaStream_t st) {
  using G = Geometry<D, INT8>;
  auto k = sums_kernel<D, INT8, CAP>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = prefix::allow_smem(k, G::kSmem, done);
  return e != cudaSuccess ? e : launch_pdl(k, dim3(grid), dim3(G::kThreads), G::kSmem, st, 0, p, map);
}

}  // namespace

cudaError_t sums_device_status(int* status, int clear) { return tu_device_status(status, clear); }
cudaError_t sums_status_attach(int* mirror) { return tu_status_attach(mirror); }

}  // namespace lkv

using namespace lkv;

extern "C" int lkv_attention_sums(const lkv_sums_args* a, void* stream) {
  static const char* who = "lkv_attention_sums";
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (a->dtype != LKV_BF16) return fail(LKV_ERR_ARG, "%s: queries are bfloat16, got dtype %d", who, a->dtype);
  if (int rc = check_cache(who, a->kind, a->dtype, a->h, a->bs, a->d, a->n_pages, a->pages, a->scales)) return rc;
  if (a->rows < 0 || a->rows > (1 << 30) || a->batch < 0 || a->batch > kMostBatch || a->table_cols < 0 || (a->batch > 1 && a->table_ld < a->table_cols) ||
      a->cap < 0 || a->cap > (1 << 30))
    return fail(LKV_ERR_ARG, "%s: bad shape (rows %d, batch %d of at most %d, table of %d columns, %d slots)", who, a->rows, a->batch, kMostBatch, a->table_cols, a->cap);
  if (a->hq < 1 || a->hq % a->h != 0 || a->hq / a->h > 1024) return fail(LKV_ERR_ARG, "%s: %d query heads for %d KV heads", who, a->hq, a->h);
  const int group = a->hq / a->h;
  if ((int64_t)a->rows * group > (1 << 30)) return fail(LKV_ERR_ARG, "%s: %d rows of %d query heads per KV head in one call", who, a->rows, group);
  if (a->last < 1) return fail(LKV_ERR_ARG, "%s: the last %d tokens of a chunk", who, a->last);
  if (!(a->cap_scores >= 0.0f) || a->cap_scores > FLT_MAX || !(fabsf(a->scale) <= FLT_MAX)) return fail(LKV_ERR_ARG, "%s: scale %g, cap %g", who, (double)a->scale, (double)a->cap_scores);
  const int64_t page_rows = a->n_pages * 2 * a->h * a->bs;
  if (page_rows > INT32_MAX) return fail(LKV_ERR_ARG, "%s: %lld rows of pages", who, (long long)page_rows);
  if (a->batch == 0 || a->cap == 0) return LKV_OK;
  if (a->lens == nullptr || a->offsets == nullptr || a->out == nullptr || (a->table == nullptr && a->table_cols > 0) || (a->rows > 0 && (a->q == nullptr || a->lse == nullptr)))
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(a->q, 16) || (a->q_st & 7) != 0 || (a->q_sh & 7) != 0) return fail(LKV_ERR_PTR, "%s: query rows must be 16-byte aligned", who);
  SumsParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.q_st = a->q_st, p.q_sh = a->q_sh, p.lse = a->lse;
  p.pages = a->pages, p.scales = a->scales, p.n_pages = (int)a->n_pages, p.page_shift = shift_of(a->bs);
  p.rows = a->rows, p.batch = a->batch, p.h = a->h, p.group = group;
  p.table = a->table, p.table_ld = a->table_ld, p.table_cols = a->table_cols, p.lens = a->lens, p.offsets = a->offsets;
  p.last = a->last, p.sums = a->sums, p.out = a->out, p.cap = a->cap;
  const bool cap = a->cap_scores > 0.0f;
  p.scale = cap ? a->scale / a->cap_scores : a->scale * kLog2e;
  p.cap_log2 = a->cap_scores * kLog2e;
  p.max_wait_ns = kMaxTensorWaitNs;
  const bool int8 = a->kind == LKV_CACHE_INT8;
  CUtensorMap map = {};
  if (!int8) {
    if (page_rows == 0) return fail(LKV_ERR_ARG, "%s: a cache without pages", who);
    const cuuint64_t dims[2] = {(cuuint64_t)a->d, (cuuint64_t)page_rows}, strides[1] = {(cuuint64_t)a->d * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)a->bs}, ones[2] = {1, 1};
    const CUresult r = encode_tiled(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a->pages, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LKV_ERR_CUDA, "%s: the pages' tensor map was refused (%d)", who, (int)r);
  }
  // One CTA per SM, or one per step that the call can have at most (some all the same: they write the other slots).
  const int64_t steps = ((int64_t)a->cap + kPair - 1) / kPair * a->h * a->batch;
  const int grid = (int)std::min<int64_t>(kNumSMs, steps);
  cudaStream_t st = as_stream(stream);
  auto go = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (int8) return cap ? launch<D, true, true>(p, map, grid, st) : launch<D, true, false>(p, map, grid, st);
    return cap ? launch<D, false, true>(p, map, grid, st) : launch<D, false, false>(p, map, grid, st);
  };
  const cudaError_t e = a->d == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 64>());
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}
