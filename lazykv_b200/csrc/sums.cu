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
// keys' bytes, long chunks by the exponentials. All jobs, 256 tokens against one chunk, in the order sequence, head,
// tokens, chunk, are one line that the CTAs share equally. Where a CTA's piece begins or ends between the chunks of a
// tile, its sums are parts that sums_merge_kernel adds, in order. Warps 0-3 and 4-7 sum, 8 issues the products, 9 copies
// keys, 10 and 11 write what no tile covers, 12-15 bring the queries; with int8 pages 16-23 turn codes into bf16 operands.
//
// Measured (8 KV heads, 4 query heads each, d 128): one token of each of 48 sequences of up to 6,000 int8 tokens 82 us
// (bf16 pages, twice the bytes: 62): the chain of a step of 256 tokens, copy, conversion, products, sums, takes 3,700 cycles, and
// shared memory holds two steps' codes beside the operands. 32 tokens' queries over 40,032 bf16 tokens 31 us, half of it the
// start, first copies and end. 499 and 999 tokens, 7 query heads a KV head, d 64, scores capped, over 9,001: 121 us (85 without
// the cap): two summing warps a scheduler, no unit busy to a half.
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
// Tiles whose scales and page bits are kept. A tile's copies begin when the codes at most six tiles before it have been turned
// into operands, that when the keys four tiles before have been multiplied, and that when the scores two steps (four tiles) back
// are read: fourteen tiles.
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
  float* part;            // [2 CTAs][kPair]: sums of a tile's first and last chunks in the CTA's piece
  int4* part_of;          // (1: a part, 3: the tile's last; sequence, head, step)
  float scale, cap_log2;  // scores x scale are in the log2 domain (capped: divided by the cap)
  uint64_t max_wait_ns;
  int stall, stall_cta;  // test hook: a warp of this CTA (-1: of every CTA) withholds an arrival
};

template <int D, bool INT8>
struct Geometry {
  static constexpr int kHalves = D / 64, kHalfBytes = kTile * 128, kBytes = kHalves * kHalfBytes;
  static constexpr int kStages = 4;  // tiles of keys: two steps
  static constexpr int kRawBytes = INT8 ? kTile * D : 0, kRaw = INT8 ? (D == 128 ? 4 : 6) : 0;
  // Two warpgroups turn codes of the two tiles of a step into operands, and each waits for its own tiles only: a place in a
  // ring has to be the same one's every time, or it could take the other's last round for its own.
  static_assert(kStages % 2 == 0 && kRaw % 2 == 0, "every place belongs to one warpgroup");
  // Query rows of a chunk: with int8 pages fewer, which leaves room for codes under way.
  static constexpr int kRows = INT8 ? 32 : 128, kQBytes = kHalves * kRows * 128;
  static constexpr int kThreads = INT8 ? 768 : 512;
  // Registers per thread: the warpgroups that sum take what the others leave of the launch's.
  static constexpr int kMany = INT8 ? 128 : 168, kFew = INT8 ? 56 : 80;
  static_assert(256 * kMany + (kThreads - 256) * kFew <= kThreads * (INT8 ? 80 : 128), "the register split is the launch's own");
  static constexpr int kSmemTiles = kStages * kBytes + kQStages * kQBytes + kRaw * kRawBytes + (INT8 ? kInfo * kTile * 4 : 0);
  static constexpr int kSmem = (kSmemTiles > kMostBatch * 8 ? kSmemTiles : kMostBatch * 8) + 1024;
};

struct Barriers {
  uint64_t k_full[4], k_empty[4], raw_full[6], raw_empty[6], q_full[kQStages], q_empty[kQStages], s_full[2][2], s_empty[2][2], info[kInfo], drain;
  alignas(16) float minus[kQStages][kTile];  // (read four at a time) -lse in the log2 domain; minus infinity: the row does not count
  alignas(16) int limit[kQStages][kTile];    // tokens that the row sees
  uint32_t have[kInfo];          // bit g: tokens 16 g .. 16 g + 15 of the tile have a page
  int64_t jobs;                  // of this CTA's piece of the line
  int b, j, step, chunk;         // its first
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
template <int kRows>
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
  s.chunks = (s.n_rows + kRows - 1) / kRows;
  return s;
}

// The first chunk with a row that sees a token of the step (row r sees tokens up to limit + r / group).
template <int kRows>
__device__ __forceinline__ int first_chunk(const SumsParams& p, const Sequence& q, int step) {
  const int64_t row = ((int64_t)step * kPair - q.limit + 1) * p.group;
  return row < kRows ? 0 : (int)min((int64_t)(q.chunks - 1), row / kRows);
}
// Jobs of a sequence, per KV head.
template <int kRows>
__device__ __forceinline__ int64_t jobs_of(const SumsParams& p, const Sequence& q) {
  int64_t n = (int64_t)q.steps * q.chunks;
  for (int step = q.steps - 1; step >= 0; --step) {  // only steps among the chunk's own tokens have fewer
    const int from = first_chunk<kRows>(p, q, step);
    if (from == 0) break;
    n -= from;
  }
  return n;
}

// The tiles of this CTA's piece, in order, each with the chunks that are the CTA's; every role walks along.
template <int kRows>
struct Walk {
  Sequence q;
  int64_t left;  // jobs from this tile on
  int b, j, step;
  int from, to;      // its chunks
  bool begun, last;  // an earlier CTA has chunks of the tile; the CTA's last tile of this sequence and head
  __device__ __forceinline__ Walk(const SumsParams& p, const Barriers& s) : left(s.jobs), b(s.b), j(s.j), step(s.step) {
    if (left > 0) q = sequence_of<kRows>(p, b), place(s.chunk), begun = from > first_chunk<kRows>(p, q, step);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ bool whole() const { return !begun && to == q.chunks; }
  __device__ __forceinline__ void place(int chunk) {
    from = chunk, to = (int)min((int64_t)q.chunks, chunk + left), begun = false;
    last = step == q.steps - 1 || left <= to - from;
  }
  __device__ __forceinline__ void next(const SumsParams& p) {
    left -= to - from;
    if (!more()) return;
    if (++step == q.steps) {
      step = 0;
      if (++j == p.h) {
        j = 0;
        do {
          if (++b == p.batch) {
            left = 0;
            return;
          }
          q = sequence_of<kRows>(p, b);
        } while (q.steps == 0);
      }
    }
    place(first_chunk<kRows>(p, q, step));
  }
};

template <int D, bool INT8, bool CAP>
__global__ void __launch_bounds__(Geometry<D, INT8>::kThreads, 1) sums_kernel(const SumsParams p, const __grid_constant__ CUtensorMap pages_map) {
  using G = Geometry<D, INT8>;
  constexpr int kStages = G::kStages;
  extern __shared__ char raw_smem[];
  __shared__ Barriers s;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  char* q_stages = smem;
  char* stages = q_stages + kQStages * G::kQBytes;
  char* raws = stages + kStages * G::kBytes;
  float* scale_ring = reinterpret_cast<float*>(raws + G::kRaw * G::kRawBytes);  // [kInfo][kTile]: the keys'
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, bs = 1 << p.page_shift;
  auto stalls = [&](int which) { return p.stall == which && (p.stall_cta < 0 || p.stall_cta == (int)blockIdx.x); };
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
    lengths[b] = jobs_of<G::kRows>(p, sequence_of<G::kRows>(p, b)) * p.h;
  }
  __syncthreads();
  if (warp == 0) {
    int64_t all = 0;
    for (int b = lane; b < p.batch; b += 32) all += lengths[b];
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const int64_t n = gridDim.x, c = blockIdx.x;
    const int64_t lo = all / n * c + all % n * c / n, hi = all / n * (c + 1) + all % n * (c + 1) / n;
    int64_t at = lo;
    int b = 0, j = 0, step = 0;
    if (lo < hi) {
      for (;; b += 32) {  // the sequence, 32 at a time
        int64_t upto = b + lane < p.batch ? lengths[b + lane] : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, upto > at);
        if (behind != 0) {
          const int first = __ffs(behind) - 1;
          if (first > 0) at -= __shfl_sync(0xffffffffu, upto, first - 1);
          b += first;
          break;
        }
        at -= __shfl_sync(0xffffffffu, upto, 31);
      }
      const Sequence q = sequence_of<G::kRows>(p, b);
      const int64_t per_head = lengths[b] / p.h;
      j = (int)(at / per_head);
      at -= j * per_head;
      step = (int)min(at / q.chunks, (int64_t)(q.steps - 1));
      // (Steps among the chunk's own tokens have fewer jobs: the quotient is too low there.)
      int64_t before = (int64_t)step * q.chunks;
      for (int x = step - 1; x >= 0; --x) {
        const int from = first_chunk<G::kRows>(p, q, x);
        if (from == 0) break;
        before -= from;
      }
      for (;; ++step) {
        const int n = q.chunks - first_chunk<G::kRows>(p, q, step);
        if (at < before + n) break;
        before += n;
      }
      at += first_chunk<G::kRows>(p, q, step) - before;
    }
    if (lane == 0) s.jobs = hi - lo, s.b = b, s.j = j, s.step = step, s.chunk = (int)at;
    if (lane < 2) p.part_of[2 * blockIdx.x + lane] = make_int4(0, 0, 0, 0);
  }
  fence_async();
  __syncthreads();

  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kMany));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kFew));
  if (warp < 8) {
    // ---- sums: a thread has a token -------------------------------------------------------------------
    // (Where a wait ran out these warps go on to the end of the CTA's piece, without waiting: every tile that is left,
    // or its part, is NaN, and every part is there for the merge.)
    const int u = warp / 4, i = tid % kTile;
    const uint32_t ts = tmem + ((uint32_t)(warp % 4) << 21) + u * 2 * kTile;
    int q_count = 0, job = 0, tile = u;
    bool ok = true;
    for (Walk<G::kRows> w(p, s); w.more(); w.next(p), tile += 2) {
      const int token = w.step * kPair + u * kTile + i, info = tile % kInfo;
      const int64_t at = ((int64_t)w.b * p.h + w.j) * p.cap + token;
      float old = 0.0f;
      if (w.whole() && p.sums != nullptr && token < min(w.q.old, w.q.seen)) old = p.sums[at];
      ok = ok && wait_for(s, &s.info[info], (tile / kInfo) & 1);
      const bool there = token < w.q.seen && (s.have[info] >> (i / 16) & 1);
      // (The codes of a page that is not there are what shared memory held: next to a capped score they would choose its form.)
      const float factor = !INT8 ? p.scale : there ? p.scale * scale_ring[info * kTile + i] : 0.0f;
      const uint64_t factor2 = pair(factor, factor);
      uint64_t sum[2] = {0, 0};
      bool wide_step = false;  // capped scores above their cap's size
      for (int c = w.from; ok && c < w.to; ++c, ++job) {
        const int buf = job & 1, stage = q_count % kQStages;
        ok = wait_for(s, &s.q_full[stage], (q_count / kQStages) & 1) && wait_for(s, &s.s_full[u][buf], (job >> 1) & 1);
        if (!ok) break;
        tc_after();
        const int n_cols = min(G::kRows, w.q.n_rows - c * G::kRows);
        const bool masked = n_cols % 32 != 0 || s.limit[stage][0] < w.step * kPair + u * kTile + kTile;
        const float4* minus = reinterpret_cast<const float4*>(s.minus[stage]);
        const int4* limit = reinterpret_cast<const int4*>(s.limit[stage]);
        // MASK: some row does not see the tile whole. WIDE: scores may be above their cap's size; false where one is and WIDE
        // is not.
        auto all = [&](auto mask, [[maybe_unused]] auto any_size) {
          constexpr bool MASK = decltype(mask)::value, WIDE = decltype(any_size)::value;
          uint64_t more[2] = {sum[0], sum[1]};
          float most = 0.0f;
          auto add = [&](const auto& f, int first) {  // columns from `first` on
            constexpr int N = sizeof(f.v) / 4;
#pragma unroll
            for (int x = 0; x < N; x += 16) {  // step by step for eight pairs: their chains of results do not wait for one another
              uint64_t z[8], by[8];
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const float4 m = minus[(first + x) / 4 + e / 2];
                by[e] = pair(m.x, m.y), by[e + 1] = pair(m.z, m.w);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) z[e] = pair(__uint_as_float(f.v[x + 2 * e]), __uint_as_float(f.v[x + 2 * e + 1]));
              if constexpr (!CAP) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = fma2(z[e], factor2, by[e]);
              } else if constexpr (WIDE) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  z[e] = mul2(z[e], pair(2.0f * kLog2e * factor, 2.0f * kLog2e * factor));
                  z[e] = add2(pair(capped(first_of(z[e]), p.cap_log2), capped(second_of(z[e]), p.cap_log2)), by[e]);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = mul2(z[e], factor2);
                capped2(z, p.cap_log2, by, most);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) z[e] = pair(ex2(first_of(z[e])), ex2(second_of(z[e])));
              if constexpr (MASK) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                  const int4 upto = limit[(first + x) / 4 + e / 2];
                  z[e] = pair(token < upto.x ? first_of(z[e]) : 0.0f, token < upto.y ? second_of(z[e]) : 0.0f);
                  z[e + 1] = pair(token < upto.z ? first_of(z[e + 1]) : 0.0f, token < upto.w ? second_of(z[e + 1]) : 0.0f);
                }
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) more[e & 1] = add2(more[e & 1], z[e]);
            }
          };
          const uint32_t from = ts + buf * kTile;
          if (n_cols <= 16) {
            Lane<16> f;
            ld(f, from);
            ld_wait(f);
            add(f, 0);
          } else {  // (columns past the last are masked)
            constexpr int N = CAP ? 16 : 32;  // capped scores take longer, and more registers
            Lane<N> f[2];
            ld(f[0], from);
            ld_wait(f[0]);
#pragma unroll 1
            for (int x = 0; x < n_cols; x += 2 * N) {
              if (x + N < n_cols) ld(f[1], from + x + N);
              add(f[0], x);
              if (x + N < n_cols) ld_wait(f[1]);
              if (x + 2 * N < n_cols) ld(f[0], from + x + 2 * N);
              if (x + N < n_cols) add(f[1], x + N);
              if (x + 2 * N < n_cols) ld_wait(f[0]);
            }
          }
          if constexpr (CAP && !WIDE) {
            if (__any_sync(0xffffffffu, most > 1.0f)) return false;
          }
          sum[0] = more[0], sum[1] = more[1];
          return true;
        };
        const std::true_type yes;
        const std::false_type no;
        if constexpr (!CAP) {
          if (masked) all(yes, no);
          else all(no, no);
        } else if (wide_step || !(masked ? all(yes, no) : all(no, no))) {
          wide_step = true;
          if (masked) all(yes, yes);
          else all(no, yes);
        }
        tc_before();
        if (!stalls(2) || warp != 0) warp_arrive(&s.s_empty[u][buf], lane);
        // (One chunk a sequence and head stays for all of its steps.)
        if (w.q.chunks > 1 || w.last) {
          warp_arrive(&s.q_empty[stage], lane);
          ++q_count;
        }
      }
      const float got = (first_of(sum[0]) + second_of(sum[0])) + (first_of(sum[1]) + second_of(sum[1]));
      const float mine = token >= w.q.seen ? 0.0f : !ok ? __uint_as_float(0x7fc00000u) : there ? got : 0.0f;
      if (w.whole()) {
        if (token < p.cap) p.out[at] = old + mine;
      } else {
        const int slot = 2 * blockIdx.x + (w.begun ? 0 : 1);
        p.part[(int64_t)slot * kPair + u * kTile + i] = mine;
        if (warp == 0 && lane == 0) p.part_of[slot] = make_int4(w.to == w.q.chunks ? 3 : 1, w.b, w.j, w.step);
      }
    }
  } else if (warp == 8) {
    // ---- matrix products ------------------------------------------------------------------------------
    const uint32_t q_u = smem_u32(q_stages), k_u = smem_u32(stages), mine = elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
    int q_count = 0, job = 0, tiles = 0;
    bool ok = true;
    for (Walk<G::kRows> w(p, s); w.more() && ok; w.next(p), tiles += 2) {
      for (int c = w.from; ok && c < w.to; ++c, ++job) {
        const int buf = job & 1, stage = q_count % kQStages;
        ok = wait_for(s, &s.q_full[stage], (q_count / kQStages) & 1);
        const uint32_t inst = instruction<false>((min(G::kRows, w.q.n_rows - c * G::kRows) + 15) / 16 * 16, false);
        for (int u = 0; ok && u < 2; ++u) {
          const int slot = (tiles + u) % kStages;
          if (c == w.from) ok = wait_for(s, &s.k_full[slot], ((tiles + u) / kStages) & 1);
          if (ok && job >= 2) ok = wait_for(s, &s.s_empty[u][buf], ((job >> 1) - 1) & 1);
          if (!ok) break;
          tc_after();
          const uint64_t a = desc_of(k_u + slot * G::kBytes, 16), b = desc_of(q_u + stage * G::kQBytes, 16);
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint32_t off = (x % 4) * 32;  // 16 channels further, or the next 64
            mma_ss(tm + u * 2 * kTile + buf * kTile, a + ((x / 4) * G::kHalfBytes + off) / 16, b + ((x / 4) * (G::kRows * 128) + off) / 16, inst, x > 0, mine);
          }
          commit(&s.s_full[u][buf], mine);
          if (c == w.to - 1) commit(&s.k_empty[slot], mine);
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
    auto look_up = [&](const Walk<G::kRows>& w) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int token = w.step * kPair + u * kTile + lane * bs;
        ahead[u] = w.more() && lane < per && token < w.q.seen ? p.table[w.b * p.table_ld + (token >> p.page_shift)] : -1;
      }
    };
    Walk<G::kRows> next(p, s);
    look_up(next);
    while (next.more() && ok) {
      const Walk<G::kRows> w = next;
      const int pages[2] = {ahead[0], ahead[1]};
      next.next(p);
      look_up(next);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int slot = filled % kSlots, page = pages[u] < p.n_pages ? pages[u] : -1;
        uint64_t* full = INT8 ? &s.raw_full[slot % 6] : &s.k_full[slot];
        if (filled >= kSlots) ok = ok && wait_for(s, INT8 ? &s.raw_empty[slot % 6] : &s.k_empty[slot], (filled / kSlots - 1) & 1);
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
    for (int n = max(0, filled - kSlots); n < filled; ++n) mbar_wait(INT8 ? &s.raw_full[n % kSlots % 6] : &s.k_full[n % kSlots], (n / kSlots) & 1);
    __syncwarp();
  } else if (warp < 12) {
    // ---- slots that no step covers: what was there goes on, new and missing tokens have nothing -----------
    const int64_t n = (int64_t)p.batch * p.h;
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
      const Sequence q = sequence_of<G::kRows>(p, (int)(row / p.h));
      const int go_on = min(q.old, q.seen);
      for (int64_t i = (int64_t)q.steps * kPair + tid - 10 * 32; i < p.cap; i += 64) {
        p.out[row * p.cap + i] = p.sums != nullptr && i < go_on ? p.sums[row * p.cap + i] : 0.0f;
      }
    }
  } else if (warp < 16) {
    // ---- queries: a thread has a row of the chunk ------------------------------------------------------
    const int r = tid % kTile;
    int q_count = 0;
    bool ok = true, here = false;  // here: the tile before had this sequence and head too
    for (Walk<G::kRows> w(p, s); w.more() && ok; w.next(p)) {
      const bool again = here;
      here = !w.last;
      if (w.q.chunks == 1 && again) continue;
      for (int c = w.from; c < w.to; ++c, ++q_count) {
        const int stage = q_count % kQStages, row = c * G::kRows + r;
        if (q_count >= kQStages) ok = wait_for(s, &s.q_empty[stage], (q_count / kQStages - 1) & 1);
        if (!ok) break;
        const bool live = r < G::kRows && row < w.q.n_rows;
        const int t = live ? row / p.group : 0, head = live ? w.j * p.group + row - t * p.group : 0;
        const __nv_bfloat16* src = p.q + (int64_t)(w.q.q0 + t) * p.q_st + (int64_t)head * p.q_sh;
        char* dst = q_stages + stage * G::kQBytes + r * 128;
        if (r < G::kRows && row < w.q.n_rows + 16) {  // (rows of the product past the last one: zeros)
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + (i / 8) * (G::kRows * 128) + (((i % 8) ^ (r & 7)) << 4))), "l"(src + 8 * i),
                         "r"(live ? 16 : 0)
                         : "memory");
        }
        const float lse = live ? p.lse[(int64_t)(w.q.q0 + t) * (p.h * p.group) + head] : -INFINITY;
        s.minus[stage][r] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
        s.limit[stage][r] = live && lse != -INFINITY ? w.q.limit + t : 0;
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        fence_async();
        if (!stalls(1) || warp != 12) warp_arrive(&s.q_full[stage], lane);
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
    for (Walk<G::kRows> w(p, s); w.more() && ok; w.next(p), n += 2) {
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

// Tiles whose chunks more than one CTA had: CTA c of the line began one and did not end it, the following ones have the
// others.
template <int kRows>
__global__ void __launch_bounds__(kPair) sums_merge_kernel(const SumsParams p) {
  pdl_wait();
  pdl_release();
  const int c = blockIdx.x;
  const int4 of = p.part_of[2 * c + 1];
  if (of.x == 0) return;
  const Sequence q = sequence_of<kRows>(p, of.y);
  const int token = of.w * kPair + threadIdx.x;
  const int64_t at = ((int64_t)of.y * p.h + of.z) * p.cap + token;
  float sum = p.part[(int64_t)(2 * c + 1) * kPair + threadIdx.x];
  for (int k = c + 1; k < (int)gridDim.x; ++k) {
    const int state = p.part_of[2 * k].x;
    if (state == 0) continue;  // (fewer jobs than CTAs: that one had none)
    sum += p.part[(int64_t)2 * k * kPair + threadIdx.x];
    if (state == 3) break;
  }
  if (token < p.cap) p.out[at] = (p.sums != nullptr && token < min(q.old, q.seen) ? p.sums[at] : 0.0f) + sum;
}

template <int D, bool INT8, bool CAP>
cudaError_t launch(const SumsParams& p, const CUtensorMap& map, int grid, cudaStream_t st) {
  using G = Geometry<D, INT8>;
  auto k = sums_kernel<D, INT8, CAP>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = prefix::allow_smem(k, G::kSmem, done);
  if (e == cudaSuccess) e = launch_pdl(k, dim3(grid), dim3(G::kThreads), G::kSmem, st, 0, p, map);
  // (Where all rows of the call are one chunk no tile is cut.)
  if (e == cudaSuccess && (int64_t)p.rows * p.group > G::kRows) e = launch_pdl(sums_merge_kernel<G::kRows>, dim3(grid), dim3(kPair), 0, st, 0, p);
  return e;
}

// One CTA per SM, or one per 256 slots (they write the slots that no job covers, too).
int grid_of(int cap, int batch, int h) { return (int)std::min<int64_t>(kNumSMs, ((int64_t)cap + kPair - 1) / kPair * h * batch); }
constexpr size_t kPartBytes = 2 * (kPair * sizeof(float) + sizeof(int4));  // of a CTA

uint64_t g_sums_wait_ns = kMaxTensorWaitNs;
int g_sums_stall_next = 0, g_sums_stall_cta = -1;

}  // namespace

int sums_set_wait(int64_t ns) {
  if (ns < 1 || ns > (int64_t)kMaxTensorWaitNs) return fail(LKV_ERR_ARG, "lkv_debug_set: sums wait bound %lld ns outside [1, %llu]", (long long)ns, (unsigned long long)kMaxTensorWaitNs);
  g_sums_wait_ns = (uint64_t)ns;
  return LKV_OK;
}
int sums_set_stall(int64_t which) {
  if (which < 0 || which > 2) return fail(LKV_ERR_ARG, "lkv_debug_set: no stall %lld of the attention sums (0, 1 or 2)", (long long)which);
  g_sums_stall_next = (int)which;
  return LKV_OK;
}
int sums_set_stall_cta(int64_t cta) {
  if (cta < -1 || cta > INT32_MAX) return fail(LKV_ERR_ARG, "lkv_debug_set: no CTA %lld of the attention sums (-1: all)", (long long)cta);
  g_sums_stall_cta = (int)cta;
  return LKV_OK;
}

cudaError_t sums_device_status(int* status, int clear) { return tu_device_status(status, clear); }
cudaError_t sums_status_attach(int* mirror) { return tu_status_attach(mirror); }

}  // namespace lkv

using namespace lkv;

extern "C" size_t lkv_attention_sums_workspace(int batch, int h, int cap) {
  return batch <= 0 || h <= 0 || cap <= 0 ? 0 : grid_of(cap, batch, h) * kPartBytes;
}

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
  if (!scores_fit(a->scale, a->cap_scores)) return fail(LKV_ERR_ARG, "%s: scale %g with cap %g leaves float32", who, (double)a->scale, (double)a->cap_scores);
  const int64_t page_rows = a->n_pages * 2 * a->h * a->bs;
  if (page_rows > INT32_MAX) return fail(LKV_ERR_ARG, "%s: %lld rows of pages", who, (long long)page_rows);
  if (a->batch == 0 || a->cap == 0) return LKV_OK;
  if (a->lens == nullptr || a->offsets == nullptr || a->out == nullptr || (a->table == nullptr && a->table_cols > 0) || (a->rows > 0 && (a->q == nullptr || a->lse == nullptr)))
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(a->q, 16) || (a->q_st & 7) != 0 || (a->q_sh & 7) != 0) return fail(LKV_ERR_PTR, "%s: query rows must be 16-byte aligned", who);
  if (!aligned(a->scales, 16)) return fail(LKV_ERR_PTR, "%s: scales must be 16-byte aligned", who);
  const int grid = grid_of(a->cap, a->batch, a->h);
  if (a->workspace == nullptr || a->workspace_bytes < grid * kPartBytes) return fail(LKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, grid * kPartBytes);
  if (!aligned(a->workspace, 16)) return fail(LKV_ERR_PTR, "%s: workspace must be 16-byte aligned", who);
  SumsParams p = {};
  p.part_of = static_cast<int4*>(a->workspace);
  p.part = reinterpret_cast<float*>(p.part_of + 2 * grid);
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.q_st = a->q_st, p.q_sh = a->q_sh, p.lse = a->lse;
  p.pages = a->pages, p.scales = a->scales, p.n_pages = (int)a->n_pages, p.page_shift = shift_of(a->bs);
  p.rows = a->rows, p.batch = a->batch, p.h = a->h, p.group = group;
  p.table = a->table, p.table_ld = a->table_ld, p.table_cols = a->table_cols, p.lens = a->lens, p.offsets = a->offsets;
  p.last = a->last, p.sums = a->sums, p.out = a->out, p.cap = a->cap;
  const bool cap = a->cap_scores > 0.0f;
  p.scale = cap ? a->scale / a->cap_scores : a->scale * kLog2e;
  p.cap_log2 = a->cap_scores * kLog2e;
  p.max_wait_ns = g_sums_wait_ns;
  p.stall = g_sums_stall_next, p.stall_cta = g_sums_stall_cta;
  g_sums_stall_next = 0;
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
