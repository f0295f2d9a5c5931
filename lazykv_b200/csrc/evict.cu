// A budget for a paged cache's own tokens: per sequence and KV head, the tokens of the highest sums are kept
// (attention_sums accumulates them), the protected ones first, ties to the lowest slot.
//
// A sequence's n tokens lie in slots 0 .. n - 1 of its pages and shall lie in slots 0 .. keep - 1. Of the
// tokens kept, those in front of slot `keep` stay where they are; the i-th of those behind it moves into the
// i-th slot in front that loses its token. Attention does not ask for an order of the slots (positions are
// turned into the keys), so nothing else has to move, and as sources lie behind all destinations, no row is
// overwritten that is still to be read.
//
// One cluster of 1 to 8 CTAs per (sequence, head), one launch: keys (sums as whole numbers of the same order)
// into shared memory, the keep-th largest by three counted digits (11, 11 and 10 bits) whose counts the CTAs
// add up over distributed shared memory, then ranks of ties, of slots that lose and of tokens that move by
// ballots in slot order, and the copies.
//
// Measured: 8 heads of 40,001 tokens down to 5,000, d 128, int8: 37 us, a third of it the copies (4,375 tokens a head); 64
// sequences of 8 heads from up to 1,040 to 1,024, bf16: 14 us. The chain of barriers and dependent loads bounds both.
#include <cooperative_groups.h>

#include <atomic>

#include "paged.cuh"

namespace lkv {
namespace {

using namespace paged;
namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMostKeys = 16384;  // keys of a CTA's slots that shared memory holds; of longer slices they are computed again
constexpr int kMovesAtOnce = 8;   // of a warp
constexpr int kMostRanks = 8;     // CTAs of a cluster

struct EvictParams {
  void* pages;
  float* scales;
  int64_t n_pages;
  int page_shift, h;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* lens;
  const float* sums;
  const int32_t* positions;
  int cap;
  float* out_sums;
  int32_t* out_positions;
  int32_t* out_lens;
  int keep, sinks;
  const int32_t* since;
  int2* moves;  // [batch * h][max_moves]: (from, to)
  int max_moves;
  int cached;  // keys that the launch's shared memory has room for
};

struct Shared {
  alignas(16) uint32_t hist[3][kBins];
  uint32_t scan[kWarps];
  uint32_t digit, left;
  uint32_t ties[kWarps], all_ties;
  uint2 moving[kWarps], all_moving;  // slots that lose their token, tokens that move
};

// Row `slot` of the sequence's keys of head j (its values bs rows further), or -1.
__device__ __forceinline__ int64_t row_of(const EvictParams& p, int b, int j, int slot) {
  const int64_t id = p.table[(int64_t)b * p.table_ld + (slot >> p.page_shift)];
  const int bs = 1 << p.page_shift;
  return id < 0 || id >= p.n_pages ? -1 : (id * p.h + j) * 2 * bs + (slot & (bs - 1));
}

// Bytes per row of pages.
template <int RB>
__global__ void __launch_bounds__(kThreads) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ Shared s;
  pdl_wait();
  pdl_release();
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), n_ranks = cluster.num_blocks();
  auto sync = [&] {
    if (n_ranks == 1) __syncthreads();
    else cluster.sync();
  };
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int row = blockIdx.x / n_ranks, b = row / p.h, j = row % p.h;
  const int n = (int)max((int64_t)0, min((int64_t)p.lens[b], min((int64_t)p.cap, (int64_t)p.table_cols << p.page_shift)));
  const int left = min(n, p.keep);
  const float* sums = p.sums + (int64_t)row * p.cap;
  const int32_t* positions = p.positions + (int64_t)row * p.cap;
  float* out_sums = p.out_sums + (int64_t)row * p.cap;
  int32_t* out_positions = p.out_positions + (int64_t)row * p.cap;
  if (j == 0 && rank == 0 && tid == 0) p.out_lens[b] = left;
  auto clear = [&] {
    for (int i = left + rank * kThreads + tid; i < p.cap; i += n_ranks * kThreads) out_sums[i] = 0.0f, out_positions[i] = -1;
  };
  if (n <= p.keep) {
    for (int i = rank * kThreads + tid; i < n; i += n_ranks * kThreads) out_sums[i] = sums[i], out_positions[i] = positions[i];
    clear();
    return;
  }

  // This CTA's slots lo .. hi - 1, and each warp's.
  const int span = ((n + n_ranks - 1) / n_ranks + 31) / 32 * 32, lo = min(n, rank * span), hi = min(n, lo + span);
  const int warp_span = ((span + kWarps - 1) / kWarps + 31) / 32 * 32, w_lo = min(hi, lo + warp * warp_span), w_hi = min(hi, w_lo + warp_span);
  const int since = p.since != nullptr ? p.since[b] : 0x7fffffff;
  const bool has_since = p.since != nullptr, cached = span <= p.cached;
  auto compute = [&](int i) {
    const float x = sums[i];
    const int at = positions[i];
    if (at < p.sinks || (has_since && at >= since)) return 0xffffffffu;
    return isnan(x) ? 0u : orderable(x);
  };
  for (int i = tid; i < 3 * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
  if (cached) {
    for (int i = lo + tid; i < hi; i += kThreads) keys[i - lo] = compute(i);
  }
  __syncthreads();
  auto key = [&](int i) { return cached ? keys[i - lo] : compute(i); };

  // The keep-th largest key, digit by digit.
  uint32_t found = 0, want = p.keep;  // the digits so far; how many of the keys that share them are kept
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above = pass == 0 ? 32 : pass == 1 ? 21 : 10;
    for (int i = lo + tid; i < hi; i += kThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> above) == found) atomicAdd(&s.hist[pass][(k >> shift) & (pass == 2 ? 1023u : 2047u)], 1u);
    }
    sync();
    // Thread t has the four bins 2047 - 4 t and below.
    uint32_t count[4] = {0, 0, 0, 0};
    uint4 of[kMostRanks];  // (asked for together: another CTA's shared memory is a microsecond away)
#pragma unroll
    for (int r = 0; r < kMostRanks; ++r)
      if (r < n_ranks) of[r] = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s.hist[pass][kBins - 4 - 4 * tid], r));
#pragma unroll
    for (int r = 0; r < kMostRanks; ++r)
      if (r < n_ranks) count[0] += of[r].w, count[1] += of[r].z, count[2] += of[r].y, count[3] += of[r].x;
    const uint32_t mine = count[0] + count[1] + count[2] + count[3];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.scan[warp] = upto;
    __syncthreads();
    uint32_t before = upto - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) before += w < warp ? s.scan[w] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < want && want <= before + count[i]) s.digit = kBins - 1 - 4 * tid - i, s.left = want - before;
      before += count[i];
    }
    __syncthreads();
    found = pass == 2 ? (found << 10) | s.digit : (found << 11) | s.digit;
    want = s.left;
  }

  // Of the keys that equal it, the first `want` are kept: ties before each warp's slots.
  uint32_t ties = 0;
  for (int i = w_lo + lane; i - lane < w_hi; i += 32) ties += __popc(__ballot_sync(0xffffffffu, i < w_hi && key(i) == found));
  if (lane == 0) s.ties[warp] = ties;
  __syncthreads();
  if (tid == 0) {
    uint32_t sum = 0;
    for (int w = 0; w < kWarps; ++w) sum += s.ties[w];
    s.all_ties = sum;
  }
  sync();
  uint32_t tie_base = 0;
#pragma unroll
  for (int r = 0; r < kMostRanks; ++r) tie_base += r < rank ? *cluster.map_shared_rank(&s.all_ties, r) : 0u;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) tie_base += w < warp ? s.ties[w] : 0u;

  // Which slots in front of `keep` lose their token and which tokens behind it stay, in slot order; `use` gets
  // each slot with its token's fate.
  const uint32_t below = (1u << lane) - 1;
  auto walk = [&](auto&& use) {
    uint32_t tie = tie_base;
    for (int i = w_lo + lane; i - lane < w_hi; i += 32) {
      const uint32_t k = i < w_hi ? key(i) : 0;
      const uint32_t equal = __ballot_sync(0xffffffffu, i < w_hi && k == found);
      const bool kept = i < w_hi && (k > found || (k == found && tie + __popc(equal & below) < want));
      use(i, kept, __ballot_sync(0xffffffffu, i < w_hi && !kept && i < p.keep), __ballot_sync(0xffffffffu, kept && i >= p.keep));
      tie += __popc(equal);
    }
  };
  uint2 moving = make_uint2(0, 0);
  walk([&](int, bool, uint32_t lose, uint32_t move) { moving.x += __popc(lose), moving.y += __popc(move); });
  if (lane == 0) s.moving[warp] = moving;
  __syncthreads();
  if (tid == 0) {
    uint2 sum = make_uint2(0, 0);
    for (int w = 0; w < kWarps; ++w) sum.x += s.moving[w].x, sum.y += s.moving[w].y;
    s.all_moving = sum;
  }
  sync();
  uint2 base = make_uint2(0, 0);
  uint32_t n_moves = 0;
#pragma unroll
  for (int r = 0; r < kMostRanks; ++r) {
    const uint2 x = r < n_ranks ? *cluster.map_shared_rank(&s.all_moving, r) : make_uint2(0, 0);
    if (r < rank) base.x += x.x, base.y += x.y;
    n_moves += x.x;
  }
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) base.x += s.moving[w].x, base.y += s.moving[w].y;
  int2* moves = p.moves + (int64_t)row * p.max_moves;
  walk([&](int i, bool kept, uint32_t lose, uint32_t move) {
    if (lose >> lane & 1) moves[base.x + __popc(lose & below)].y = i;
    if (move >> lane & 1) moves[base.y + __popc(move & below)].x = i;
    base.x += __popc(lose), base.y += __popc(move);
    if (kept && i < p.keep) out_sums[i] = sums[i], out_positions[i] = positions[i];
  });
  sync();

  constexpr int kChunks = RB / 16, kPer = 2 * kChunks;  // 16-byte pieces of a row, of a token's key and value
  const int bs = 1 << p.page_shift;
  char* pages = static_cast<char*>(p.pages);
  for (int at = (rank * kWarps + warp) * kMovesAtOnce; at < (int)n_moves; at += n_ranks * kWarps * kMovesAtOnce) {
    int64_t from = -1, to = -1;
    if (lane < kMovesAtOnce && at + lane < (int)n_moves) {
      const int2 m = moves[at + lane];
      out_sums[m.y] = sums[m.x], out_positions[m.y] = positions[m.x];
      from = row_of(p, b, j, m.x), to = row_of(p, b, j, m.y);
      if (from < 0 || to < 0) from = to = -1;  // without either page there is no row to move (its sum and position have)
    }
    if (p.scales != nullptr && to >= 0) {
      const float ks = p.scales[from], vs = p.scales[from + bs];
      p.scales[to] = ks, p.scales[to + bs] = vs;
    }
    constexpr int kIters = kMovesAtOnce * kPer / 32;
    uint4 x[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int q = i * 32 + lane, c = q % kPer;
      const int64_t r = __shfl_sync(0xffffffffu, from, q / kPer);
      if (r >= 0) x[i] = *reinterpret_cast<const uint4*>(pages + (r + (c / kChunks) * bs) * RB + (c % kChunks) * 16);
    }
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int q = i * 32 + lane, c = q % kPer;
      const int64_t r = __shfl_sync(0xffffffffu, to, q / kPer);
      if (r >= 0) *reinterpret_cast<uint4*>(pages + (r + (c / kChunks) * bs) * RB + (c % kChunks) * 16) = x[i];
    }
  }
  sync();  // (in place, the tail's sums are read by the moves)
  clear();
}

template <int RB>
cudaError_t launch(const EvictParams& p, int rows, int n_ranks, cudaStream_t st) {
  auto k = evict_kernel<RB>;
  static std::atomic<uint64_t> done{0};  // devices that have been asked for the shared memory, a bit each
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostKeys * 4);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_pdl(k, dim3((unsigned)rows * n_ranks), dim3(kThreads), (size_t)p.cached * 4, st, n_ranks, p);
}

}  // namespace
}  // namespace lkv

using namespace lkv;

extern "C" {

size_t lkv_paged_evict_workspace(int batch, int h, int cap, int keep) {
  if (batch <= 0 || h <= 0 || keep < 0 || cap <= keep) return 0;
  const size_t most = keep < cap - keep ? keep : cap - keep;
  return (size_t)batch * h * most * sizeof(int2);
}

int lkv_paged_evict(const lkv_evict_args* a, void* stream) {
  static const char* who = "lkv_paged_evict";
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (int rc = check_cache(who, a->kind, a->dtype, a->h, a->bs, a->d, a->n_pages, a->pages, a->scales)) return rc;
  if (a->batch < 0 || a->cap < 0 || a->cap > (1 << 30) || a->table_cols < 0 || (a->batch > 1 && a->table_ld < a->table_cols) || (int64_t)a->batch * a->h > INT32_MAX / 8)
    return fail(LKV_ERR_ARG, "%s: bad shape (batch %d, %d slots, table of %d columns)", who, a->batch, a->cap, a->table_cols);
  if (a->keep < 1) return fail(LKV_ERR_ARG, "%s: a budget of %d tokens", who, a->keep);
  if (a->batch == 0) return LKV_OK;
  if (a->lens == nullptr || a->out_lens == nullptr || (a->table == nullptr && a->table_cols > 0) ||
      (a->cap > 0 && (a->sums == nullptr || a->positions == nullptr || a->out_sums == nullptr || a->out_positions == nullptr)))
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (a->lens == a->out_lens) return fail(LKV_ERR_PTR, "%s: the lengths left cannot replace the lengths in place", who);
  const size_t need = lkv_paged_evict_workspace(a->batch, a->h, a->cap, a->keep);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return fail(LKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, need);
  if (!aligned(a->workspace, 8)) return fail(LKV_ERR_PTR, "%s: misaligned workspace", who);
  EvictParams p = {};
  p.pages = a->pages;
  p.scales = a->kind == LKV_CACHE_INT8 ? a->scales : nullptr;
  p.n_pages = a->n_pages;
  p.page_shift = shift_of(a->bs), p.h = a->h;
  p.table = a->table, p.table_ld = a->table_ld, p.table_cols = a->table_cols;
  p.lens = a->lens, p.sums = a->sums, p.positions = a->positions, p.cap = a->cap;
  p.out_sums = a->out_sums, p.out_positions = a->out_positions, p.out_lens = a->out_lens;
  p.keep = a->keep, p.sinks = a->sinks, p.since = a->since;
  p.moves = static_cast<int2*>(a->workspace);
  p.max_moves = (int)(need / ((size_t)a->batch * a->h * sizeof(int2)));
  // CTAs of a cluster: as many as leave each some 2,048 slots, while the GPU has room for them.
  const int rows = a->batch * a->h;
  int n_ranks = 1;
  while (n_ranks < kMostRanks && a->cap / n_ranks > 2048 && (int64_t)rows * n_ranks < 2 * kNumSMs) n_ranks *= 2;
  const int span = (int)(((int64_t)a->cap + n_ranks - 1) / n_ranks + 31) / 32 * 32;
  p.cached = span <= kMostKeys ? span : 0;
  const int rb = a->d * (a->kind == LKV_CACHE_INT8 ? 1 : (int)dtype_size(a->dtype));
  cudaStream_t st = as_stream(stream);
  const cudaError_t e = rb == 64    ? launch<64>(p, rows, n_ranks, st)
                        : rb == 128 ? launch<128>(p, rows, n_ranks, st)
                        : rb == 256 ? launch<256>(p, rows, n_ranks, st)
                                    : launch<512>(p, rows, n_ranks, st);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
