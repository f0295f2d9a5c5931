// Verification of drafted tokens against the target's probabilities, with the random numbers given.
//
// Per sequence: token i of the k drafted is kept while u_i q_i(x_i) < p_i(x_i) (that is, with
// probability min(1, p / q)); the product of two float32 is exact in float64, so the comparison is too.
// Let n be the number kept. The next token is drawn by inverting the cumulative sum of the weights
//   w_v = max(p_n(v) - q_n(v), 0) after a rejection, w_v = p_n(v) where every drafted token was kept:
// the least v with w_0 + ... + w_v > u_k (w_0 + ... + w_{V-1}). Together the kept tokens and the drawn
// one are distributed as samples of the target. Differences and sums are float64: a vocabulary's
// float32 sum would move the border between neighbouring tokens by more than a token's own weight.
//
// Only one row (or pair of rows) of the vocabulary is read per sequence: one cluster of CTAs per
// sequence, a slice of the row each. A slice's sums per tile of 512 stay in shared
// memory, the cluster exchanges the slices' totals, and the CTA whose slice holds the border finds the
// tile, then reads that tile once more and finds the element.
//
// Measured: 64 sequences, 7 drafted, a vocabulary of 128,256: 20 us, 3.3 TB/s (the floor at a copy's rate is
// 10 us): one wave of reads stands between the chain that decides n (three loads in turn) and two cluster
// barriers, and is not overlapped with either. One sequence, 4 drafted, 32,000: 7.5 us, those chains alone.
#include <cooperative_groups.h>

#include "common.cuh"

namespace lkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 512;        // elements a warp sums at a time
constexpr int kMaxTiles = 1024;   // tile sums a CTA keeps
constexpr double kBelowOne = 0.99999999999999988897769753748;  // 1 - 2^-53

struct VerifyParams {
  const float* target;  // [b, k + 1, v], element strides
  int64_t p_sb, p_st;
  const float* draft;  // [b, k, v] or null: the draft proposed its token with certainty
  int64_t q_sb, q_st;
  const int64_t* tokens;  // [b, k]
  int64_t t_sb;
  const float* uniforms;  // [b, k + 1]
  int64_t u_sb;
  int k, vocab;
  int per_cta;     // elements of a CTA's slice, a multiple of kTile
  int32_t* kept;   // [b]
  int64_t* token;  // [b]
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The weight of element v; a NaN weighs nothing.
struct Weights {
  const float* p;
  const float* q;  // null: p alone, without `struck`
  int64_t struck;  // the rejected token of a draft without probabilities, or -1
  int vocab;
  __device__ __forceinline__ double one(float a, float b, int v) const {
    if (v == struck) return 0.0;
    return fmax((double)a - (double)b, 0.0);
  }
  __device__ __forceinline__ double at(int v) const { return v < vocab ? one(p[v], q != nullptr ? q[v] : 0.0f, v) : 0.0; }
};

template <bool VEC>
__device__ __forceinline__ double tile_sum(const Weights& w, int base, int lane) {
  double s = 0.0;
  if (VEC && base + kTile <= w.vocab && (w.struck < base || w.struck >= base + kTile)) {
    float4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = reinterpret_cast<const float4*>(w.p + base)[i * 32 + lane];
    if (w.q != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = reinterpret_cast<const float4*>(w.q + base)[i * 32 + lane];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // A positive difference of two float32 as d + r, exactly: d rounded, r what that lost. The d are summed
    // in float64, the r, 2^-24 of them, in float32: half the conversions, and 2^-48 of the sum is still there.
    float lost = 0.0f;
    auto add = [&](float x, float y) {
      const float d = x - y;
      if (d > 0.0f) {
        s += (double)d;
        lost += (x - d) - y;
      }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) add(a[i].x, b[i].x), add(a[i].y, b[i].y), add(a[i].z, b[i].z), add(a[i].w, b[i].w);
    s += (double)lost;
  } else {
    for (int i = lane; i < kTile; i += 32) s += w.at(base + i);
  }
  return warp_sum(s);
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(const VerifyParams p) {
  __shared__ double tiles[kMaxTiles];
  __shared__ double total;
  __shared__ int first_bad;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_ranks = (int)cluster.num_blocks();
  const int b = blockIdx.x / n_ranks;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  pdl_wait();
  pdl_release();
  // How many drafted tokens are kept (every CTA of the cluster for itself).
  if (tid == 0) first_bad = p.k;
  __syncthreads();
  for (int i = tid; i < p.k; i += kThreads) {
    const int64_t x = p.tokens[b * p.t_sb + i];
    bool keep = x >= 0 && x < p.vocab;
    if (keep) {
      const double px = p.target[b * p.p_sb + i * p.p_st + x];
      const double qx = p.draft == nullptr ? 1.0 : (double)p.draft[b * p.q_sb + i * p.q_st + x];
      keep = (double)p.uniforms[b * p.u_sb + i] * qx < px;
    }
    if (!keep) atomicMin(&first_bad, i);
  }
  __syncthreads();
  const int n = first_bad;
  Weights w;
  w.p = p.target + b * p.p_sb + n * p.p_st;
  w.q = nullptr;
  w.struck = -1;
  w.vocab = p.vocab;
  if (n < p.k) {
    const int64_t x = p.tokens[b * p.t_sb + n];
    if (x >= 0 && x < p.vocab) {  // otherwise the sequence has no more drafted tokens: as if all were kept
      if (p.draft != nullptr) w.q = p.draft + b * p.q_sb + n * p.q_st;
      else w.struck = x;
    }
  }
  const int lo = min((int64_t)rank * p.per_cta, (int64_t)p.vocab), hi = min((int64_t)lo + p.per_cta, (int64_t)p.vocab);
  const int n_tiles = (hi - lo + kTile - 1) / kTile;
  double before = 0.0, all = 0.0, mine = 0.0;
  for (int pass = 0;; ++pass) {
    for (int i = warp; i < n_tiles; i += kWarps) {
      const double s = tile_sum<VEC>(w, lo + i * kTile, lane);
      if (lane == 0) tiles[i] = s;
    }
    __syncthreads();
    if (warp == 0) {
      double s = 0.0;
      for (int i = lane; i < n_tiles; i += 32) s += tiles[i];
      s = warp_sum(s);
      if (lane == 0) total = s;
    }
    cluster.sync();
    before = all = 0.0;
    for (int r = 0; r < n_ranks; ++r) {
      const double s = *cluster.map_shared_rank(&total, r);
      if (r == rank) before = all, mine = s;
      all += s;
    }
    cluster.sync();
    // Where the draft's row covers the target's everywhere, nothing is left: the target's own row.
    if (all > 0.0 || pass > 0 || (w.q == nullptr && w.struck < 0)) break;
    w.q = nullptr;
    w.struck = -1;
  }
  if (rank == 0 && tid == 0) p.kept[b] = n;
  if (!(all > 0.0 && all < (double)INFINITY)) {  // no weight at all, or no finite sum of them
    if (rank == 0 && tid == 0) p.token[b] = -1;
    return;
  }
  const double at = fmin(fmax((double)p.uniforms[b * p.u_sb + p.k], 0.0), kBelowOne) * all;
  const bool last = rank == n_ranks - 1;
  if (warp != 0 || !(at >= before && (at < before + mine || last))) return;
  // This CTA's slice holds the border. Lanes take consecutive tiles, then consecutive elements. Sums in another order
  // may round to the border's other side: only what weighs something is ever taken, and the last of it where no
  // sum passes the border.
  double base = before;
  int tile = 0;
  const int share = (n_tiles + 31) / 32;
  {
    double s = 0.0;
    for (int i = lane * share; i < min((lane + 1) * share, n_tiles); ++i) s += tiles[i];
    double upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, s > 0.0), over = some & __ballot_sync(0xffffffffu, before + upto > at);
    const int who = over != 0 ? __ffs(over) - 1 : 31 - __clz(some);
    double run = before + __shfl_sync(0xffffffffu, upto - s, who);
    for (int i = who * share; i < min((who + 1) * share, n_tiles); ++i) {
      if (!(tiles[i] > 0.0)) continue;
      tile = i;
      base = run;
      run += tiles[i];
      if (run > at) break;
    }
  }
  const int first = lo + tile * kTile + lane * (kTile / 32);
  double x[kTile / 32], s = 0.0;
#pragma unroll
  for (int i = 0; i < kTile / 32; ++i) {
    x[i] = first + i < hi ? w.at(first + i) : 0.0;
    s += x[i];
  }
  double upto = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  int found = -1, heaviest = -1;
  double run = base + (upto - s);
#pragma unroll
  for (int i = 0; i < kTile / 32; ++i) {
    run += x[i];
    if (x[i] > 0.0) {
      heaviest = first + i;
      if (found < 0 && run > at) found = first + i;
    }
  }
  const uint32_t hit = __ballot_sync(0xffffffffu, found >= 0);
  const uint32_t any = __ballot_sync(0xffffffffu, heaviest >= 0);
  const int who = hit != 0 ? __ffs(hit) - 1 : any != 0 ? 31 - __clz(any) : 0;
  if (lane == who) p.token[b] = found >= 0 ? found : heaviest;
}

}  // namespace
}  // namespace lkv

using namespace lkv;

extern "C" {

int lkv_verify_drafts(const lkv_verify_args* a, void* stream) {
  if (a == nullptr) return fail(LKV_ERR_PTR, "lkv_verify_drafts: null arguments");
  const int batch = a->batch, vocab = a->vocab;
  if (batch < 0 || a->k < 0 || vocab < 1 || vocab > (1 << 22))
    return fail(LKV_ERR_ARG, "lkv_verify_drafts: bad shape (batch %d, drafted %d, vocabulary %d of at most 4,194,304)", batch, a->k, vocab);
  if (batch == 0) return LKV_OK;
  if (a->target == nullptr || (a->k > 0 && a->tokens == nullptr) || a->uniforms == nullptr || a->kept == nullptr || a->token == nullptr)
    return fail(LKV_ERR_PTR, "lkv_verify_drafts: null pointer");
  if (!aligned(a->target, 4) || !aligned(a->draft, 4) || !aligned(a->tokens, 8) || !aligned(a->uniforms, 4) || !aligned(a->kept, 4) || !aligned(a->token, 8))
    return fail(LKV_ERR_PTR, "lkv_verify_drafts: misaligned pointer");
  // As many CTAs per sequence (a power of two, 8 at most) as keep all of them resident at four to an
  // SM, and no more than a slice of one tile per warp fills; always enough that the tile sums fit.
  int c = 1;
  while (c < 8 && (int64_t)batch * c * 2 <= 4 * kNumSMs && (int64_t)kTile * kWarps * c < vocab) c *= 2;
  while (c < 8 && (int64_t)kTile * kMaxTiles * c < vocab) c *= 2;
  VerifyParams p = {};
  p.target = a->target;
  p.p_sb = a->p_sb, p.p_st = a->p_st;
  p.draft = a->draft;
  p.q_sb = a->q_sb, p.q_st = a->q_st;
  p.tokens = a->tokens;
  p.t_sb = a->t_sb;
  p.uniforms = a->uniforms;
  p.u_sb = a->u_sb;
  p.k = a->k;
  p.vocab = vocab;
  p.per_cta = ((vocab + c - 1) / c + kTile - 1) / kTile * kTile;
  p.kept = a->kept;
  p.token = a->token;
  if ((int64_t)batch * c > INT32_MAX) return fail(LKV_ERR_ARG, "lkv_verify_drafts: batch of %d", batch);
  const bool vec = aligned(a->target, 16) && a->p_sb % 4 == 0 && a->p_st % 4 == 0 &&
                   (a->draft == nullptr || (aligned(a->draft, 16) && a->q_sb % 4 == 0 && a->q_st % 4 == 0));
  const cudaError_t e = vec ? launch_pdl(verify_kernel<true>, dim3((unsigned)(batch * c)), dim3(kThreads), 0, as_stream(stream), c, p)
                            : launch_pdl(verify_kernel<false>, dim3((unsigned)(batch * c)), dim3(kThreads), 0, as_stream(stream), c, p);
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "lkv_verify_drafts: %s", cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
