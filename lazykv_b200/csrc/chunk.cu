// Attention of chunks of new tokens over a paged cache (and a prefix that the sequences share), on the
// 5th-generation tensor cores.
//
// A sequence's n new tokens have n G query rows per KV head (G query heads share it); row r is token r / G. A
// unit of work is a block of up to 256 rows of one sequence and KV head against the tokens that its last row
// sees, 128 at a time: the prefix's tiles, then the sequence's own. All units, in the order sequence, head,
// block, are one line of tiles of which every CTA takes an equal piece: nobody waits for the longest sequence or
// for the late blocks of a causal chunk, and a single short chunk over a long cache still uses every SM. A CTA
// finishes the units that lie whole in its piece; of the one it begins with and the one it ends with it may hold
// a part, whose rows' (m, l, o) chunk_merge_kernel folds together. Lengths are read on the device.
//
// In a CTA two tiles of 128 rows take turns, so that one computes weights while the tensor cores work for the
// other: S = Q K^T (tcgen05.mma, operands in shared memory, S in tensor memory); w = 2^(s - m) in registers,
// float32, m the row's reference (set anew only when weights outgrow 2^20); w as bf16 over S; O += w V. With 128
// rows or fewer both tiles are the same queries and take the tiles of tokens by turns; they are joined at the end.
// Warps 0-3 and 4-7 are the two tiles' rows, warp 8 issues the products, warp 9 the copies, warp 10 walks the
// line, warp 11 cleans values (below); with int8 pages warps 12-15 turn codes of keys into bf16 operands, 16-19
// those of values into f16. mbarriers join them, every wait bounded.
//
// Roundings: scores, references, sums are float32; a weight is rounded once, and the output to bf16. bf16 pages: the
// weight to bf16, 2^-8 of it at most, since both operands of a product have one type and values need bf16's
// range; a second term would cost a third of the time (prefix_tile.cu has it for float32 outputs). int8 pages: the weight
// times its value's scale to f16, 2^-11 of it (and 2^-31 of the row's largest; prefix.cuh, kScaleShift), in which codes are
// exact too. Codes, and bf16 queries, keys and values, are exact operands. Capped scores are c tanh(x / c), by a polynomial while a warp's scores of a tile stay within the cap,
// and otherwise by exponentials (scores.cuh).
//
// Masks: a row sees a token if its page exists and the token is in front of the row's limit. Weights of others are
// zero, but 0 x infinity is a NaN, and a tile's values multiply all of its rows: in tiles that some row does not see
// whole, values that are not finite are taken out of the operand (warp 11) and, where there were any, added to
// the rows that do see them at the end.
//
// Measured (8 KV heads, 4 query heads each, d 128): 4,096 tokens on 32,768 in 2,050 us in a short burst, 1.14 PFLOP/s (2,400 under
// the power cap, 0.97); 2,048 on 16,384 int8 777 us (770 with weights of int8 pages in bf16, 2^-8). A row tile's period of 3,800 cycles a tile: its weights 1,830 (1,290 alone: the
// other row tile's exponentials share the unit), 320 until the products' warp has seen them, 960 for the two products, and the
// waits between; products alone would take 1,760 us of the 2,050, weights alone 1,790.
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
using prefix::kLn2;
using prefix::kLog2e;
using prefix::kMostF16;
using prefix::kScaleDown;
using prefix::kScaleShift;
using prefix::pack_bf16;
using prefix::pack_f16;
using prefix::scaled_room;
using prefix::scaled_top;
using prefix::times_ex2;

constexpr int kBlock = 2 * kTile;  // rows of a unit
constexpr int kInfo = 8;           // tiles whose scales and page bits are kept (see the copies)
constexpr int kRing = 4;           // units that are handed out ahead
constexpr int kClean = 8;          // tiles to be cleaned or cleaned ahead of their product: more than the stages hold
constexpr int kPad = 1;            // a unit's start and end count as this many tiles more on the line
constexpr int kMinShare = 2;       // tiles of the line that a CTA takes at least
constexpr int kMostBatch = 8192;
constexpr int kLost = 4;           // of a part: its CTA gave up a wait, it may hold anything
constexpr float kMostWeight = 1048576.0f;  // 2^20: what the sum of a thread's weights of bf16 pages may grow to before its references are set again

struct ChunkParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const void* pages;
  const float* scales;
  int n_pages, page_shift;
  int rows, batch, h, group;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t* lens;
  const int32_t* offsets;
  const int32_t* prefix_table;
  int prefix_cols, prefix_len;
  float scale;     // scores x this are in the log2 domain (capped: scores divided by the cap); not negative
  uint32_t flip;   // the queries' sign bits to turn (a negative softmax scale)
  float cap_log2;  // cap x log2(e)
  __nv_bfloat16* out;  // [rows, hq, d]
  float* lse;          // [rows, hq]
  // Parts of units, two slots a CTA: 2 c the unit it begins in the middle of, 2 c + 1 the one it does not end.
  float* part_o;    // [slots][kBlock][d], not divided by the sum
  float2* part_ml;  // [slots][kBlock]: (reference in the log2 domain, sum)
  int4* part_of;    // [slots]: (1: a part, 3: the unit's last, + kLost: not to be used), sequence, head, first row
  uint64_t max_wait_ns;
  int stall, stall_cta;  // test hook: warp 0 of this CTA (-1: of every CTA) withholds an arrival
};

// A place in a ring of n entries, and how often it was filled before.
struct Cursor {
  int slot, round;
  __device__ __forceinline__ uint32_t phase() const { return round & 1; }
  __device__ __forceinline__ void step(int by, int n) {
    slot += by;
    if (slot >= n) slot -= n, ++round;
  }
};

// A piece of a unit.
struct Unit {
  int b, j;          // sequence, KV head; b < 0: the end
  int row0, n_rows;  // of the sequence's rows
  int t0, n_tiles;   // tiles of the prefix and of own tokens, in this order
  int base;          // own tokens in front of the chunk (lens - n)
  int seen;          // own tokens that the last row sees, as far as the table reaches
  int q0;            // the chunk's first packed row
  int slot;          // of its part, or -1: the whole unit
};

template <int D, bool INT8>
struct Tiles {
  static constexpr int kHalves = D / 64;                // 64 channels (128 bytes) per swizzled column
  static constexpr int kHalfBytes = kTile * 128;
  static constexpr int kBytes = kHalves * kHalfBytes;   // one operand tile
  static constexpr int kStages = INT8 ? (D == 128 ? 3 : 6) : (D == 128 ? 5 : 8);
  static constexpr int kRawBytes = INT8 ? kTile * D : 0;
  // Codes under way: a ring for keys and one for values. (One ring for both would give a place to the two warpgroups that turn
  // codes into operands by turns; each waits for its own tiles only, and could take the other's last round for its own.)
  static constexpr int kRawKeys = INT8 ? (D == 128 ? 2 : 3) : 0, kRawValues = INT8 ? (D == 128 ? 1 : 3) : 0, kRaw = kRawKeys + kRawValues;
  static constexpr int kThreads = INT8 ? 640 : 384;     // five warpgroups, or three
  // Registers per thread: the warpgroups that compute weights take what the others leave of the launch's.
  static constexpr int kMany = INT8 ? 160 : 208, kFew = INT8 ? 48 : 88;
  static_assert(256 * kMany + (kThreads - 256) * kFew <= kThreads * (INT8 ? 96 : 168), "the register split is the launch's own");
  static constexpr int kScaleBytes = INT8 ? kInfo * (2 * kTile + 4) * 4 : 0;
  static constexpr int kSmem = 2 * kBytes + kStages * kBytes + kRaw * kRawBytes + kScaleBytes + 1024;
  static constexpr int kReaders = INT8 ? 18 : 11;       // warps that read a unit: weights, products, copies, and cleaning or converters
  static_assert((2 + kStages) * kBytes >= kMostBatch * 12, "the plan fits the tiles");
};

struct Barriers {
  uint64_t q_full, o_full[2], s_full[2], p_full[2], drain, other_full, other_empty;
  uint64_t full[9], empty[2][9], raw_full[6], raw_empty[6], info[kInfo], dirty[kClean], clean[kClean], unit_full[kRing], unit_empty[kRing];
  uint32_t have[kInfo][4];  // together, bit g: tokens 16 g .. 16 g + 15 of the tile have a page
  Unit unit[kRing];
  int bad[kRing];           // values that are not finite were taken out of a tile of this unit
  float2 other[kTile];      // (m, l) of the second tile's rows, where both tiles are the same queries
  uint64_t max_wait_ns;
  uint32_t tmem;
  int quit;
  int n_long;
  int4 of[2];               // the parts that the walk handed out
};

static_assert(sizeof(Barriers) + std::max({Tiles<64, false>::kSmem, Tiles<128, false>::kSmem, Tiles<64, true>::kSmem, Tiles<128, true>::kSmem}) <= 227 * 1024, "a CTA's shared memory");

// Tiles of row block i of a chunk of n tokens behind `base` others (a block that sees nothing has one all the same).
__device__ __forceinline__ int own_seen(const ChunkParams& p, int64_t i, int n, int base, int reach) {
  const int64_t end = min((int64_t)n, ((i + 1) * kBlock + p.group - 1) / p.group);
  return (int)max((int64_t)0, min((int64_t)base + end, (int64_t)reach));
}
__device__ __forceinline__ int prefix_tiles(const ChunkParams& p) { return (p.prefix_len + kTile - 1) / kTile; }
__device__ __forceinline__ int tiles_of(const ChunkParams& p, int64_t i, int n, int base, int reach) {
  return max(1, prefix_tiles(p) + (own_seen(p, i, n, base, reach) + kTile - 1) / kTile);
}

struct Sequence {
  int q0, n, base, reach;
  int blocks;
};
__device__ __forceinline__ Sequence sequence_of(const ChunkParams& p, int b) {
  Sequence s;
  const int from = max(0, p.offsets[b]), end = min(p.rows, p.offsets[b + 1]);
  s.q0 = from;
  s.n = max(0, end - from);
  // Lengths and offsets may be anything: base is a difference of two int32.
  const int64_t base = (int64_t)p.lens[b] - s.n;
  s.base = (int)max((int64_t)INT32_MIN / 2, min(base, (int64_t)INT32_MAX / 2));
  s.reach = (int)max((int64_t)0, min((int64_t)p.lens[b], min((int64_t)p.table_cols << p.page_shift, (int64_t)INT32_MAX / 2)));
  s.blocks = (int)(((int64_t)s.n * p.group + kBlock - 1) / kBlock);
  return s;
}

// Does the tile hold tokens that a row of the unit does not see (`first`: the limit of its first row)?
__device__ __forceinline__ int first_limit(const ChunkParams& p, const Unit& u) { return min(max(0, u.base + u.row0 / p.group + 1), u.seen); }
__device__ __forceinline__ bool partly_seen(const ChunkParams& p, int tile, int n_prefix, int first) {
  return tile < n_prefix ? tile == n_prefix - 1 && p.prefix_len % kTile != 0 : (tile - n_prefix + 1) * kTile > first;
}

__device__ __forceinline__ bool not_finite(uint32_t two) {
  return ((two & 0x7f80u) == 0x7f80u) || ((two & 0x7f800000u) == 0x7f800000u);
}

template <int D, bool INT8, bool CAP>
__global__ void __launch_bounds__(Tiles<D, INT8>::kThreads, 1) chunk_kernel(const ChunkParams p, const __grid_constant__ CUtensorMap pages_map) {
  using T = Tiles<D, INT8>;
  extern __shared__ char raw_smem[];
  __shared__ Barriers s;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  char* q_tiles = smem;
  char* raws = q_tiles + (2 + T::kStages) * T::kBytes;
  float* scale_ring = reinterpret_cast<float*>(raws + T::kRaw * T::kRawBytes);  // [kInfo][2][kTile]: keys', values' x kScaleDown
  [[maybe_unused]] int4* tops = reinterpret_cast<int4*>(scale_ring + kInfo * 2 * kTile);  // [kInfo]: 2^top is above every finite value scale x kScaleDown, per warp of converters
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int n_prefix = prefix_tiles(p), bs = 1 << p.page_shift;
  auto stalls = [&](int which) { return p.stall == which && (p.stall_cta < 0 || p.stall_cta == (int)blockIdx.x); };
  if (tid == 0) {
    mbar_init(&s.q_full, 8);
    mbar_init(&s.drain, 1);
    mbar_init(&s.other_full, 4);
    mbar_init(&s.other_empty, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.o_full[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
    }
    for (int i = 0; i <= T::kStages; ++i) {
      mbar_init(&s.full[i], INT8 ? 4 : 1);
      mbar_init(&s.empty[0][i], 1);
      mbar_init(&s.empty[1][i], 1);
    }
    for (int i = 0; i < T::kRaw; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_empty[i], 4);
    }
    for (int i = 0; i < kInfo; ++i) mbar_init(&s.info[i], INT8 ? 8 : 1);
    for (int i = 0; i < kClean; ++i) {
      mbar_init(&s.dirty[i], 1);
      mbar_init(&s.clean[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&s.unit_full[i], 1);
      mbar_init(&s.unit_empty[i], T::kReaders);
    }
    s.max_wait_ns = p.max_wait_ns;
    s.quit = 0;
    s.n_long = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s.tmem;  // columns: S or weights of the two row tiles at 0 and 128, O at 256 and 256 + D
  pdl_wait();
  pdl_release();

  // Every sequence's length on the line, per KV head, into shared memory that nothing else uses yet: short chunks
  // by a thread, long ones by all.
  int64_t* lengths = reinterpret_cast<int64_t*>(smem);
  int two_tiles = 0;  // has some unit two tiles of rows
  int* longs = reinterpret_cast<int*>(lengths + kMostBatch);
  for (int b = tid; b < p.batch; b += T::kThreads) {
    const Sequence q = sequence_of(p, b);
    two_tiles |= (int64_t)q.n * p.group > kTile;
    int64_t sum = 0;
    if (q.blocks <= 8) {
      for (int i = 0; i < q.blocks; ++i) sum += tiles_of(p, i, q.n, q.base, q.reach) + kPad;
    } else {
      longs[atomicAdd(&s.n_long, 1)] = b;
    }
    lengths[b] = sum;
  }
  two_tiles = __syncthreads_or(two_tiles);
  // The second tile of queries is one stage more where no unit has one.
  const int n_stages = T::kStages + (two_tiles ? 0 : 1);
  char* stages = q_tiles + (two_tiles ? 2 : 1) * T::kBytes;
  for (int k = 0; k < s.n_long; ++k) {
    const int b = longs[k];
    const Sequence q = sequence_of(p, b);
    int64_t sum = 0;
    for (int i = tid; i < q.blocks; i += T::kThreads) sum += tiles_of(p, i, q.n, q.base, q.reach) + kPad;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&lengths[b]), (unsigned long long)sum);
  }
  fence_async();
  __syncthreads();

  // A stage is free to be filled: what was in it has been multiplied. Keys and values take an odd number of stages by turns;
  // each kind's products have barriers of their own, so that whoever fills a stage has waited for every phase of the barrier
  // that it waits on (keys' and values' codes are turned into operands by different warps).
  auto wait_empty = [&](const Cursor& c) {
    if (c.round == 0) return true;
    const int before = c.round - 1;
    const bool both = n_stages % 2 != 0;
    return wait_for(s, &s.empty[(both ? c.slot + before : c.slot) & 1][c.slot], (both ? before >> 1 : before) & 1);
  };

  // The next unit of the line, for a whole warp: a copy of it, or b < 0 at the end (or where a wait ran out).
  int unit_count = 0;
  auto next_unit = [&](bool& ok) {
    const int slot = unit_count % kRing;
    ok = ok && wait_for(s, &s.unit_full[slot], (unit_count / kRing) & 1);
    Unit u;
    u.b = -1;
    if (ok) u = s.unit[slot];
    return u;
  };
  auto unit_done = [&] {
    warp_arrive(&s.unit_empty[unit_count % kRing], lane);
    ++unit_count;
  };

  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kMany));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kFew));
  if (warp < 8) {
    // ---- weights: a warp has 32 rows, a thread four of them (Frag) -----------------------------------
    const int u = warp / 4, g = lane / 4, c2 = 2 * (lane % 4);
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;  // lane 32 (warp % 4) of tensor memory
    const uint32_t ts = tmem + lanes + u * kTile, to = tmem + lanes + 2 * kTile + u * D;
    const float scale = p.scale;
    int jobs = 0, tiles = 0, singles = 0;  // of all units so far: jobs of this row tile, tiles, units of one row tile
    bool ok = true;
    for (;; unit_done()) {
      const Unit un = next_unit(ok);
      if (un.b < 0) break;
      const bool two = un.n_rows > kTile;
      const int base = (two ? u * kTile : 0) + (warp % 4) * 32 + g;  // this thread's rows: base + 8 i
      const bool any_live = base - g < un.n_rows;                    // does this warp hold a row at all
      {
        const int r = tid % kTile, row = two ? u * kTile + r : r;
        const uint4* src = nullptr;
        if (row < un.n_rows) {
          const int x = un.row0 + row, t = x / p.group;
          src = reinterpret_cast<const uint4*>(p.q + (int64_t)(un.q0 + t) * p.q_st + (int64_t)(un.j * p.group + x - t * p.group) * p.q_sh);
        }
        if (two || u == 0) {
          char* tile = q_tiles + (two ? u * T::kBytes : 0);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            uint4 w = src != nullptr ? src[i] : make_uint4(0, 0, 0, 0);
            w.x ^= p.flip, w.y ^= p.flip, w.z ^= p.flip, w.w ^= p.flip;
            *reinterpret_cast<uint4*>(tile + (i / 8) * (kTile * 128) + r * 128 + (((i % 8) ^ (r & 7)) << 4)) = w;
          }
        }
        fence_async();
        if (!stalls(1) || warp != 0) warp_arrive(&s.q_full, lane);
      }
      int limit[4];  // own tokens that a row sees
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = base + 8 * i;
        limit[i] = row < un.n_rows ? min(max(0, un.base + (un.row0 + row) / p.group + 1), un.seen) : INT32_MAX;
      }
      const int lowest = __shfl_sync(0xffffffffu, limit[0], 0);  // of the warp's rows
      float from[4], l[4];  // per row: the reference that weights are taken from (log2 domain), their sum
#pragma unroll
      for (int i = 0; i < 4; ++i) from[i] = -INFINITY, l[i] = 0.0f;
      bool unset = true;  // has some row no reference yet
      [[maybe_unused]] bool wide_unit = false;  // had a tile scores above their cap's size
      const int n_jobs = two ? 2 * un.n_tiles : un.n_tiles;  // job i: rows i % 2, tile two ? i / 2 : i
      int n_done = 0;
      for (int i = u; i < n_jobs; i += 2, ++n_done) {
        const int t = two ? i >> 1 : i, slot = (tiles + t) % kInfo, tile = un.t0 + t;
        ok = wait_for(s, &s.info[slot], ((tiles + t) / kInfo) & 1);
        const uint32_t have = (s.have[slot][0] | s.have[slot][1]) | (s.have[slot][2] | s.have[slot][3]);
        const int start = tile < n_prefix ? 0 : (tile - n_prefix) * kTile;
        const bool masked = have != 0xffu || (tile < n_prefix ? p.prefix_len - tile * kTile : lowest - start) < kTile;
        float most_weight = kMostWeight;
        if constexpr (INT8) {
          const int4 top = tops[slot];
          most_weight = __int_as_float((127 + kMostF16 - max(max(top.x, top.y), max(top.z, top.w))) << 23);
        }
        // Pair 4 k: columns 8 k + c2, + 1.
        [[maybe_unused]] const uint64_t* ks = reinterpret_cast<const uint64_t*>(scale_ring + slot * 2 * kTile + c2);
        [[maybe_unused]] const uint64_t* vs = ks + kTile / 2;
        ok = ok && wait_for(s, &s.s_full[u], (jobs + n_done) & 1);
        if (!ok) break;
        tc_after();
        if (any_live) {
          // WIDE: a score may be above its cap's size; false where one is and WIDE is not (nothing is written then).
          auto weigh = [&](auto mask, [[maybe_unused]] auto any_size) {
            constexpr bool MASK = decltype(mask)::value;
            [[maybe_unused]] constexpr bool WIDE = decltype(any_size)::value;
            [[maybe_unused]] float most = 0.0f;  // of the squares of scores divided by their cap
            constexpr int N = kTile / 16;
            [[maybe_unused]] int upto[4];  // columns of the tile that a row sees
            if constexpr (MASK) {
#pragma unroll
              for (int r = 0; r < 4; ++r) upto[r] = tile < n_prefix ? p.prefix_len - tile * kTile : limit[r] - start;
            }
            // The scores of column pair k of fragment n, row r, up to their factor.
            auto raw_score = [&](const Frag& a, int k, int r, [[maybe_unused]] uint64_t kk) {
              const uint64_t z = pair(__uint_as_float(a.v[r / 2][4 * k + 2 * (r & 1)]), __uint_as_float(a.v[r / 2][4 * k + 2 * (r & 1) + 1]));
              return INT8 ? mul2(z, kk) : z;
            };
            auto wide = [&](uint64_t z) { return pair(capped(first_of(z) * (2.0f * kLog2e * scale), p.cap_log2), capped(second_of(z) * (2.0f * kLog2e * scale), p.cap_log2)); };
            auto seen = [&](uint64_t z, int n, int k, int r) {  // minus infinity where a row does not see a column
              if constexpr (MASK) {
                const int col = 16 * n + 8 * k + c2, to_col = (have >> n) & 1 ? upto[r] : 0;
                z = pair(col < to_col ? first_of(z) : -INFINITY, col + 1 < to_col ? second_of(z) : -INFINITY);
              }
              return z;
            };
            // The tile's scores 16 columns at a time, the next under way.
            auto sweep = [&](auto&& use) {
              Frag f[2];
              ld(f[0], ts);
              ld_wait(f[0]);
#pragma unroll
              for (int n = 0; n < N; ++n) {
                if (n + 1 < N) ld(f[(n + 1) & 1], ts + 16 * (n + 1));
                use(f[n & 1], n);
                if (n + 1 < N) ld_wait(f[(n + 1) & 1]);
              }
            };
            // One pass, from the references as they are; where there are none yet or a score has outgrown them, they
            // are set from the tile's maxima first.
#pragma unroll 1
            for (bool set = unset, again = false;; again = true) {
              if (set) {
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                for (int n = 0; n < N; ++n) {
                  Frag f;
                  ld(f, ts + 16 * n);
                  ld_wait(f);
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    [[maybe_unused]] uint64_t kk = 0, room = 0;
                    if constexpr (INT8) {
                      kk = ks[4 * (2 * n + k)];
                      const uint64_t v = vs[4 * (2 * n + k)];
                      room = pair(scaled_room(first_of(v)), scaled_room(second_of(v)));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                      uint64_t z = raw_score(f, k, r, kk);
                      if constexpr (CAP) z = wide(z);
                      if constexpr (INT8) z = CAP ? add2(z, room) : fma2(z, pair(scale, scale), room);
                      z = seen(z, n, k, r);
                      top[r] = fmaxf(fmaxf(top[r], first_of(z)), second_of(z));
                    }
                  }
                }
                float by[4];
                bool none = false;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                  top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                  const float want = CAP || INT8 ? top[r] : top[r] * scale, to_ref = fmaxf(from[r], want);
                  by[r] = to_ref == -INFINITY ? 1.0f : ex2(from[r] - to_ref);
                  l[r] = INT8 && to_ref > from[r] ? times_ex2(l[r], from[r] - to_ref) : l[r] * by[r];
                  from[r] = to_ref;
                  none = none || to_ref == -INFINITY;
                }
                unset = __any_sync(0xffffffffu, none);
                if (n_done > 0) {  // the products of this row tile's last job are done: its scores came after them
                  Frag f;
#pragma unroll 1
                  for (int n = 0; n < D / 16; ++n) {
                    ld(f, to + 16 * n);
                    ld_wait(f);
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                      uint32_t& w = f.v[x / 8][x % 8];
                      w = __float_as_uint(__uint_as_float(w) * by[2 * (x / 8) + (x % 4) / 2]);
                    }
                    st(to + 16 * n, f);
                  }
                }
              }
              uint64_t ref[4], sum[4] = {0, 0, 0, 0};
              const uint64_t scale2 = pair(scale, scale);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float x = from[r] == -INFINITY ? 0.0f : -from[r];
                ref[r] = pair(x, x);
              }
              uint32_t w[N][2][4];
              sweep([&](const Frag& f, int n) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  [[maybe_unused]] uint64_t kk = 0, vv = 0;
                  if constexpr (INT8) kk = ks[4 * (2 * n + k)], vv = vs[4 * (2 * n + k)];
                  // (Capped scores step by step for four rows: their longer chains of results do not wait for one another.)
                  constexpr int R = CAP ? 4 : 1;
#pragma unroll
                  for (int r0 = 0; r0 < 4; r0 += R) {
                    uint64_t z[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) z[r] = raw_score(f, k, r0 + r, kk);
                    if constexpr (CAP && WIDE) {
#pragma unroll
                      for (int r = 0; r < R; ++r) z[r] = add2(wide(z[r]), ref[r0 + r]);
                    } else if constexpr (CAP) {
#pragma unroll
                      for (int r = 0; r < R; ++r) z[r] = mul2(z[r], scale2);
                      capped2(z, p.cap_log2, ref, most);
                    } else {
                      z[0] = fma2(z[0], scale2, ref[r0]);
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                      z[r] = seen(z[r], n, k, r0 + r);
                      z[r] = pair(ex2(first_of(z[r])), ex2(second_of(z[r])));
                      sum[r0 + r] = add2(sum[r0 + r], z[r]);
                      if constexpr (INT8) {
                        const uint64_t x = mul2(z[r], vv);
                        // A scale of a token that the row does not see may be anything.
                        z[r] = MASK ? pair(first_of(z[r]) == 0.0f ? 0.0f : first_of(x), second_of(z[r]) == 0.0f ? 0.0f : second_of(x)) : x;
                      }
                      w[n][(r0 + r) / 2][2 * k + ((r0 + r) & 1)] = INT8 ? pack_f16(first_of(z[r]), second_of(z[r])) : pack_bf16(first_of(z[r]), second_of(z[r]));
                    }
                  }
                }
              });
              if constexpr (CAP && !WIDE) {
                if (__any_sync(0xffffffffu, most > 1.0f)) return false;
              }
              // No weight is above the sum that it is part of.
              bool over = false;
#pragma unroll
              for (int r = 0; r < 4; ++r) over = over || fmaxf(first_of(sum[r]), second_of(sum[r])) > most_weight;
              set = !again && __any_sync(0xffffffffu, over);
              if (set) continue;
#pragma unroll
              for (int n = 0; n < N; ++n) st_packed(ts + 8 * n, w[n]);  // over the scores
#pragma unroll
              for (int r = 0; r < 4; ++r) l[r] += first_of(sum[r]) + second_of(sum[r]);
              return true;
            }
          };
          const std::true_type yes;
          const std::false_type no;
          if constexpr (!CAP) {
            if (masked) weigh(yes, no);
            else weigh(no, no);
          } else if (wide_unit || !(masked ? weigh(yes, no) : weigh(no, no))) {
            wide_unit = true;  // large scores come together
            if (masked) weigh(yes, yes);
            else weigh(no, yes);
          }
          st_wait();
        }
        tc_before();
        if (!stalls(2) || warp != 0) warp_arrive(&s.p_full[u], lane);
      }
      jobs += n_done;
      // ---- the rows' results ------------------------------------------------------------------------
      const int at_unit = unit_count;
      ok = ok && wait_for(s, &s.o_full[u], at_unit & 1);
      if (!two && u == 0) ok = ok && wait_for(s, &s.o_full[1], at_unit & 1);
      tc_after();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      bool mine = two || u == 0, any_other = false;
      float f0[4] = {1.f, 1.f, 1.f, 1.f}, f1[4] = {0.f, 0.f, 0.f, 0.f};
      if (!two) {
        // Both row tiles hold the same rows: the first reads the second's sums here and its O, which lies in the
        // same lanes of tensor memory, below.
        if (u == 1) {
          if (c2 == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s.other[base + 8 * i] = make_float2(from[i], l[i]);
          }
          warp_arrive(&s.other_full, lane);
        } else {
          ok = ok && wait_for(s, &s.other_full, singles & 1);
          any_other = n_jobs > 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 other = any_other ? s.other[base + 8 * i] : make_float2(-INFINITY, 0.0f);
            const float both = fmaxf(from[i], other.x), ref = both == -INFINITY ? 0.0f : both;
            f0[i] = ex2(from[i] - ref), f1[i] = ex2(other.x - ref);
            l[i] = INT8 ? times_ex2(l[i], from[i] - ref) + times_ex2(other.y, other.x - ref) : l[i] * f0[i] + other.y * f1[i];
            from[i] = both;
          }
        }
      }
      if (mine && any_live) {
        const bool part = un.slot >= 0;
        const bool bad = !INT8 && *static_cast<volatile int*>(&s.bad[unit_count % kRing]) != 0;
        ok = ok && *static_cast<volatile int*>(&s.quit) == 0;
        float by[4];
        int64_t to_row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = base + 8 * i, x = un.row0 + row, t = x / p.group;
          to_row[i] = part ? (int64_t)un.slot * kBlock + row : (int64_t)(un.q0 + t) * (p.h * p.group) + un.j * p.group + (x - t * p.group);
          if (INT8) from[i] += kScaleShift, l[i] *= kScaleDown;  // as the values' scales are
          by[i] = part ? 1.0f : l[i] == 0.0f ? 0.0f : 1.0f / l[i];
          if (!ok) by[i] = l[i] = __uint_as_float(0x7fc00000u);  // where a wait ran out the row is poisoned (its status word tells why)
          f0[i] *= by[i], f1[i] *= by[i];
          if (row < un.n_rows && c2 == 0) {
            if (part) p.part_ml[to_row[i]] = make_float2(from[i], l[i]);
            else p.lse[to_row[i]] = l[i] == 0.0f ? -INFINITY : (from[i] + log2f(l[i])) * kLn2;
          }
        }
#pragma unroll 1
        for (int n = 0; n < D / 16; ++n) {
          Frag f, f2;
          ld(f, to + 16 * n);
          ld_wait(f);
          if (any_other) {
            ld(f2, to + D + 16 * n);
            ld_wait(f2);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) {  // x = 4 k + i: column group k, row i
            const int i = x % 4, e = 4 * (x / 4) + 2 * (i & 1), ch = 16 * n + 8 * (x / 4) + c2;
            float2 o = make_float2(__uint_as_float(f.v[i / 2][e]) * f0[i], __uint_as_float(f.v[i / 2][e + 1]) * f0[i]);
            if (any_other) o.x = fmaf(__uint_as_float(f2.v[i / 2][e]), f1[i], o.x), o.y = fmaf(__uint_as_float(f2.v[i / 2][e + 1]), f1[i], o.y);
            const bool live = base + 8 * i < un.n_rows;
            if (bad && live) {
              // Values that were taken out of the operand: an infinity or a NaN that the row sees is its output's.
#pragma unroll 1
              for (int tile = un.t0; tile < un.t0 + un.n_tiles; ++tile) {
                if (!partly_seen(p, tile, n_prefix, first_limit(p, un))) continue;
                const bool pre = tile < n_prefix;
                const int tok0 = (pre ? tile : tile - n_prefix) * kTile, end = min(kTile, (pre ? p.prefix_len : limit[i]) - tok0);
#pragma unroll 1
                for (int c = 0; c < end; ++c) {
                  const int tok = tok0 + c, blk = tok >> p.page_shift;
                  const int id = pre ? (blk < p.prefix_cols ? p.prefix_table[blk] : -1) : (blk < p.table_cols ? p.table[un.b * p.table_ld + blk] : -1);
                  if (id < 0 || id >= p.n_pages) continue;
                  const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.pages) + ((((int64_t)id * p.h + un.j) * 2 + 1) * bs + (tok & (bs - 1))) * D + ch;
                  const float a = to_f32(v[0]), b = to_f32(v[1]);
                  if (!isfinite(a)) o.x += a;
                  if (!isfinite(b)) o.y += b;
                }
              }
            }
            if (live) {
              if (part) *reinterpret_cast<float2*>(p.part_o + to_row[i] * D + ch) = o;
              else *reinterpret_cast<uint32_t*>(p.out + to_row[i] * D + ch) = pack_bf16(o.x, o.y);
            }
          }
        }
        tc_before();
      }
      if (!two) {  // the second tile's O and sums are read before its next unit overwrites them
        if (u == 0) warp_arrive(&s.other_empty, lane);
        else ok = ok && wait_for(s, &s.other_empty, singles & 1);
        ++singles;
      }
      tiles += un.n_tiles;
      if (!ok) break;
    }
    tc_before();
  } else if (warp == 8) {
    // ---- matrix products: issued by one lane, in order -----------------------------------------------
    constexpr uint32_t kQk = instruction<false>(kTile, false), kPv = instruction<INT8>(D, true);
    const uint32_t q_u = smem_u32(q_tiles), st_u = smem_u32(stages), mine = elect(), tm = __reduce_max_sync(0xffffffffu, tmem);
    int jobs[2] = {0, 0}, cleaned = 0;
    Cursor keys = {0, 0}, values = {1, 0};  // stages of the next tile's
    bool ok = true;
    for (;; unit_done()) {
      const Unit un = next_unit(ok);
      if (un.b < 0) break;
      // What a vote or a reduction gives is known to be the whole warp's: the loop and the operands' addresses stay in uniform
      // registers, and a product issues in a few cycles.
      const bool two = __any_sync(0xffffffffu, un.n_rows > kTile);
      const int n_tiles = __reduce_max_sync(0xffffffffu, un.n_tiles), t0 = __reduce_max_sync(0xffffffffu, un.t0);
      const int n_jobs = two ? 2 * n_tiles : n_tiles, first = __reduce_max_sync(0xffffffffu, first_limit(p, un));
      // Keys of job i's tile, or its values, are in place (asked once per tile).
      auto wait_keys = [&](int i) { return i >= n_jobs || (two && (i & 1) != 0) || wait_for(s, &s.full[keys.slot], keys.phase()); };
      auto wait_values = [&](int i) {
        const int t = two ? i >> 1 : i;
        if (two && (i & 1) != 0) return true;
        if (!wait_for(s, &s.full[values.slot], values.phase())) return false;
        if (!INT8 && partly_seen(p, t0 + t, n_prefix, first)) {
          if (!wait_for(s, &s.clean[cleaned % kClean], (cleaned / kClean) & 1)) return false;
          ++cleaned;
        }
        return true;
      };
      auto qk = [&](int i) {
        const int u = i & 1, slot = keys.slot;
        const uint64_t a = desc_of(q_u + (two ? u * T::kBytes : 0), 16), b = desc_of(st_u + slot * T::kBytes, 16);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {  // 16 channels further: 32 bytes, in units of 16
          const uint64_t step = ((x / 4) * T::kHalfBytes + (x % 4) * 32) / 16;
          mma_ss(tm + u * kTile, a + step, b + step, kQk, x > 0, mine);
        }
        commit(&s.s_full[u], mine);
        if (!two || u == 1) {
          commit(&s.empty[0][slot], mine);
          keys.step(2, n_stages);
        }
      };
      auto pv = [&](int i) {
        const int u = i & 1, slot = values.slot;
        const uint64_t b = desc_of(st_u + slot * T::kBytes, T::kHalfBytes);
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x)  // 16 tokens further: 2 KB of V, 8 columns of weights
          mma_ts(tm + 2 * kTile + u * D, tm + u * kTile + 8 * x, b + x * (2048 / 16), kPv, x > 0 || i > 1, mine);
        if (!two || u == 1) {
          commit(&s.empty[1][slot], mine);
          values.step(2, n_stages);
        }
        if (two && i + 2 >= n_jobs) commit(&s.o_full[u], mine);
      };
      // The scores of job i + 2 follow the output of job i at once (the weights wait for both).
      ok = wait_for(s, &s.q_full, unit_count & 1);
      for (int i = 0; ok && i < 2 && i < n_jobs; ++i) {
        ok = wait_keys(i);
        tc_after();
        if (ok) qk(i);
      }
      for (int i = 0; ok && i < n_jobs; ++i) {
        ok = wait_values(i) && wait_for(s, &s.p_full[i & 1], jobs[i & 1] & 1);
        if (!ok) break;
        tc_after();
        pv(i);
        ++jobs[i & 1];
        // (Behind the product: three stages may hold the keys of job i + 2 only once its values' has left them.)
        ok = wait_keys(i + 2);
        if (ok && i + 2 < n_jobs) qk(i + 2);
      }
      if (!ok) break;
      if (!two) {
        commit(&s.o_full[0], mine);
        commit(&s.o_full[1], mine);
      }
    }
    // Nothing is freed under a product in flight, whoever gave up and when.
    commit(&s.drain, mine);
    mbar_wait(&s.drain, 0);
    __syncwarp();
  } else if (warp == 9) {
    // ---- copies: the pages of one operand tile at a time, keys then values ----------------------------
    // An entry of the info ring is written again kInfo = 8 tiles later. That tile's keys, or the tile's before
    // it, have a stage that a tile's at most (n_stages + 1) / 2 = 5 before has left, and its products follow the
    // weights of all but the two jobs before them: the entry's last reader is done.
    const int per = kTile >> p.page_shift;  // pages per tile
    int tiles = 0, filled = 0;
    Cursor at = {0, 0}, raw[2] = {{0, 0}, {T::kRawKeys, 0}};
    [[maybe_unused]] int dirty = 0;
    bool ok = true;
    for (;; unit_done()) {
      const Unit un = next_unit(ok);
      if (un.b < 0) break;
      [[maybe_unused]] const int first = first_limit(p, un);
      // Lane i has page i of the tile, looked up a tile ahead (its id, checked where it is used).
      int page = -1, next = -1;
      auto look_up = [&](int t) {
        const int tile = un.t0 + t, own = tile - n_prefix;
        next = -1;
        if (t >= un.n_tiles || lane >= per) return;
        const int tok = (own < 0 ? tile : own) * kTile + lane * bs, blk = tok >> p.page_shift;
        if (own < 0) {
          if (tok < p.prefix_len && blk < p.prefix_cols) next = p.prefix_table[blk];
        } else if (tok < un.seen && blk < p.table_cols) {
          next = p.table[un.b * p.table_ld + blk];
        }
      };
      look_up(0);
      for (int n = 0; ok && n < 2 * un.n_tiles; ++n) {
        const int t = n >> 1, kv = n & 1, info = (tiles + t) % kInfo;
        if (kv == 0) {
          page = next < p.n_pages ? next : -1;
          look_up(t + 1);
        }
        if constexpr (!INT8) {
          const int slot = at.slot;
          ok = wait_empty(at);
          if (!ok) break;
          const uint32_t granules = lane < per && page >= 0 ? ((1u << (bs / 16)) - 1) << (lane * (bs / 16)) : 0u;
          const uint32_t have = __reduce_or_sync(0xffffffffu, granules);
          if (lane == 0) mbar_arrive_expect_tx(&s.full[slot], T::kBytes);
          __syncwarp();
          if (lane < per) {
            const int rows = p.n_pages * 2 * p.h * bs;  // one past the last: zeros
            const int y = page >= 0 ? ((page * p.h + un.j) * 2 + kv) * bs : rows;
            const uint32_t dst = smem_u32(stages) + slot * T::kBytes + lane * bs * 128;
#pragma unroll
            for (int h2 = 0; h2 < T::kHalves; ++h2) tma_2d(dst + h2 * T::kHalfBytes, &pages_map, 64 * h2, y, &s.full[slot]);
          }
          ++filled;
          at.step(1, n_stages);
          // To be cleaned: said behind the copies, so that the cleaner never waits for a filling before the last one.
          if (kv == 1 && partly_seen(p, un.t0 + t, n_prefix, first)) warp_arrive(&s.dirty[dirty++ % kClean], lane);
          if (lane == 0 && kv == 0) {
            s.have[info][0] = have;
            s.have[info][1] = s.have[info][2] = s.have[info][3] = 0;
            mbar_arrive(&s.info[info]);
          }
        } else {
          const int slot = raw[kv].slot;
          ok = wait_for(s, &s.raw_empty[slot], raw[kv].phase() ^ 1);  // (of the first round: at once)
          if (!ok) break;
          const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, page >= 0));
          if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[slot], n_copies * bs * D);
          __syncwarp();
          if (page >= 0)
            tma_load_1d(raws + slot * T::kRawBytes + lane * bs * D,
                        static_cast<const char*>(p.pages) + (((int64_t)page * p.h + un.j) * 2 + kv) * ((int64_t)bs * D), bs * D, &s.raw_full[slot]);
          ++filled;
          if (++raw[kv].slot == (kv == 0 ? T::kRawKeys : T::kRaw)) raw[kv].slot = kv == 0 ? 0 : T::kRawKeys, ++raw[kv].round;
        }
      }
      if (!ok) break;
      tiles += un.n_tiles;
    }
    // No copy may land after the CTA has gone, also where the others gave up behind this warp's last copy.
    if constexpr (INT8) {
      // The last round of each ring: keys are every other copy, the first one theirs.
      const int n_of[2] = {(filled + 1) / 2, filled / 2};
      for (int kv = 0; kv < 2; ++kv) {
        const int size = kv == 0 ? T::kRawKeys : T::kRawValues;
        for (int n = max(0, n_of[kv] - size); n < n_of[kv]; ++n) mbar_wait(&s.raw_full[kv * T::kRawKeys + n % size], (n / size) & 1);
      }
    } else {
      for (int n = max(0, filled - n_stages); n < filled; ++n) mbar_wait(&s.full[n % n_stages], (n / n_stages) & 1);
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---- the walk along the line -----------------------------------------------------------------------
    int64_t all = 0;
    for (int b = lane; b < p.batch; b += 32) all += lengths[b] * p.h;
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const int64_t n_ctas = max((int64_t)1, min((int64_t)gridDim.x, all / kMinShare));
    const int c = blockIdx.x;
    int64_t at = c < n_ctas ? all / n_ctas * c + all % n_ctas * c / n_ctas : all;
    int64_t left = c < n_ctas ? all / n_ctas * (c + 1) + all % n_ctas * (c + 1) / n_ctas - at : 0;
    int4 of[2] = {make_int4(0, 0, 0, 0), make_int4(0, 0, 0, 0)};
    // The sequence, head and block that `at` lies in.
    int b = 0, j = 0;
    int64_t i = 0;
    int pos = 0;
    Sequence q = {};
    bool ok = true;
    if (left > 0) {
      for (; b < p.batch; b += 32) {  // 32 sequences at a time
        int64_t mine = b + lane < p.batch ? lengths[b + lane] * p.h : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, mine, o);
          if (lane >= o) mine += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, mine > at);
        if (behind != 0) {
          const int first = __ffs(behind) - 1;
          if (first > 0) at -= __shfl_sync(0xffffffffu, mine, first - 1);
          b += first;
          break;
        }
        at -= __shfl_sync(0xffffffffu, mine, 31);
      }
      q = sequence_of(p, b);
      j = (int)(at / lengths[b]);
      at -= j * lengths[b];
      for (;; i += 32) {
        int64_t mine = i + lane < q.blocks ? tiles_of(p, i + lane, q.n, q.base, q.reach) + kPad : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, mine, o);
          if (lane >= o) mine += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, mine > at);
        if (behind != 0) {
          const int first = __ffs(behind) - 1;
          if (first > 0) at -= __shfl_sync(0xffffffffu, mine, first - 1);
          i += first;
          break;
        }
        at -= __shfl_sync(0xffffffffu, mine, 31);
      }
      pos = (int)at;
    }
    fence_async();  // the plan is read: queries and copies may have its place
    int count = 0;
    auto hand_out = [&](const Unit& un) {
      const int slot = count % kRing;
      if (count >= kRing) ok = ok && wait_for(s, &s.unit_empty[slot], (count / kRing - 1) & 1);
      if (!ok) return;
      if (lane == 0) {
        s.unit[slot] = un;
        s.bad[slot] = 0;
      }
      warp_arrive(&s.unit_full[slot], lane);
      ++count;
    };
    while (ok && left > 0) {
      if (i >= q.blocks) {  // (also a sequence without new tokens)
        i = 0;
        if (q.blocks == 0 || ++j == p.h) {
          j = 0;
          if (++b == p.batch) break;
          q = sequence_of(p, b);
        }
        continue;
      }
      const int n_tiles = tiles_of(p, i, q.n, q.base, q.reach), length = n_tiles + kPad;
      const int take = (int)min(left, (int64_t)(length - pos)), end = min(pos + take, n_tiles);
      if (pos < end) {
        Unit un;
        un.b = b, un.j = j, un.row0 = (int)(i * kBlock), un.n_rows = (int)min((int64_t)kBlock, (int64_t)q.n * p.group - i * kBlock);
        un.t0 = pos, un.n_tiles = end - pos, un.base = q.base, un.seen = own_seen(p, i, q.n, q.base, q.reach), un.q0 = q.q0;
        un.slot = -1;
        if (pos > 0 || end < n_tiles) {
          const int k = pos > 0 ? 0 : 1;
          of[k] = make_int4(end == n_tiles ? 3 : 1, b, j, un.row0);
          un.slot = 2 * c + k;
        }
        hand_out(un);
      }
      left -= take;
      pos += take;
      if (pos == length) pos = 0, ++i;
    }
    if (ok) {
      Unit un = {};
      un.b = -1;
      hand_out(un);
    }
    if (lane < 2) s.of[lane] = of[lane];
    __syncwarp();
  } else if (warp == 11) {
    if constexpr (!INT8) {
      // ---- values that are not finite are taken out of tiles that some row does not see whole --------------
      int cleaned = 0;
      Cursor values = {1, 0};
      bool ok = true;
      for (;; unit_done()) {
        const Unit un = next_unit(ok);
        if (un.b < 0) break;
        const int first = first_limit(p, un);
        for (int t = 0; ok && t < un.n_tiles; ++t, values.step(2, n_stages)) {
          if (!partly_seen(p, un.t0 + t, n_prefix, first)) continue;
          const int slot = values.slot;
          ok = wait_for(s, &s.dirty[cleaned % kClean], (cleaned / kClean) & 1) && wait_for(s, &s.full[slot], values.phase());
          if (!ok) break;
          uint4* v = reinterpret_cast<uint4*>(stages + slot * T::kBytes);
          bool found = false;
#pragma unroll 8
          for (int x = lane; x < T::kBytes / 16; x += 32) {
            const uint4 w = v[x];
            if (not_finite(w.x) || not_finite(w.y) || not_finite(w.z) || not_finite(w.w)) {
              uint32_t y[4] = {w.x, w.y, w.z, w.w};
              for (int k = 0; k < 4; ++k) {
                if ((y[k] & 0x7f80u) == 0x7f80u) y[k] &= 0xffff0000u;
                if ((y[k] & 0x7f800000u) == 0x7f800000u) y[k] &= 0xffffu;
              }
              v[x] = make_uint4(y[0], y[1], y[2], y[3]);
              found = true;
            }
          }
          if (found) *static_cast<volatile int*>(&s.bad[unit_count % kRing]) = 1;
          fence_async();
          warp_arrive(&s.clean[cleaned % kClean], lane);
          ++cleaned;
        }
        if (!ok) break;
      }
    }
  } else {
    if constexpr (INT8) {
      // ---- codes to operands: warps 12-15 the keys' to bf16, 16-19 the values' to f16; thread i carries token i's scale --
      const int i = tid % kTile, kv = (tid - 12 * 32) / kTile;
      // A thread's pieces of 16 codes, one channel range of every kStep-th token. Eight lanes take 128 bytes
      // that lie in 32 different banks, and so do the chunks they write: two tokens of different parity, of
      // which the swizzle puts even chunks into even and odd places.
      constexpr int kPer = D / 16, kStep = kTile / kPer;  // kStep is a multiple of 8
      const int odd = (i >> 2) & 1, half = odd ^ ((i >> 3) & 1);
      const int tok0 = kPer == 8 ? (i >> 4) * 2 + odd : i / kPer, c = kPer == 8 ? half * 4 + (i & 3) : i % kPer;
      const int from = (tok0 * kPer + c) * 16, row = (c / 4) * T::kHalfBytes + tok0 * 128, at = (c % 4) * 2;
      const int to0 = row + ((at ^ (tok0 & 7)) << 4), to1 = row + (((at + 1) ^ (tok0 & 7)) << 4);
      int tiles = 0;
      Cursor to = {kv, 0}, raw = {kv * T::kRawKeys, 0};
      bool ok = true;
      for (;; unit_done()) {
        const Unit un = next_unit(ok);
        if (un.b < 0) break;
        // Scales are loaded a tile ahead, and their page's id (checked where it is used) a tile before that:
        // neither load is waited for where it is issued.
        float scale = 0.0f;
        bool there = false;
        int id = -1;
        auto page_of = [&](int t) {
          const int tile = un.t0 + t, own = tile - n_prefix, pos = (own < 0 ? tile : own) * kTile + i, blk = pos >> p.page_shift;
          id = -1;
          if (t >= un.n_tiles) return;
          if (own < 0) {
            if (pos < p.prefix_len && blk < p.prefix_cols) id = p.prefix_table[blk];
          } else if (pos < un.seen && blk < p.table_cols) {
            id = p.table[un.b * p.table_ld + blk];
          }
        };
        auto scales_of = [&](int t) {
          scale = 0.0f;  // of a token that is not there (its codes are what shared memory held: they choose no form of a capped score)
          there = id >= 0 && id < p.n_pages;
          if (there) {
            const int tile = un.t0 + t, pos = (tile < n_prefix ? tile : tile - n_prefix) * kTile + i;
            scale = p.scales[(((int64_t)id * p.h + un.j) * 2 + kv) * bs + (pos & (bs - 1))];
          }
          page_of(t + 1);
        };
        page_of(0);
        scales_of(0);
        for (int t = 0; t < un.n_tiles; ++t) {
          const int info = (tiles + t) % kInfo;
          // The ring entry's last reader is more than two tiles behind (see the copies): it is free.
          scale_ring[(info * 2 + kv) * kTile + i] = kv == 0 ? scale : scale * kScaleDown;
          if (kv == 1) {
            const int top = __reduce_max_sync(0xffffffffu, scaled_top(scale * kScaleDown));
            if (lane == 0) reinterpret_cast<int*>(tops + info)[warp - 16] = top;
          } else {
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (lane == 0) s.have[info][warp - 12] = ((mask & 0xffffu) != 0 ? 1u : 0u) << (2 * (warp - 12)) | (mask >> 16 != 0 ? 2u : 0u) << (2 * (warp - 12));
          }
          warp_arrive(&s.info[info], lane);
          scales_of(t + 1);
          ok = ok && wait_for(s, &s.raw_full[raw.slot], raw.phase()) && wait_empty(to);
          if (!ok) break;
          const char* src = raws + raw.slot * T::kRawBytes + from;
          char* dst = stages + to.slot * T::kBytes;
          auto convert = [&](auto&& operand) {
#pragma unroll
            for (int x0 = 0; x0 < kPer; x0 += 4) {
              uint4 w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) w[x] = *reinterpret_cast<const uint4*>(src + (x0 + x) * (kStep * kPer * 16));
              if (x0 + 4 >= kPer) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.raw_empty[raw.slot]);
              }
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint2 a = operand(w[x].x), b = operand(w[x].y), d = operand(w[x].z), e = operand(w[x].w);
                *reinterpret_cast<uint4*>(dst + to0 + kStep * (x0 + x) * 128) = make_uint4(a.x, a.y, b.x, b.y);
                *reinterpret_cast<uint4*>(dst + to1 + kStep * (x0 + x) * 128) = make_uint4(d.x, d.y, e.x, e.y);
              }
            }
          };
          if (kv == 0) convert([](uint32_t x) { return codes_to_bf16(x); });
          else convert([](uint32_t x) { return prefix::codes_to_f16(x); });
          fence_async();
          warp_arrive(&s.full[to.slot], lane);
          to.step(2, n_stages);
          if (++raw.slot == (kv == 0 ? T::kRawKeys : T::kRaw)) raw.slot = kv * T::kRawKeys, ++raw.round;
        }
        if (!ok) break;
        tiles += un.n_tiles;
      }
      __syncwarp();
    }
  }
  __syncthreads();
  // Units are handed out ahead: a part that is named here need not have been written where a wait ran out.
  if (tid < 2) {
    int4 of = s.of[tid];
    if (of.x != 0 && *static_cast<volatile int*>(&s.quit) != 0) of.x |= kLost;
    p.part_of[2 * blockIdx.x + tid] = of;
  }
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Units that more than one CTA had a part of: CTA c of the line began one and did not end it, the following ones
// have the others. A warp folds a row.
template <int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const ChunkParams p) {
  pdl_wait();
  pdl_release();
  const int c = blockIdx.x, lane = threadIdx.x % 32;
  const int4 of = p.part_of[2 * c + 1];
  if (of.x == 0) return;
  int last = c + 1, found = of.x | p.part_of[2 * last].x;
  while (last + 1 < (int)gridDim.x && (p.part_of[2 * last].x & 3) == 1) found |= p.part_of[2 * ++last].x;
  const bool lost = (found & kLost) != 0;
  const Sequence q = sequence_of(p, of.y);
  const int n_rows = (int)min((int64_t)kBlock, (int64_t)q.n * p.group - of.w);
  for (int row = blockIdx.y * 8 + threadIdx.x / 32; row < n_rows; row += gridDim.y * 8) {
    float m = -INFINITY;
    for (int k = c; k <= last; ++k) m = fmaxf(m, p.part_ml[(int64_t)(k == c ? 2 * c + 1 : 2 * k) * kBlock + row].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = lost ? __uint_as_float(0x7fc00000u) : 0.0f, o[D / 32] = {};
    for (int k = c; k <= last; ++k) {
      const int64_t at = (int64_t)(k == c ? 2 * c + 1 : 2 * k) * kBlock + row;
      const float2 ml = p.part_ml[at];
      const float f = ex2(ml.x - ref);
      l += times_ex2(ml.y, ml.x - ref);  // (of int8 pages references are as far apart as value scales may be)
#pragma unroll
      for (int x = 0; x < D / 32; x += 2) {
        const float2 v = *reinterpret_cast<const float2*>(p.part_o + at * D + (x / 2) * 64 + 2 * lane);
        o[x] = fmaf(v.x, f, o[x]), o[x + 1] = fmaf(v.y, f, o[x + 1]);
      }
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    const int x = of.w + row, t = x / p.group;
    const int64_t to = (int64_t)(q.q0 + t) * (p.h * p.group) + of.z * p.group + (x - t * p.group);
#pragma unroll
    for (int k = 0; k < D / 32; k += 2) *reinterpret_cast<uint32_t*>(p.out + to * D + (k / 2) * 64 + 2 * lane) = pack_bf16(o[k] * by, o[k + 1] * by);
    if (lane == 0) p.lse[to] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

template <int D, bool INT8, bool CAP>
cudaError_t launch_chunk(const ChunkParams& p, const CUtensorMap& map, int grid, cudaStream_t st) {
  using T = Tiles<D, INT8>;
  auto k = chunk_kernel<D, INT8, CAP>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = prefix::allow_smem(k, T::kSmem, done);
  if (e == cudaSuccess) e = launch_pdl(k, dim3(grid), dim3(T::kThreads), T::kSmem, st, 0, p, map);
  if (e == cudaSuccess) e = launch_pdl(chunk_merge_kernel<D>, dim3(grid, 8), dim3(256), 0, st, 0, p);
  return e;
}

// CTAs of a launch: one per SM, or fewer where the call's bounds leave less on the line.
int grid_of(int rows, int batch, int h, int group, int64_t prefix_len, int64_t own_reach) {
  const int64_t blocks = (int64_t)rows * group / kBlock + std::min(rows, batch), tiles = (prefix_len + kTile - 1) / kTile + (own_reach + kTile - 1) / kTile;
  const double line = (double)blocks * h * (double)(std::max<int64_t>(1, tiles) + kPad) / kMinShare;
  return line >= kNumSMs ? kNumSMs : std::max(1, (int)line);
}

size_t slot_bytes(int d) { return (size_t)kBlock * d * 4 + (size_t)kBlock * 8 + 16; }

uint64_t g_chunk_wait_ns = kMaxTensorWaitNs;
int g_chunk_stall_next = 0, g_chunk_stall_cta = -1;

}  // namespace

int chunk_set_wait(int64_t ns) {
  if (ns < 1 || ns > (int64_t)kMaxTensorWaitNs) return fail(LKV_ERR_ARG, "lkv_debug_set: chunk wait bound %lld ns outside [1, %llu]", (long long)ns, (unsigned long long)kMaxTensorWaitNs);
  g_chunk_wait_ns = (uint64_t)ns;
  return LKV_OK;
}
int chunk_set_stall(int64_t which) {
  if (which < 0 || which > 2) return fail(LKV_ERR_ARG, "lkv_debug_set: no stall %lld of the chunk attention (0, 1 or 2)", (long long)which);
  g_chunk_stall_next = (int)which;
  return LKV_OK;
}
int chunk_set_stall_cta(int64_t cta) {
  if (cta < -1 || cta > INT32_MAX) return fail(LKV_ERR_ARG, "lkv_debug_set: no CTA %lld of the chunk attention (-1: all)", (long long)cta);
  g_chunk_stall_cta = (int)cta;
  return LKV_OK;
}
cudaError_t chunk_device_status(int* status, int clear) { return tu_device_status(status, clear); }
cudaError_t chunk_status_attach(int* mirror) { return tu_status_attach(mirror); }

}  // namespace lkv

using namespace lkv;

extern "C" {

size_t lkv_chunk_attention_workspace(int rows, int batch, int hq, int h, int d, int64_t prefix_len, int64_t own_reach) {
  if (rows <= 0 || batch <= 0 || h <= 0 || hq <= 0 || d <= 0 || prefix_len < 0 || own_reach < 0) return 0;
  return 2 * (size_t)grid_of(rows, batch, h, hq / h, prefix_len, own_reach) * slot_bytes(d);
}

int lkv_chunk_attention(const lkv_chunk_args* a, void* stream) {
  static const char* who = "lkv_chunk_attention";
  if (a == nullptr) return fail(LKV_ERR_PTR, "%s: null arguments", who);
  if (a->dtype != LKV_BF16) return fail(LKV_ERR_ARG, "%s: queries are bfloat16, got dtype %d", who, a->dtype);
  if (int rc = check_cache(who, a->kind, a->dtype, a->h, a->bs, a->d, a->n_pages, a->pages, a->scales)) return rc;
  if (a->rows < 0 || a->rows > (1 << 30) || a->batch < 0 || a->batch > kMostBatch || a->table_cols < 0 || (a->batch > 1 && a->table_ld < a->table_cols))
    return fail(LKV_ERR_ARG, "%s: bad shape (rows %d, batch %d of at most %d, table of %d columns)", who, a->rows, a->batch, kMostBatch, a->table_cols);
  if (a->hq < 1 || a->hq % a->h != 0 || a->hq / a->h > 1024) return fail(LKV_ERR_ARG, "%s: %d query heads for %d KV heads", who, a->hq, a->h);
  const int group = a->hq / a->h;
  if ((int64_t)a->rows * group > (1 << 30)) return fail(LKV_ERR_ARG, "%s: %d rows of %d query heads per KV head in one call", who, a->rows, group);
  if (a->prefix_len < 0 || a->prefix_len > (1 << 30) || a->prefix_len > (int64_t)a->prefix_cols * a->bs)
    return fail(LKV_ERR_ARG, "%s: a prefix of %lld tokens in %d pages of %d", who, (long long)a->prefix_len, a->prefix_cols, a->bs);
  if (!scores_fit(a->scale, a->cap)) return fail(LKV_ERR_ARG, "%s: scale %g with cap %g leaves float32", who, (double)a->scale, (double)a->cap);
  const int64_t page_rows = a->n_pages * 2 * a->h * a->bs;
  if (page_rows > INT32_MAX) return fail(LKV_ERR_ARG, "%s: %lld rows of pages", who, (long long)page_rows);
  if (a->rows == 0 || a->batch == 0) return LKV_OK;
  if (a->q == nullptr || a->lens == nullptr || a->offsets == nullptr || (a->table == nullptr && a->table_cols > 0) || (a->prefix_table == nullptr && a->prefix_len > 0) ||
      a->out == nullptr || a->lse == nullptr)
    return fail(LKV_ERR_PTR, "%s: null pointer", who);
  if (!aligned(a->q, 16) || (a->q_st & 7) != 0 || (a->q_sh & 7) != 0) return fail(LKV_ERR_PTR, "%s: query rows must be 16-byte aligned", who);
  if (!aligned(a->out, 16) || !aligned(a->workspace, 16)) return fail(LKV_ERR_PTR, "%s: output and workspace must be 16-byte aligned", who);
  const int64_t reach = (int64_t)a->table_cols * a->bs;
  const size_t need = lkv_chunk_attention_workspace(a->rows, a->batch, a->hq, a->h, a->d, a->prefix_len, reach);
  if (a->workspace == nullptr || a->workspace_bytes < need) return fail(LKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, need);
  ChunkParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.q_st = a->q_st, p.q_sh = a->q_sh;
  p.pages = a->pages, p.scales = a->scales, p.n_pages = (int)a->n_pages, p.page_shift = shift_of(a->bs);
  p.rows = a->rows, p.batch = a->batch, p.h = a->h, p.group = group;
  p.table = a->table, p.table_ld = a->table_ld, p.table_cols = a->table_cols, p.lens = a->lens, p.offsets = a->offsets;
  p.prefix_table = a->prefix_table, p.prefix_cols = a->prefix_cols, p.prefix_len = (int)a->prefix_len;
  const bool cap = a->cap > 0.0f;
  // (At least a number: a score of -infinity stays one under a softmax scale of zero.)
  const float size = fabsf(a->scale) * kLog2e;
  p.scale = cap ? fabsf(a->scale) / a->cap : size == 0.0f ? FLT_MIN : size;
  p.flip = a->scale < 0.0f ? 0x80008000u : 0u;
  p.cap_log2 = a->cap * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(a->out), p.lse = a->lse;
  const int grid = grid_of(a->rows, a->batch, a->h, group, a->prefix_len, reach);
  p.part_of = static_cast<int4*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_of + 2 * grid);
  p.part_o = reinterpret_cast<float*>(p.part_ml + (size_t)2 * grid * kBlock);
  p.max_wait_ns = g_chunk_wait_ns;
  p.stall = g_chunk_stall_next, p.stall_cta = g_chunk_stall_cta;
  g_chunk_stall_next = 0;
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
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (int8) return cap ? launch_chunk<D, true, true>(p, map, grid, st) : launch_chunk<D, true, false>(p, map, grid, st);
    return cap ? launch_chunk<D, false, true>(p, map, grid, st) : launch_chunk<D, false, false>(p, map, grid, st);
  };
  const cudaError_t e = a->d == 128 ? launch(std::integral_constant<int, 128>()) : launch(std::integral_constant<int, 64>());
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // extern "C"
