// The prefix's part of the shared-prefix attention for batches of many rows, on the 5th-generation
// tensor cores.
//
// A CTA holds up to 256 query rows of one KV head as two tiles of 128 and takes a chunk of the prefix
// through them, 128 tokens at a time. Per tile of rows: S = Q K^T (tcgen05.mma, both operands in shared
// memory, S in tensor memory), each warp turns its 32 rows' 128 scores into weights (running maximum and
// sum in registers, float32), writes them back as 16-bit P over S, and O += P V (P read from tensor
// memory, V from shared memory) accumulates in tensor memory. The two tiles alternate, so that one
// computes weights while the tensor core works for the other. With 128 rows or fewer both tiles are the
// same queries and take the prefix's tiles in turn; their results are merged at the end. Each CTA writes
// one partial (m, l, o) per row, which combine_kernel (prefix.cu) folds into the output.
//
// Warps 0-3 and 4-7 are the two tiles' rows, warp 8 issues the matrix products, warp 9 the copies; with
// int8 pages warps 12-15 turn codes of keys into f16 operands and warps 16-19 those of values. All of it is
// joined by mbarriers, every wait bounded.
//
// Measured at 512 rows of each of 8 KV heads on 32,768 tokens, d 128: int8 105 us, the tensor cores busy 32% of the
// time and the exponentials' unit 38%; bf16 78 us, 43% and 51%. 128 sequences of 8 KV heads with 4 query heads each
// on 131,072 int8 tokens: 332 us, 0.83 PFLOP/s, and 402 to 413 us with up to 2,000 own tokens each, which the stream
// takes behind the tiles (no CTA of it fits beside one of these). What bounds it is the chain of one tile
// of rows, scores -> weights -> products -> next scores: S and P share 128 columns of tensor memory (two tiles
// of S and O of d 128 fill it), so a tile's next scores wait for its present product, and two tiles do not
// fill each other's gaps. Short prefixes add a start of 5 to 8 us (tensor memory, queries, the first pages).
// Registers: the int8 forms store 72 bytes of a thread's to local memory and the two-term ones 172; the bf16
// forms 4.
//
// bf16 pages: P and V are bf16; the pages come by tensor-map TMA straight into the swizzled operand layout (a
// page that is missing as a row past the tensor's end, that is as zeros). For a float32 output P has two terms
// (prefix.cuh, rest_of: 2^-15 of a weight is lost), each multiplied by V. For a bfloat16 output, which
// is rounded itself, it has one (2^-8 at most): the second costs a third of the time (512 rows of each of 8 heads
// on 32,768 tokens, d 128: 85 and 111 us), and without it such an output's mean error is 1.4 times the rounding's.
// int8 pages: codes are exact in f16, and so is a query row after a power of two that brings its largest
// element to [1, 2) (smaller ones lose bits below 2^-25 of it). A key's scale multiplies its column of
// scores in float32 and a value's scale its column of weights, which are then rounded to f16: the one rounding
// of the second product's operands (prefix.cuh, weight_room, says what is left of it).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cuda_fp16.h>
#include <float.h>

#include <type_traits>

#include "prefix.cuh"
#include "tma.cuh"

namespace lkv {
namespace prefix {
namespace {

constexpr int kTile = 128;       // rows of a tile of queries, tokens of a tile of the prefix
constexpr int kInfo = 8;         // tiles whose scales and page bits are kept (see the producer)
// What the sum of a thread's weights may grow to before its references are set again: a bf16 weight has
// float32's range, of which the accumulated values need the rest.
constexpr float kMostBf16 = 1048576.0f;  // 2^20
// int8: a weight times its value's scale has to stay below 2^kMostF16. That is asked of the sum and the tile's
// largest scale: where a token of little weight has that scale, references are looked up for nothing.
constexpr int kMostF16 = 15;
// int8: sums of codes times a query's f16 are below 2^15, and a key's scale may be 2^121: it is kept 2^9 smaller, and
// the row's factor that much larger, so that no product passes float32's end. (A scale below 2^-117 loses bits: fourteen
// are left at the least. The product of the two factors first would cost 3% of the time.)
constexpr float kKeyDown = 1.0f / 512.0f, kKeyUp = 512.0f;

template <int D, bool INT8>
struct Tiles {
  static constexpr int kHalves = D / 64;                 // 64 channels (128 bytes) per swizzled column
  static constexpr int kHalfBytes = kTile * 128;
  static constexpr int kBytes = kHalves * kHalfBytes;    // one operand tile
  static constexpr int kStages = INT8 ? (D == 128 ? 3 : 6) : (D == 128 ? 5 : 8);
  static constexpr int kRawBytes = INT8 ? kTile * D : 0; // one tile of codes
  static constexpr int kRaw = INT8 ? 3 : 0;
  static constexpr int kThreads = INT8 ? 640 : 384;      // five warpgroups, or three
  // Registers per thread: the warpgroups that compute weights take what the others leave of the launch's
  // 96 (or 168) per thread. The split's sum stays within the launch's.
  static constexpr int kMany = INT8 ? 160 : 208, kFew = INT8 ? 48 : 88;
  static_assert(256 * kMany + (kThreads - 256) * kFew <= kThreads * (INT8 ? 96 : 168), "the register split is the launch's own");
  static constexpr int kScaleBytes = INT8 ? kInfo * 2 * kTile * 4 : 0;
  static constexpr int kSmem = 2 * kBytes + kStages * kBytes + kRaw * kRawBytes + kScaleBytes + 1024;
};

struct Barriers {
  uint64_t q_full, o_full[2], s_full[2], p_full[2], tail, drain;
  uint64_t full[9], empty[9], raw_full[3], raw_empty[3], info[kInfo];
  uint32_t have[kInfo][4];   // together, bit g: tokens 16 g .. 16 g + 15 of the tile have a page
  int32_t top[kInfo][4];     // int8: 2^top is above every finite value scale x kScaleDown, per warp of converters
  float back[2][kTile];      // int8: what a row's scores are multiplied with (stage_query)
  uint64_t max_wait_ns;
  uint32_t tmem;
  int quit;
};

// Waits for the phase of `bar` with the given parity, max_wait_ns at most, or until another role gave up.
// Without a suspend-time hint: the waits here are short and many, and a hinted one was seen to resume late.
constexpr uint64_t kMaxWaitNs = 2000000000ull;  // unless a test asks for less
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool try_once(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(done)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return done != 0;
}
__device__ __forceinline__ bool wait_long(Barriers& s, uint64_t* bar, uint32_t parity) {
  const uint64_t from = now_ns();
  while (!try_once(bar, parity)) {
    if (*static_cast<volatile int*>(&s.quit)) return false;
    if (now_ns() - from > s.max_wait_ns) {
      *static_cast<volatile int*>(&s.quit) = 1;
      record_status(LKV_DEV_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}
// For the whole warp, every lane for itself (each needs what the barrier makes visible); the warp leaves it
// together, with one answer.
__device__ __forceinline__ bool wait_for(Barriers& s, uint64_t* bar, uint32_t parity) {
  const bool ok = __all_sync(0xffffffffu, try_once(bar, parity) || wait_long(s, bar, parity)) != 0;
  __syncwarp();
  return ok;
}

// One arrival for the warp, after what all of its lanes did before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// A value scale that kScaleDown has multiplied is below 2^scaled_top, one that is not finite claims nothing;
// weight_room is 7 less.
__device__ __forceinline__ int scaled_top(float scaled) {
  const int bits = (__float_as_int(scaled) >> 23) & 0xff;
  return bits == 0xff ? -80 : max(bits - 126, -80);
}
__device__ __forceinline__ float scaled_room(float scaled) { return (float)scaled_top(scaled) - 7.0f; }

// Packed float32 pairs.
__device__ __forceinline__ uint64_t pair(float a, float b) { return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32); }
__device__ __forceinline__ float first_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float second_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
               : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle: rows of 128 bytes, eight of them an atom of 1 KB.
// K-major (Q, K): atoms of eight rows 1 KB apart. MN-major (V: rows are tokens, the product's K): atoms of
// eight tokens 1 KB apart, the next 64 channels a half tile further.
__device__ __forceinline__ uint64_t desc_of(uint32_t addr, uint32_t leading) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// kind::f16 instruction descriptor: float32 accumulator, M = 128, both operands f16 or both bf16.
template <bool F16>
constexpr uint32_t instruction(int n, bool b_mn_major) {
  return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// The whole warp comes here with the same operands, so that they are computed in uniform registers, and
// the lane that elect() chose issues (issued by one thread of a diverged warp, each product took 80 to
// 100 cycles of moves to uniform registers).
__device__ __forceinline__ uint32_t elect() {
  uint32_t mine;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(mine));
  return mine;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t inst, bool add, uint32_t mine) {
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
               "l"(a), "l"(b), "r"(inst), "r"((uint32_t)add), "r"(mine)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t inst, bool add, uint32_t mine) {
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
               "r"(a), "l"(b), "r"(inst), "r"((uint32_t)add), "r"(mine)
               : "memory");
}
// Arrives on `bar` when every product issued so far is done.
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t mine) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
                   smem_u32(bar)),
               "r"(mine)
               : "memory");
}

#define LKV_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define LKV_S8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])

// Tensor memory is read and written in the shape of mma fragments: lane (g, c) = (lane / 4, lane % 4) of
// a warp holds rows g + 8 i of the warp's 32 (i = 0 .. 3) and columns 8 k + 2 c, 8 k + 2 c + 1. A thread
// then needs the scales of a quarter of the columns, each for four rows; with a thread per row every
// scale is a broadcast to every thread, and shared memory's return path was the bound (three
// broadcasts of 128 floats per row and tile).
//
// 16 columns of the 32 rows: word 4 k + e of rows 16 h ..: column group k, rows g (e < 2) and g + 8.
struct Frag {
  uint32_t v[2][8];
};
// In flight until ld_wait.
__device__ __forceinline__ void ld(Frag& f, uint32_t addr) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : LKV_R8(f.v[h], 0) : "r"(addr + (h << 20)));
}
// The registers pass through the wait, so that no use of them is scheduled before it.
__device__ __forceinline__ void ld_wait(Frag& f) {
  asm volatile("tcgen05.wait::ld.sync.aligned;");  // (no clobber: the scales' loads may move over it)
#pragma unroll
  for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(f.v[i / 8][i % 8]));
}
__device__ __forceinline__ void st(uint32_t addr, const Frag& f) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr + (h << 20)), LKV_S8(f.v[h], 0) : "memory");
}
// The 16 columns packed to 8 words of two: word 2 k + e: column group k, rows g and g + 8.
__device__ __forceinline__ void st_packed(uint32_t addr, const uint32_t (&w)[2][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr + (h << 20)), "r"(w[h][0]), "r"(w[h][1]), "r"(w[h][2]),
                 "r"(w[h][3])
                 : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// This thread's query row into its place of the operand tile; returns what its scores have to be
// multiplied with for int8 pages (a power of two). `flip`: negated (a negative softmax scale).
template <int D, bool INT8>
__device__ __forceinline__ float stage_query(const __nv_bfloat16* row, char* tile, int r, bool write, uint32_t flip) {
  uint4 w[D / 8];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    w[i] = row != nullptr ? reinterpret_cast<const uint4*>(row)[i] : make_uint4(0, 0, 0, 0);
    w[i].x ^= flip, w[i].y ^= flip, w[i].z ^= flip, w[i].w ^= flip;
  }
  float back = 1.0f;
  if constexpr (INT8) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(x[k] & 0x7fffu, (x[k] >> 16) & 0x7fffu));
    }
    const float2 by = row_scales(top);
    const float down = by.x;
    back = by.y;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = pack_f16(__uint_as_float(x[k] << 16) * down, __uint_as_float(x[k] & 0xffff0000u) * down);
      w[i] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
  if (write) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(tile + (i / 8) * (kTile * 128) + r * 128 + (((i % 8) ^ (r & 7)) << 4)) = w[i];
  }
  return back;
}

// FINE (bf16 pages): weights in two bf16 terms.
template <int D, bool INT8, bool FINE>
__global__ void __launch_bounds__(Tiles<D, INT8>::kThreads, 1) prefix_tile_kernel(const Params p, const __grid_constant__ CUtensorMap pages_map, int chunk) {
  static_assert(!(INT8 && FINE));
  using T = Tiles<D, INT8>;
  constexpr int kWords = FINE ? 16 : 8;  // columns of tensor memory that 16 tokens' weights take
  extern __shared__ char raw_smem[];
  __shared__ Barriers s;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  char* q_tiles = smem;
  char* raws = q_tiles + (2 + T::kStages) * T::kBytes;
  float* scale_ring = reinterpret_cast<float*>(raws + T::kRaw * T::kRawBytes);  // [kInfo][2][kTile]: keys' x kKeyDown, values' x kScaleDown
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int split = blockIdx.x, j = blockIdx.y, row0 = blockIdx.z * 2 * kTile;
  const int n_rows = min(2 * kTile, p.rows - row0);
  const bool two = n_rows > kTile;
  // The second tile of queries is one stage more where there is none.
  const int n_stages = T::kStages + (two ? 0 : 1);
  char* stages = q_tiles + (two ? 2 : 1) * T::kBytes;
  const int first = split * chunk;                                               // this CTA's tiles of the prefix
  const int n_tiles = min(chunk, (p.prefix_len + kTile - 1) / kTile - first);
  const int n_jobs = two ? 2 * n_tiles : n_tiles;                                // job i: rows i % 2, tile two ? i / 2 : i
  const int end = p.prefix_len - first * kTile;                                  // tokens from the chunk's start on
  if (tid == 0) {
    mbar_init(&s.q_full, 8);
    mbar_init(&s.tail, 1);
    mbar_init(&s.drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.o_full[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
    }
    for (int i = 0; i <= T::kStages; ++i) {
      mbar_init(&s.full[i], INT8 ? 4 : 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < T::kRaw; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_empty[i], 4);
    }
    for (int i = 0; i < kInfo; ++i) mbar_init(&s.info[i], INT8 ? 8 : 1);
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
  const uint32_t tmem = s.tmem;  // columns: S or P of the two row tiles at 0 and 128, O at 256 and 256 + D
  pdl_wait();
  pdl_release();

  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kMany));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kFew));
  if (warp < 8) {
    // ---- weights: a warp has 32 rows, a thread four of them (Frag) -----------------------------------
    const int u = warp / 4, g = lane / 4, c2 = 2 * (lane % 4);
    const int base = (two ? u * kTile : 0) + (warp % 4) * 32 + g;  // this thread's rows: base + 8 i
    const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
    {
      const int r = tid % kTile, row = two ? u * kTile + r : r;
      const __nv_bfloat16* src = nullptr;
      if (row < n_rows) {
        const int x = row0 + row, gr = x % p.group, bt = x / p.group;
        src = p.q + (int64_t)(bt / p.tokens) * p.q_sb + (int64_t)(bt % p.tokens) * p.q_st + (int64_t)(j * p.group + gr) * p.q_sh;
      }
      const float back = stage_query<D, INT8>(src, q_tiles + (two ? u * T::kBytes : 0), r, two || u == 0, sign < 0.0f ? 0x80008000u : 0u);
      if (INT8) s.back[u][r] = (p.scale_log2 == 0.0f ? 1.0f : back) * kKeyUp;
      fence_async();
      if (p.stall != 1 || warp != 0) warp_arrive(&s.q_full, lane);
    }
    float scale[4];
    // (At least a number: a score of -infinity stays one under a softmax scale of zero.)
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = (p.scale_log2 == 0.0f ? FLT_MIN : p.scale_log2 * sign) * (INT8 ? s.back[u][(warp % 4) * 32 + g + 8 * i] : 1.0f);  // its own warp's rows
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;  // lane 32 (warp % 4) of tensor memory
    const uint32_t ts = tmem + lanes + u * kTile, to = tmem + lanes + 2 * kTile + u * D;
    const bool any_live = base - g < n_rows;  // does this warp hold a row at all
    float from[4], l[4];                      // per row: the reference that weights are taken from (log2 domain), their sum
#pragma unroll
    for (int i = 0; i < 4; ++i) from[i] = -INFINITY, l[i] = 0.0f;
    bool ok = true, unset = true;  // has some row no reference yet
    int n_done = 0;
    for (int i = u; i < n_jobs; i += 2, ++n_done) {
      const int t = two ? i >> 1 : i, slot = t % kInfo;
      ok = wait_for(s, &s.info[slot], (t / kInfo) & 1);
      const uint32_t have = (s.have[slot][0] | s.have[slot][1]) | (s.have[slot][2] | s.have[slot][3]);
      const int seen = end - t * kTile;  // tokens of this tile inside the prefix
      // Pair 4 k: columns 8 k + c2, + 1.
      [[maybe_unused]] const uint64_t* ks = reinterpret_cast<const uint64_t*>(scale_ring + slot * 2 * kTile + c2);
      [[maybe_unused]] const uint64_t* vs = ks + kTile / 2;
      const float most = INT8 ? __int_as_float((127 + kMostF16 - max(max(s.top[slot][0], s.top[slot][1]), max(s.top[slot][2], s.top[slot][3]))) << 23) : kMostBf16;
      ok = ok && wait_for(s, &s.s_full[u], n_done & 1);
      if (!ok) break;
      tc_after();
      if (any_live) {
        constexpr int N = kTile / 16;
        Frag f[2];
        if (have != 0xffu || seen < kTile) {
          // Columns without a token, or past the prefix's end, get scores of -infinity (their key scales are 1).
#pragma unroll 1
          for (int n = 0; n < N; ++n) {
            ld(f[0], ts + 16 * n);
            ld_wait(f[0]);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const int col = 16 * n + 8 * ((x % 8) / 4) + c2 + (x & 1);
              if (col >= seen || !((have >> n) & 1)) f[0].v[x / 8][x % 8] = 0xff800000u;
            }
            st(ts + 16 * n, f[0]);
          }
          st_wait();
        }
        auto score = [&](const Frag& a, int k, int r) {
          return pair(__uint_as_float(a.v[r / 2][4 * k + 2 * (r & 1)]), __uint_as_float(a.v[r / 2][4 * k + 2 * (r & 1) + 1]));
        };
        // One pass, from the references as they are; where there are none yet or a score has outgrown them, they
        // are set from the tile's maxima first. (One copy of each loop: the kernel's first jobs wait for code.)
#pragma unroll 1
        for (bool set = unset, again = false;; again = true) {
          if (set) {
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int n = 0; n < N; ++n) {
              ld(f[0], ts + 16 * n);
              ld_wait(f[0]);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                [[maybe_unused]] uint64_t kk = 0, up = 0;
                if constexpr (INT8) {
                  kk = ks[4 * (2 * n + k)];
                  const uint64_t v = vs[4 * (2 * n + k)];
                  up = pair(scaled_room(first_of(v)), scaled_room(second_of(v)));
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  uint64_t z = score(f[0], k, r);
                  if constexpr (INT8) z = fma2(mul2(z, kk), pair(scale[r], scale[r]), up);
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
              // Rounded up, a reference leaves no score above it.
              const float want = INT8 || top[r] == -INFINITY ? top[r] : __fmul_ru(top[r], scale[r]), to_ref = fmaxf(from[r], want);
              by[r] = to_ref == -INFINITY ? 1.0f : ex2(from[r] - to_ref);
              l[r] = INT8 && to_ref > from[r] ? times_ex2(l[r], from[r] - to_ref) : l[r] * by[r];
              from[r] = to_ref;
              none = none || to_ref == -INFINITY;
            }
            unset = __any_sync(0xffffffffu, none);
            if (n_done > 0) {  // the products of this row tile's last job are done: its scores came after them
#pragma unroll 1
              for (int n = 0; n < D / 16; ++n) {
                ld(f[0], to + 16 * n);
                ld_wait(f[0]);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                  uint32_t& w = f[0].v[x / 8][x % 8];
                  w = __float_as_uint(__uint_as_float(w) * by[2 * (x / 8) + (x % 4) / 2]);
                }
                st(to + 16 * n, f[0]);
              }
            }
          }
          uint64_t ref[4], scale2[4], sum[4] = {0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = from[r] == -INFINITY ? 0.0f : -from[r];
            ref[r] = pair(x, x), scale2[r] = pair(scale[r], scale[r]);
          }
          uint32_t w[N][2][4];
          [[maybe_unused]] uint32_t low[FINE ? N : 1][2][4];
          ld(f[0], ts);
          ld_wait(f[0]);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (n + 1 < N) ld(f[(n + 1) & 1], ts + 16 * (n + 1));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              [[maybe_unused]] uint64_t kk = 0, vv = 0;
              if constexpr (INT8) kk = ks[4 * (2 * n + k)], vv = vs[4 * (2 * n + k)];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                uint64_t z = score(f[n & 1], k, r);
                if constexpr (INT8) z = mul2(z, kk);
                z = fma2(z, scale2[r], ref[r]);
                z = pair(ex2(first_of(z)), ex2(second_of(z)));
                sum[r] = add2(sum[r], z);
                if constexpr (INT8) z = mul2(z, vv);
                uint32_t& to = w[n][r / 2][2 * k + (r & 1)];
                if constexpr (!FINE) {
                  to = INT8 ? pack_f16(first_of(z), second_of(z)) : pack_bf16(first_of(z), second_of(z));
                } else {  // as upper_halves and rest_of
                  to = upper_halves(first_of(z), second_of(z));
                  z = fma2(z, pair(kAndMore, kAndMore), (z & 0xffff0000ffff0000ull) ^ 0x8000000080000000ull);
                  low[n][r / 2][2 * k + (r & 1)] = pack_bf16(first_of(z), second_of(z));
                }
              }
            }
            if (n + 1 < N) ld_wait(f[(n + 1) & 1]);
          }
          // No weight is above the sum that it is part of.
          bool over = false;
#pragma unroll
          for (int r = 0; r < 4; ++r) over = over || fmaxf(first_of(sum[r]), second_of(sum[r])) > most;
          set = !again && __any_sync(0xffffffffu, over);
          if (set) continue;
#pragma unroll
          for (int n = 0; n < N; ++n) {  // over the scores
            st_packed(ts + kWords * n, w[n]);
            if constexpr (FINE) st_packed(ts + kWords * n + 8, low[n]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) l[r] += first_of(sum[r]) + second_of(sum[r]);
          break;
        }
        st_wait();
      }
      tc_before();
      if (p.stall != 2 || warp != 0) warp_arrive(&s.p_full[u], lane);
    }
    // ---- the rows' partials -------------------------------------------------------------------------
    const bool any_job = n_done > 0;
    if (ok && any_job) ok = wait_for(s, &s.o_full[u], 0);
    tc_after();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    const int64_t at = ((int64_t)split * p.h + j) * p.rows + row0 + base;  // row i: at + 8 i
    constexpr int kLd = D + 8;  // a row of the hand-over
    float* swap = reinterpret_cast<float*>(stages);
    float2* swap_ml = reinterpret_cast<float2*>(swap + kTile * kLd);
    float f0[4] = {1.f, 1.f, 1.f, 1.f}, f1[4] = {0.f, 0.f, 0.f, 0.f};
    if (!two) {
      // Both row tiles hold the same rows: the second hands its part over in shared memory. The stages are
      // free: every product that read them is done once both have passed o_full.
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (u == 1 && any_live) {
#pragma unroll 1
        for (int n = 0; n < D / 16; ++n) {
          Frag f;
          if (any_job) {
            ld(f, to + 16 * n);
            ld_wait(f);
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) f.v[x / 8][x % 8] = 0;
          }
#pragma unroll
          for (int x = 0; x < 8; ++x)  // x = 4 k + i: column group k, row i
            *reinterpret_cast<uint2*>(swap + (base + 8 * (x % 4)) * kLd + 16 * n + 8 * (x / 4) + c2) =
                make_uint2(f.v[(x % 4) / 2][4 * (x / 4) + 2 * (x & 1)], f.v[(x % 4) / 2][4 * (x / 4) + 2 * (x & 1) + 1]);
        }
        if (c2 == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) swap_ml[base + 8 * i] = make_float2(from[i], l[i]);
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (u == 0 && any_live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 other = swap_ml[base + 8 * i];
          const float both = fmaxf(from[i], other.x), ref = both == -INFINITY ? 0.0f : both;
          f0[i] = ex2(from[i] - ref), f1[i] = ex2(other.x - ref);
          l[i] = INT8 ? times_ex2(l[i], from[i] - ref) + times_ex2(other.y, other.x - ref) : l[i] * f0[i] + other.y * f1[i];
          from[i] = both;
        }
      }
    }
    if ((two || u == 0) && any_live) {
#pragma unroll 1
      for (int n = 0; n < D / 16; ++n) {
        Frag f;
        ld(f, to + 16 * n);
        ld_wait(f);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int i = x % 4, ch = 16 * n + 8 * (x / 4) + c2;
          float2 o = make_float2(__uint_as_float(f.v[i / 2][4 * (x / 4) + 2 * (i & 1)]), __uint_as_float(f.v[i / 2][4 * (x / 4) + 2 * (i & 1) + 1]));
          if (!two) {
            const float2 other = *reinterpret_cast<const float2*>(swap + (base + 8 * i) * kLd + ch);
            o.x = o.x * f0[i] + other.x * f1[i], o.y = o.y * f0[i] + other.y * f1[i];
          }
          if (base + 8 * i < n_rows) *reinterpret_cast<float2*>(p.tile_o + (at + 8 * i) * D + ch) = o;
        }
      }
      ok = ok && *static_cast<volatile int*>(&s.quit) == 0;
      // Where a wait ran out the row is poisoned (its status word tells why).
      if (c2 == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (base + 8 * i < n_rows) p.tile_ml[at + 8 * i] = ok ? (INT8 ? make_float2(from[i] + kScaleShift, l[i] * kScaleDown) : make_float2(from[i], l[i])) : make_float2(0.0f, __uint_as_float(0x7fc00000u));
      }
    }
    tc_before();
  } else if (warp == 8) {
    // ---- matrix products: issued by one lane, in order -----------------------------------------------
    constexpr uint32_t kQk = instruction<INT8>(kTile, false), kPv = instruction<INT8>(D, true);
    const uint32_t q_u = smem_u32(q_tiles), st_u = smem_u32(stages), mine = elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
    // Keys of job i's tile, or its values, are in place (asked once per tile).
    auto wait_keys = [&](int i) {
      const int n = 2 * (two ? i >> 1 : i);
      return i >= n_jobs || (two && (i & 1) != 0) || wait_for(s, &s.full[n % n_stages], (n / n_stages) & 1);
    };
    auto wait_values = [&](int i) {
      const int t = two ? i >> 1 : i, n = 2 * t + 1;
      return (two && (i & 1) != 0) || (wait_for(s, &s.full[n % n_stages], (n / n_stages) & 1) && (INT8 || end - t * kTile >= kTile || wait_for(s, &s.tail, 0)));
    };
    auto qk = [&](int i) {
      const int t = two ? i >> 1 : i, u = i & 1, slot = 2 * t % n_stages;
      const uint64_t a = desc_of(q_u + (two ? u * T::kBytes : 0), 16), b = desc_of(st_u + slot * T::kBytes, 16);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {  // 16 channels further: 32 bytes, in units of 16
        const uint64_t step = ((x / 4) * T::kHalfBytes + (x % 4) * 32) / 16;
        mma_ss(tm + u * kTile, a + step, b + step, kQk, x > 0, mine);
      }
      commit(&s.s_full[u], mine);
      if (!two || u == 1) commit(&s.empty[slot], mine);
    };
    auto pv = [&](int i) {
      const int t = two ? i >> 1 : i, u = i & 1, slot = (2 * t + 1) % n_stages;
      const uint64_t b = desc_of(st_u + slot * T::kBytes, T::kHalfBytes);
#pragma unroll
      for (int x = 0; x < kTile / 16; ++x)  // 16 tokens further: 2 KB of V, 8 columns of P
        mma_ts(tm + 2 * kTile + u * D, tm + u * kTile + kWords * x, b + x * (2048 / 16), kPv, x > 0 || i > 1, mine);
      if constexpr (FINE) {
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x) mma_ts(tm + 2 * kTile + u * D, tm + u * kTile + kWords * x + 8, b + x * (2048 / 16), kPv, true, mine);
      }
      if (!two || u == 1) commit(&s.empty[slot], mine);
      if (i + 2 >= n_jobs) commit(&s.o_full[u], mine);
    };
    // The scores of job i + 2 follow the output of job i at once (the weights wait for both): their
    // operands are asked for before the weights are.
    bool ok = wait_for(s, &s.q_full, 0);
    for (int i = 0; ok && i < 2 && i < n_jobs; ++i) {
      ok = wait_keys(i);
      tc_after();
      if (ok) qk(i);
    }
    for (int i = 0; ok && i < n_jobs; ++i) {
      ok = wait_values(i) && wait_keys(i + 2) && wait_for(s, &s.p_full[i & 1], (i >> 1) & 1);
      if (!ok) break;
      tc_after();
      pv(i);
      if (i + 2 < n_jobs) qk(i + 2);
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
    const int bs = 1 << p.page_shift, per = kTile >> p.page_shift;  // pages per tile
    int filled = 0;
    bool ok = true;
    // Lane i has page i of the tile, looked up a tile ahead (its id, checked where it is used).
    int page = -1, next = -1;
    auto look_up = [&](int t) {
      const int tok = (first + t) * kTile + lane * bs, blk = tok >> p.page_shift;
      next = t < n_tiles && lane < per && tok < p.prefix_len && blk < p.prefix_cols ? p.prefix_table[blk] : -1;
    };
    look_up(0);
    for (int n = 0; ok && n < 2 * n_tiles; ++n) {
      const int t = n >> 1, kv = n & 1;
      if (kv == 0) {
        page = next < p.n_pages ? next : -1;
        look_up(t + 1);
      }
      if constexpr (!INT8) {
        const int slot = n % n_stages;
        if (n >= n_stages) ok = wait_for(s, &s.empty[slot], (n / n_stages - 1) & 1);
        if (!ok) break;
        const uint32_t granules = lane < per && page >= 0 ? ((1u << (bs / 16)) - 1) << (lane * (bs / 16)) : 0u;
        const uint32_t have = __reduce_or_sync(0xffffffffu, granules);
        if (lane == 0) mbar_arrive_expect_tx(&s.full[slot], T::kBytes);
        __syncwarp();
        if (lane < per) {
          const int rows = p.n_pages * 2 * p.h * bs;  // one past the last: zeros
          const int y = page >= 0 ? ((page * p.h + j) * 2 + kv) * bs : rows;
          const uint32_t dst = smem_u32(stages) + slot * T::kBytes + lane * bs * 128;
#pragma unroll
          for (int h2 = 0; h2 < T::kHalves; ++h2) tma_2d(dst + h2 * T::kHalfBytes, &pages_map, 64 * h2, y, &s.full[slot]);
        }
        filled = n + 1;
        if (lane == 0 && kv == 0) {
          s.have[t % kInfo][0] = have;
          s.have[t % kInfo][1] = s.have[t % kInfo][2] = s.have[t % kInfo][3] = 0;
          mbar_arrive(&s.info[t % kInfo]);
        }
        const int seen = end - t * kTile;
        if (kv == 1 && seen < kTile) {
          // Rows of the last page past the prefix hold anything, a NaN too, and 0 x NaN is NaN.
          ok = wait_for(s, &s.full[slot], (n / n_stages) & 1);
          if (!ok) break;
          for (int h2 = 0; h2 < T::kHalves; ++h2)
            for (int x = seen * 8 + lane; x < kTile * 8; x += 32)
              reinterpret_cast<uint4*>(stages + slot * T::kBytes + h2 * T::kHalfBytes)[x] = make_uint4(0, 0, 0, 0);
          fence_async();
          warp_arrive(&s.tail, lane);
        }
      } else {
        const int slot = n % T::kRaw;
        if (n >= T::kRaw) ok = wait_for(s, &s.raw_empty[slot], (n / T::kRaw - 1) & 1);
        if (!ok) break;
        const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[slot], n_copies * bs * D);
        __syncwarp();
        if (page >= 0)
          tma_load_1d(raws + slot * T::kRawBytes + lane * bs * D,
                      static_cast<const char*>(p.pages) + (((int64_t)page * p.h + j) * 2 + kv) * ((int64_t)bs * D), bs * D, &s.raw_full[slot]);
        filled = n + 1;
      }
    }
    // No copy may land after the CTA has gone, also where the others gave up behind this warp's last copy.
    const int kSlots = INT8 ? T::kRaw : n_stages;
    for (int n = max(0, filled - kSlots); n < filled; ++n) mbar_wait(INT8 ? &s.raw_full[n % kSlots] : &s.full[n % kSlots], (n / kSlots) & 1);
    __syncwarp();
  } else if (warp >= 12) {
    if constexpr (INT8) {
      // ---- codes to f16 operands: warps 12-15 the keys', 16-19 the values'; thread i carries token i's scale --
      const int i = tid % kTile, kv = (tid - 12 * 32) / kTile;
      bool ok = true;
      // Scales are loaded a tile ahead, and their page's id (checked where it is used) a tile before that:
      // neither load is waited for where it is issued.
      float scale = 0.0f;
      bool there = false;
      int id = -1;
      auto page_of = [&](int t) {
        const int pos = (first + t) * kTile + i, blk = pos >> p.page_shift;
        id = t < n_tiles && pos < p.prefix_len && blk < p.prefix_cols ? p.prefix_table[blk] : -1;
      };
      auto scales_of = [&](int t) {
        scale = kv == 0 ? 1.0f : 0.0f;  // of a token that is not there
        there = id >= 0 && id < p.n_pages;
        if (there) {
          const int bs = 1 << p.page_shift, pos = (first + t) * kTile + i;
          scale = p.scales[(((int64_t)id * p.h + j) * 2 + kv) * bs + (pos & (bs - 1))];
        }
        page_of(t + 1);
      };
      page_of(0);
      scales_of(0);
      // A thread's pieces of 16 codes, one channel range of every kStep-th token. Eight lanes take 128 bytes
      // that lie in 32 different banks, and so do the chunks they write: two tokens of different parity, of
      // which the swizzle puts even chunks into even and odd places.
      constexpr int kPer = D / 16, kStep = kTile / kPer;  // kStep is a multiple of 8
      const int odd = (i >> 2) & 1, half = odd ^ ((i >> 3) & 1);
      const int tok0 = kPer == 8 ? (i >> 4) * 2 + odd : i / kPer, c = kPer == 8 ? half * 4 + (i & 3) : i % kPer;
      const int from = (tok0 * kPer + c) * 16, row = (c / 4) * T::kHalfBytes + tok0 * 128, at = (c % 4) * 2;
      const int to0 = row + ((at ^ (tok0 & 7)) << 4), to1 = row + (((at + 1) ^ (tok0 & 7)) << 4);
      for (int t = 0; t < n_tiles; ++t) {
        const int n = 2 * t + kv, raw = n % T::kRaw, slot = n % n_stages, info = t % kInfo;
        // The ring entry's last reader is more than two tiles behind (see the copies): it is free.
        float* ring = scale_ring + (info * 2 + kv) * kTile;
        ring[i] = scale * (kv == 1 ? kScaleDown : kKeyDown);
        if (kv == 1) {
          const int top = __reduce_max_sync(0xffffffffu, scaled_top(scale * kScaleDown));
          if (lane == 0) s.top[info][warp - 16] = top;
        } else {
          const uint32_t mask = __ballot_sync(0xffffffffu, there);
          if (lane == 0) s.have[info][warp - 12] = ((mask & 0xffffu) != 0 ? 1u : 0u) << (2 * (warp - 12)) | (mask >> 16 != 0 ? 2u : 0u) << (2 * (warp - 12));
        }
        warp_arrive(&s.info[info], lane);
        scales_of(t + 1);
        ok = ok && wait_for(s, &s.raw_full[raw], (n / T::kRaw) & 1);
        if (ok && n >= n_stages) ok = wait_for(s, &s.empty[slot], (n / n_stages - 1) & 1);
        if (!ok) break;
        const char* src = raws + raw * T::kRawBytes + from;
        char* dst = stages + slot * T::kBytes;
#pragma unroll
        for (int x0 = 0; x0 < kPer; x0 += 4) {
          uint4 w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = *reinterpret_cast<const uint4*>(src + (x0 + x) * (kStep * kPer * 16));
          if (x0 + 4 >= kPer) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.raw_empty[raw]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint2 a = codes_to_f16(w[x].x), b = codes_to_f16(w[x].y), d = codes_to_f16(w[x].z), e = codes_to_f16(w[x].w);
            *reinterpret_cast<uint4*>(dst + to0 + kStep * (x0 + x) * 128) = make_uint4(a.x, a.y, b.x, b.y);
            *reinterpret_cast<uint4*>(dst + to1 + kStep * (x0 + x) * 128) = make_uint4(d.x, d.y, e.x, e.y);
          }
        }
        fence_async();
        warp_arrive(&s.full[slot], lane);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int D, bool INT8, bool FINE>
cudaError_t launch_tile(const Params& p, const CUtensorMap& map, int chunk, cudaStream_t st) {
  using T = Tiles<D, INT8>;
  auto k = prefix_tile_kernel<D, INT8, FINE>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, T::kSmem, done);
  if (e != cudaSuccess) return e;
  const dim3 grid(p.n_splits, p.h, (p.rows + 2 * kTile - 1) / (2 * kTile));
  return launch_pdl(k, grid, dim3(T::kThreads), T::kSmem, st, 0, p, map, chunk);
}

}  // namespace

// One CTA per SM: the number of splits whose waves of CTAs take the least time, a CTA's start and end
// counted as two tiles of the prefix. (One or four in its place: the same times within 0.5% at 20 to 512 rows of 8
// heads on 8,191 to 131,072 tokens.)
int tile_splits(int rows, int h, int64_t prefix_len) {
  const int64_t tiles = (prefix_len + kTile - 1) / kTile, units = (int64_t)h * ((rows + 2 * kTile - 1) / (2 * kTile));
  int64_t best = 0, best_cost = 0;
  for (int64_t n = 1; n <= tiles && (n == 1 || units * n <= 4 * kNumSMs); ++n) {
    const int64_t chunk = (tiles + n - 1) / n, cost = ((units * n + kNumSMs - 1) / kNumSMs) * (chunk + 2);
    if (best == 0 || cost < best_cost) best = n, best_cost = cost;
  }
  const int64_t chunk = (tiles + best - 1) / best;
  return (int)((tiles + chunk - 1) / chunk);
}

// Test hooks (lkv_debug_set): the bound of the waits, and what warp 0 of every CTA of the next call withholds.
static uint64_t g_max_wait_ns = kMaxWaitNs;
static int g_stall_next = 0;

int set_tile_wait(int64_t ns) {
  if (ns < 1 || ns > (int64_t)kMaxWaitNs) return fail(LKV_ERR_ARG, "lkv_debug_set: prefix wait bound %lld ns outside [1, %llu]", (long long)ns, (unsigned long long)kMaxWaitNs);
  g_max_wait_ns = (uint64_t)ns;
  return LKV_OK;
}
int set_tile_stall(int64_t which) {
  if (which < 0 || which > 2) return fail(LKV_ERR_ARG, "lkv_debug_set: no stall %lld of the prefix tiles (0, 1 or 2)", (long long)which);
  g_stall_next = (int)which;
  return LKV_OK;
}

int run_tiles(Params p, int d, bool int8, cudaStream_t st) {
  static const char* who = "lkv_prefix_attention";
  p.max_wait_ns = g_max_wait_ns;
  p.stall = g_stall_next;
  g_stall_next = 0;
  const int tiles = (p.prefix_len + kTile - 1) / kTile, chunk = (tiles + p.n_splits - 1) / p.n_splits;
  if ((p.rows + 2 * kTile - 1) / (2 * kTile) > 65535) return fail(LKV_ERR_ARG, "%s: too many rows", who);
  CUtensorMap map = {};
  if (!int8) {
    const int bs = 1 << p.page_shift;
    const int64_t rows = (int64_t)p.n_pages * 2 * p.h * bs;
    if (rows > INT32_MAX) return fail(LKV_ERR_ARG, "%s: %lld rows of pages", who, (long long)rows);
    if (rows == 0) return fail(LKV_ERR_ARG, "%s: a prefix in a cache without pages", who);
    const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)d * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)bs}, ones[2] = {1, 1};
    const CUresult r = encode_tiled(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p.pages), dims, strides, box, ones,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LKV_ERR_CUDA, "%s: the pages' tensor map was refused (%d)", who, (int)r);
  }
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (int8) return launch_tile<D, true, false>(p, map, chunk, st);
    return p.out_f32 ? launch_tile<D, false, true>(p, map, chunk, st) : launch_tile<D, false, false>(p, map, chunk, st);
  };
  const cudaError_t e = d == 128 ? launch(std::integral_constant<int, 128>()) : launch(std::integral_constant<int, 64>());
  if (e != cudaSuccess) return fail(LKV_ERR_CUDA, "%s (prefix): %s", who, cudaGetErrorString(e));
  return LKV_OK;
}

}  // namespace prefix

cudaError_t prefix_device_status(int* status, int clear) { return tu_device_status(status, clear); }
cudaError_t prefix_status_attach(int* mirror) { return tu_status_attach(mirror); }

}  // namespace lkv
