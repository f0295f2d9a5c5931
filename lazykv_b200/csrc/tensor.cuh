// What the kernels on the 5th-generation tensor cores have in common: bounded waits that the roles of a CTA
// leave together, operand and instruction descriptors, tcgen05.mma, and tensor memory in fragments.
#pragma once

#include <cuda.h>

#include "tma.cuh"

namespace lkv {
namespace tc {

constexpr int kTile = 128;  // rows of an operand tile

// Waits for the phase of `bar` with the given parity, s.max_wait_ns at most, or until another role gave up (s.quit).
// Without a suspend-time hint: the waits here are short and many, and a hinted one was seen to resume late.
constexpr uint64_t kMaxTensorWaitNs = 2000000000ull;  // unless a test asks for less
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
template <typename S>
__device__ __forceinline__ bool wait_long(S& s, uint64_t* bar, uint32_t parity) {
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
template <typename S>
__device__ __forceinline__ bool wait_for(S& s, uint64_t* bar, uint32_t parity) {
  const bool ok = __all_sync(0xffffffffu, try_once(bar, parity) || wait_long(s, bar, parity)) != 0;
  __syncwarp();
  return ok;
}

// One arrival for the warp, after what all of its lanes did before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

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

}  // namespace tc
}  // namespace lkv
