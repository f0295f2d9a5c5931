// Shared helpers for the sm_100a kernels of liblkv_sm100.so.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/lkv.h"

namespace lkv {

// Records `code` with a printf-style message for lkv_last_error(); returns `code`.
int fail(int code, const char* fmt, ...);
// Checks cudaGetLastError() after a launch; returns LKV_OK or LKV_ERR_CUDA with the message.
int launched(const char* what);

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// The driver's cuTensorMapEncodeTiled (null when the driver does not provide it).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();
// cuTensorMapEncodeTiled through a cache of recently encoded argument sets (same arguments, same map).
CUresult encode_tiled(CUtensorMap* out, CUtensorMapDataType dt, cuuint32_t rank, void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                      const cuuint32_t* box, const cuuint32_t* estr, CUtensorMapInterleave il, CUtensorMapSwizzle sw, CUtensorMapL2promotion l2,
                      CUtensorMapFloatOOBfill oob);
// The status word of select.cu's kernels with bounded waits (see tma.cuh).
cudaError_t select_device_status(int* status, int clear);
// Points select.cu's kernels on the current device at the host mirror of the status word.
cudaError_t select_status_attach(int* mirror);
// The status word of prefix_tile.cu's kernels and its host mirror.
cudaError_t prefix_device_status(int* status, int clear);
cudaError_t prefix_status_attach(int* mirror);
// Test hooks of those kernels' waits (prefix_tile.cu).
namespace prefix {
int set_tile_wait(int64_t ns);
int set_tile_stall(int64_t which);
}
// The exchange's status word (exchange.cu), its host mirror, and the bound of its wait.
cudaError_t exchange_device_status(int* status, int clear);
cudaError_t exchange_status_attach(int* mirror);
int exchange_set_wait_iters(int64_t iters);

constexpr int kNumSMs = 148;  // B200

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

// Round to nearest even, as torch's .to(bfloat16) does.
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float x) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

__device__ __forceinline__ float bf16_round(float x) { return bf16_bits_to_f32(f32_to_bf16_bits(x)); }

// float -> uint32 whose unsigned order is the float order (+0.0 and -0.0 made equal first).
__device__ __forceinline__ uint32_t orderable(float x) {
  uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float from_orderable(uint32_t o) {
  uint32_t u = (o & 0x80000000u) ? (o & 0x7fffffffu) : ~o;
  return __uint_as_float(u);
}

// Programmatic dependent launch: a kernel launched with the programmatic-serialization attribute may
// start while its predecessor in the stream still runs. It calls pdl_wait() before it touches
// anything the predecessor writes (or that a still-running earlier kernel reads), and pdl_release()
// after that, so that its own dependent can start early; both are no-ops in an ordinary launch.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch with the programmatic-serialization attribute (and a cluster of cluster_x CTAs when > 0).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster_x, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  if (cluster_x > 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Loads of 8 consecutive elements as float (16 B of bf16 or 32 B of float32), read-only path.
template <typename T>
struct Vec8;

template <>
struct Vec8<__nv_bfloat16> {
  __device__ __forceinline__ static void load(const __nv_bfloat16* p, float* out) {
    uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = __uint_as_float(w[i] << 16);
      out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

template <>
struct Vec8<float> {
  __device__ __forceinline__ static void load(const float* p, float* out) {
    float4 a = __ldg(reinterpret_cast<const float4*>(p));
    float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    out[0] = a.x; out[1] = a.y; out[2] = a.z; out[3] = a.w;
    out[4] = b.x; out[5] = b.y; out[6] = b.z; out[7] = b.w;
  }
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Asynchronous 16-byte global -> shared copy (all of a thread's copies fly together), and the wait
// for every copy the thread issued.
__device__ __forceinline__ void cp_async16(void* smem_dst, const void* gmem_src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem_dst)), "l"(gmem_src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
}

inline size_t dtype_size(int dtype) { return dtype == LKV_BF16 ? 2 : 4; }
inline bool dtype_ok(int dtype) { return dtype == LKV_F32 || dtype == LKV_BF16; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace lkv
