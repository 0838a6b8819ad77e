// Conversions, loads and launches shared by the transformer-block operators.
#pragma once

#include "common.cuh"

#include <atomic>

namespace peco {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

// Eight 16-bit elements as fp32: one access when ``vec`` (aligned to 16 bytes),
// otherwise the first ``count`` of them one at a time (the rest read as 0).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int vec, int count, float (&v)[8]) {
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? to_f32<T>(p[i]) : 0.0f;
  }
}

// A kernel that may be launched while the one before it in the stream is still
// ending touches no memory before wait_for_prior(); one that lets the next such
// kernel come early says so with let_next_start() (the next one still waits for
// all of it).
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A caller's workspace: large enough, and on the 16 bytes that vector stores and TMA start on.
inline bool usable_workspace(const void* workspace, long long bytes, long long need) {
  return workspace && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0;
}

// Dynamic shared memory of a kernel, granted once per device.
inline cudaError_t grant_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launch of a kernel that begins with wait_for_prior().
template <typename... P, typename... A>
int launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  const int st = launch_status();
  return e != cudaSuccess ? static_cast<int>(e) : st;
}

}  // namespace peco
