// Loads and stores of short runs of a row as fp32 values, shared by the
// transformer-block operators: one vector access where the row is aligned,
// element by element elsewhere.
#pragma once

#include "common.cuh"

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

// N (2, 4 or 8) 16-bit elements at an address aligned to 2N bytes, or N fp32
// elements at one aligned to 16 bytes (N = 4 or 8)
template <int N, typename T>
__device__ __forceinline__ void load_aligned(const T* p, float (&v)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
  } else {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (N == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <int N, typename T>
__device__ __forceinline__ void store_aligned(T* p, const float (&v)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// N elements, aligned when ``vec``; otherwise the first ``count`` of them, one
// at a time (the rest read as 0 and are not written)
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* p, int vec, int count, float (&v)[N]) {
  if (vec) {
    load_aligned<N>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < count ? to_f32<T>(p[i]) : 0.0f;
  }
}

template <int N, typename T>
__device__ __forceinline__ void store_vec(T* p, int vec, int count, const float (&v)[N]) {
  if (vec) {
    store_aligned<N>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) p[i] = from_f32<T>(v[i]);
  }
}

// A kernel that may be launched while the one before it in the stream is still
// ending touches no memory before wait_for_prior(); one that lets the next such
// kernel come early says so with let_next_start() (the next one still waits for
// all of it).
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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
