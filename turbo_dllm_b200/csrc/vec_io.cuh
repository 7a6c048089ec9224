// 16-byte vectors of bf16, fp16 or fp32 values as 32-bit floats, for the bandwidth-bound kernels that take all three.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace tdllm {
namespace vio {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// N consecutive values of T: one 16-byte access when N fills it, else value by value
template <class T, int N>
struct alignas(N * sizeof(T) == 16 ? 16 : sizeof(T)) Raw {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, N>*>(p);
}
template <class T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& r, float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f(r.v[i]);
}
template <class T, int N>
__device__ __forceinline__ void load(const T* p, float* f) {
  unpack<T, N>(load_raw<T, N>(p), f);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const float* f) {
  Raw<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Raw<T, N>*>(p) = r;
}

}  // namespace vio
}  // namespace tdllm
