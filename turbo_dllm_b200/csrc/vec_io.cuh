// 16-byte vectors of bf16, fp16 or fp32 values as 32-bit floats, for the bandwidth-bound kernels that take all three.
// Values are handled as pairs of floats in one 64-bit register: one instruction unpacks each value (none for fp32), one
// rounds and packs two, and the packed fp32 instructions do two values of arithmetic.
#pragma once
#include <type_traits>
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

// N (a power of two) consecutive values of T in one access of at most 16 bytes, aligned to its size
template <class T, int N>
struct alignas(N * sizeof(T)) Raw {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, N>*>(p);
}

// N values (a whole 16-byte vector) <-> N / 2 pairs of floats
template <class T, int N>
__device__ __forceinline__ void to_pairs(const Raw<T, N>& r, uint64_t* p) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (sizeof(T) == 4) {
      p[i] = pair_f32(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      p[i] = pair_f32(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(u + i));
      p[i] = pair_f32(f.x, f.y);
    }
  }
}
template <class T, int N>
__device__ __forceinline__ Raw<T, N> from_pairs(const uint64_t* p) {
  Raw<T, N> r;
  uint32_t* u = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float a, b;
    unpair_f32(p[i], a, b);
    if constexpr (sizeof(T) == 4) {
      u[2 * i] = __float_as_uint(a);
      u[2 * i + 1] = __float_as_uint(b);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      u[i] = pack_bf16x2(a, b);
    } else {
      const __half2 h = __floats2half2_rn(a, b);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return r;
}
// values outside [0, H) of the N that start at e become zero
template <int N>
__device__ __forceinline__ void trim_pairs(uint64_t* p, int e, int H) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float a, b;
    unpair_f32(p[i], a, b);
    p[i] = pair_f32(e + 2 * i >= 0 && e + 2 * i < H ? a : 0.f, e + 2 * i + 1 >= 0 && e + 2 * i + 1 < H ? b : 0.f);
  }
}
// the same N values by single accesses, those outside [0, H) left out (read as zero)
template <class T, int N>
__device__ __forceinline__ void load_pairs_each(const T* row, int e, int H, uint64_t* p) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const int c = e + 2 * i;
    p[i] = pair_f32(row && c >= 0 && c < H ? to_f(row[c]) : 0.f, row && c + 1 >= 0 && c + 1 < H ? to_f(row[c + 1]) : 0.f);
  }
}
template <class T, int N>
__device__ __forceinline__ void store_pairs_each(T* row, int e, int H, const uint64_t* p) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const int c = e + 2 * i;
    float a, b;
    unpair_f32(p[i], a, b);
    if (c >= 0 && c < H) row[c] = from_f<T>(a);
    if (c + 1 >= 0 && c + 1 < H) row[c + 1] = from_f<T>(b);
  }
}
__device__ __forceinline__ uint64_t twice(float v) { return pair_f32(v, v); }
__device__ __forceinline__ float sum_of(uint64_t p) {
  float a, b;
  unpair_f32(p, a, b);
  return a + b;
}

}  // namespace vio
}  // namespace tdllm
