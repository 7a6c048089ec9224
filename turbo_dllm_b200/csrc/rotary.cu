// Rotary positions on the first `part` values of each head, as pairs (i, i + part/2) or (2i, 2i + 1):
//
//   angle = pos * f_i       a' = s (a cos - b sin)       b' = s (b cos + a sin)       the other values pass through
//
// f_i are the (scaled) inverse frequencies, s the factor of cosine and sine. The backward pass is the same kernel with
// the angle negated. x [rows, H, D] may have any row and head stride; the result is packed.
//
// Angles of far positions lose everything in 32 bits (position 10^6 at frequency 1 is known to 0.03 rad), so the number
// of turns pos * f / 2 pi is formed in 64 bits, whole turns are dropped there, and only the rest goes to 32 bits. All
// heads of a row share their angles: a block computes the cosines and sines of its rows once, in shared memory.
//
// Bound by memory: every value is read once and written once.
#include "common.cuh"
#include "vec_io.cuh"
#include "api.h"

namespace tdllm {
namespace rot {

constexpr int THREADS = 256;

// V values per access: V consecutive pairs (half layout: V values from each half) or V / 2 adjacent pairs
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const T* __restrict__ x, T* __restrict__ out,
                                                         const int* __restrict__ pos, const float* __restrict__ freqs,
                                                         int rows, int H, int D, int part, long long ld_row,
                                                         long long ld_head, int rows_per_block, float scale, float dir) {
  extern __shared__ float2 cs[];   // [rows_per_block][part / 2]
  const int np = part >> 1;
  const long long row0 = (long long)blockIdx.x * rows_per_block;
  const int nr = (int)min((long long)rows_per_block, rows - row0);
  for (int i = threadIdx.x; i < nr * np; i += THREADS) {
    const int r = i / np, j = i - r * np;
    const double turns = (double)pos[row0 + r] * (double)freqs[j] * 0.15915494309189533577;   // 1 / (2 pi)
    const float rest = (float)(2.0 * (turns - rint(turns)));   // half turns, in [-1, 1]
    float s, c;
    sincospif(rest, &s, &c);
    cs[i] = make_float2(c * scale, s * scale * dir);
  }
  __syncthreads();
  // units of a head: pairs first, then the values that pass through
  const int pair_units = (HALF ? np : part) / V;
  constexpr int PV = V * sizeof(T) == 16 ? V : 1;
  const int units = pair_units + (D - part) / PV;
  const int total = nr * H * units;
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const int u = i % units, rh = i / units;
    const int h = rh % H, r = rh / H;
    const T* src = x + (row0 + r) * ld_row + h * ld_head;
    T* dst = out + ((row0 + r) * H + h) * (long long)D;
    const float2* t = cs + r * np;
    if (u < pair_units) {
      float a[V];
      if (HALF) {
        const int j = u * V;
        float b[V];
        vio::load<T, V>(src + j, a);
        vio::load<T, V>(src + np + j, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 k = t[j + e];
          const float p = a[e], q = b[e];
          a[e] = p * k.x - q * k.y;
          b[e] = q * k.x + p * k.y;
        }
        vio::store<T, V>(dst + j, a);
        vio::store<T, V>(dst + np + j, b);
      } else {
        const int j = u * V;   // even; V is 2 at least
        vio::load<T, V>(src + j, a);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 k = t[(j + e) >> 1];
          const float p = a[e], q = a[e + 1];
          a[e] = p * k.x - q * k.y;
          a[e + 1] = q * k.x + p * k.y;
        }
        vio::store<T, V>(dst + j, a);
      }
    } else {
      const int j = part + (u - pair_units) * PV;
      *reinterpret_cast<vio::Raw<T, PV>*>(dst + j) = vio::load_raw<T, PV>(src + j);
    }
  }
}

}  // namespace rot
}  // namespace tdllm

using namespace tdllm;

template <class T>
static int rotary_launch(const T* x, T* out, const int* pos, const float* freqs, int rows, int H, int D, int part,
                         long long ld_row, long long ld_head, int half, float scale, float dir, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte accesses when every piece of a head starts on 16 bytes and fills whole vectors
  const bool vec = !((uintptr_t)x % 16) && !((uintptr_t)out % 16) && !(ld_row % V) && !(ld_head % V) && !(D % V) &&
                   !((half ? part / 2 : part) % V);
  const int np = part / 2;
  const long long per_row = (long long)H * D;
  int rpb = (int)(8192 / per_row);          // about 8192 values per block
  if (rpb < 1) rpb = 1;
  if (rpb > 16) rpb = 16;
  const unsigned grid = (unsigned)((rows + rpb - 1) / rpb);
  const size_t smem = (size_t)rpb * np * sizeof(float2);
#define ROT(VV, HALFV) \
  rot::rotary_kernel<T, VV, HALFV><<<grid, rot::THREADS, smem, st>>>(x, out, pos, freqs, rows, H, D, part, ld_row, ld_head, rpb, scale, dir)
  if (half) {
    if (vec) ROT(V, true);
    else ROT(1, true);
  } else {
    if (vec) ROT(V, false);
    else ROT(2, false);
  }
#undef ROT
  return 0;
}

// dtype: 0 bf16, 1 fp16, 2 fp32. x [rows, H, D] with row and head strides in elements, out packed; pos [rows]; freqs
// [part / 2]; half: pairs (i, i + part/2), else (2i, 2i + 1); dir 1 turns forward, -1 back.
extern "C" int tdllm_rotary(const void* x, void* out, const int* pos, const float* freqs, int rows, int H, int D, int part,
                            long long ld_row, long long ld_head, int half, int dtype, float scale, float dir,
                            void* stream) {
  if (rows < 0 || H < 1 || D < 2 || part < 2 || part > D || part % 2 || part > 2048 || dtype < 0 || dtype > 2) {
    tdllm_host::set_last_error("rotary: an even part of 2..min(D, 2048) values per head (got D %d, part %d)", D, part);
    return 1;
  }
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0)
    rotary_launch((const __nv_bfloat16*)x, (__nv_bfloat16*)out, pos, freqs, rows, H, D, part, ld_row, ld_head, half, scale, dir, st);
  else if (dtype == 1)
    rotary_launch((const __half*)x, (__half*)out, pos, freqs, rows, H, D, part, ld_row, ld_head, half, scale, dir, st);
  else
    rotary_launch((const float*)x, (float*)out, pos, freqs, rows, H, D, part, ld_row, ld_head, half, scale, dir, st);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("rotary launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}
