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
// Bound by memory: every value is read once and written once. A head is cut into units of 16 bytes (two of them, one from
// each half, for half pairs); a thread keeps one unit's place, and its cosines and sines in registers, for all the heads
// it takes of a row, two heads' loads at a time. The first are on their way while the angles are formed.
// 16384 rows x 40 heads x 128 bf16: 268 MB read and written in 60 us (5.6 TB/s); with one unit per thread, found by divisions, 88.
#include "common.cuh"
#include "vec_io.cuh"
#include "api.h"

namespace tdllm {
namespace rot {

constexpr int THREADS = 256;

// V values per access: V consecutive pairs (half layout: V values from each half) or V / 2 adjacent pairs (V 1: one pair)
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(THREADS, 4) rotary_kernel(const T* __restrict__ x, T* __restrict__ out,
                                                         const int* __restrict__ pos, const float* __restrict__ freqs,
                                                         int rows, int H, int D, int part, long long ld_row,
                                                         long long ld_head, int rows_per_block, int units, float scale,
                                                         float dir) {
  constexpr int AHEAD = HALF ? 2 : 4;   // heads of a thread whose loads are in flight: 64 bytes
  extern __shared__ __align__(16) float cs[];   // cosines [rows_per_block][part / 2], then sines
  const int np = part >> 1;
  const long long row0 = (long long)blockIdx.x * rows_per_block;
  const int nr = (int)min((long long)rows_per_block, rows - row0);
  constexpr bool ODD = !HALF && V == 1;             // a unit that turns is a pair in two accesses
  const int pair_units = HALF ? np / V : part / (ODD ? 2 : V);
  // threads: unit fastest, then row, then head (each takes every step-th head)
  const int span = min(units, THREADS);             // threads to a (row, head)
  const int lanes = THREADS / span;
  const int lane = threadIdx.x / span, r = lane % rows_per_block, h0 = lane / rows_per_block;
  const int step = lanes / rows_per_block;
  const bool mine = lane < step * rows_per_block && r < nr;
  for (int u = threadIdx.x % span; u < units; u += span) {   // (one pass unless a head has more than 256 units)
    const bool turns = u < pair_units;
    const int j = turns ? u * (ODD ? 2 : V) : part + (u - pair_units) * V;
    const T* src = x + (row0 + r) * ld_row + j;
    T* dst = out + (row0 + r) * H * (long long)D + j;
    vio::Raw<T, V> a[AHEAD], b[AHEAD];
    auto fetch = [&](int h) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const T* at = src + (h + i * step) * ld_head;
        if (!mine || h + i * step >= H) continue;
        if (turns) {
          a[i] = vio::load_raw<T, V>(at);
          if (HALF || ODD) b[i] = vio::load_raw<T, V>(at + (HALF ? np : 1));
        } else {
          a[i] = vio::load_raw<T, V>(at);
        }
      }
    };
    auto pairs_of = [](const vio::Raw<T, V>& w, uint64_t* p) {
      if constexpr (V > 1) vio::to_pairs<T, V>(w, p);
      else p[0] = pair_f32(vio::to_f(w.v[0]), 0.f);
    };
    auto put = [](T* to, const uint64_t* p) {
      if constexpr (V > 1) {
        *reinterpret_cast<vio::Raw<T, V>*>(to) = vio::from_pairs<T, V>(p);
      } else {
        float m, n;
        unpair_f32(p[0], m, n);
        to[0] = vio::from_f<T>(m);
      }
    };
    fetch(h0);
    if (u < span) {   // first pass: the block's angles
      for (int i = threadIdx.x; i < nr * np; i += THREADS) {
        const int rr = i / np, jj = i - rr * np;
        const double whole = (double)pos[row0 + rr] * (double)freqs[jj] * 0.15915494309189533577;   // turns: 1 / (2 pi)
        const float rest = (float)(2.0 * (whole - rint(whole)));   // half turns, in [-1, 1]
        float sn, cn;
        sincospif(rest, &sn, &cn);
        cs[i] = cn * scale;
        cs[rows_per_block * np + i] = sn * scale * dir;
      }
    }
    if (u < span) __syncthreads();
    // cosines and sines of the unit's pairs, two values to a register as the arithmetic wants them
    constexpr int P = V > 1 ? V / 2 : 1;
    uint64_t ck[P], sk[P];
    if (turns && mine) {
      const float* c = cs + r * np + (HALF ? j : j / 2);
      const float* n = c + rows_per_block * np;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        if (!HALF && !ODD) {
          ck[e] = pair_f32(c[e], c[e]);
          sk[e] = pair_f32(-n[e], n[e]);
        } else if (V > 1) {
          ck[e] = pair_f32(c[2 * e], c[2 * e + 1]);
          sk[e] = pair_f32(n[2 * e], n[2 * e + 1]);
        } else {
          ck[e] = pair_f32(c[e], 0.f);
          sk[e] = pair_f32(n[e], 0.f);
        }
      }
    }
    for (int h = h0; mine && h < H; h += AHEAD * step) {
      if (h != h0) fetch(h);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (h + i * step >= H) continue;
        T* to = dst + (long long)(h + i * step) * D;
        if (!turns) {
          *reinterpret_cast<vio::Raw<T, V>*>(to) = a[i];
          continue;
        }
        uint64_t p[P], q[P];
        pairs_of(a[i], p);
        if (HALF || ODD) {
          pairs_of(b[i], q);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const uint64_t m = p[e], n = q[e];
            // (rounded as in the other forms: results do not depend on the layout or the alignment)
            p[e] = fma_f32x2(mul_f32x2(n, vio::twice(-1.f)), sk[e], mul_f32x2(m, ck[e]));
            q[e] = fma_f32x2(m, sk[e], mul_f32x2(n, ck[e]));
          }
          put(to, p);
          put(to + (HALF ? np : 1), q);
        } else {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            float m, n;
            unpair_f32(p[e], m, n);
            p[e] = fma_f32x2(pair_f32(n, m), sk[e], mul_f32x2(p[e], ck[e]));
          }
          put(to, p);
        }
      }
    }
  }
}

}  // namespace rot
}  // namespace tdllm

using namespace tdllm;

template <class T>
static int rotary_launch(const T* x, T* out, const int* pos, const float* freqs, int rows, int H, int D, int part,
                         long long ld_row, long long ld_head, int half, float scale, float dir, cudaStream_t st) {
  // the widest access that every piece of a head fills whole and starts on (a pair of values at least when interleaved)
  const int np = part / 2;
  const long long all = (long long)((uintptr_t)x / sizeof(T)) | (long long)((uintptr_t)out / sizeof(T)) | ld_row | ld_head |
                        D | (half ? np : part) | (D - part);
  int v = 16 / (int)sizeof(T);
  while (v > 1 && all % v) v /= 2;
  // interleaved pairs at odd addresses, or with an odd rest behind them: value by value
  const bool odd = !half && v == 1;
  const int units = (half ? np : part) / (odd ? 2 : v) + (D - part) / v;
  // rows per block: enough heads for a thread to use its angles on, few enough to spread a short call over the GPU
  const int lanes = rot::THREADS / (units < rot::THREADS ? units : rot::THREADS);
  int rpb = 1;
  while (rpb * 2 <= lanes && rpb < 16 && rpb * 2 * np <= 4096 && lanes / rpb * 2 > H / 4 &&
         (long long)rows > 2LL * rpb * tdllm_num_sms())
    rpb *= 2;
  const unsigned grid = (unsigned)((rows + rpb - 1) / rpb);
  const size_t smem = (size_t)rpb * np * 2 * sizeof(float);
#define ROT(VV, HALFV)                                                                                                \
  rot::rotary_kernel<T, VV, HALFV><<<grid, rot::THREADS, smem, st>>>(x, out, pos, freqs, rows, H, D, part, ld_row,    \
                                                                     ld_head, rpb, units, scale, dir)
  constexpr int V = 16 / sizeof(T);
  if (half) {
    if (v == V) ROT(V, true);
    else if (v == V / 2) ROT(V / 2, true);
    else if (V == 8 && v == 2) ROT(2, true);
    else ROT(1, true);
  } else {
    if (v == V) ROT(V, false);
    else if (v == V / 2) ROT(V / 2, false);
    else if (V == 8 && v == 2) ROT(2, false);
    else ROT(1, false);
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
