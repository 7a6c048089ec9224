// The norms behind and in front of a block, with the block's gate and residual, forward and backward:
//
//   u = x / rms(x)          b = g * (u * w_post)          h = a * res + b
//   t = h / rms(h)          y = t * w_pre                 rms(v) = sqrt(mean(v^2) + eps)
//
// x is the block's output, res the residual stream, g absent, one value per channel or one per element. Backward, with
// the pull-back of v / rms(v) being (d - (v / rms) mean(d v / rms)) / rms:
//
//   dt = dy * w_pre         d = dh + (dt - t mean(dt t)) / rms(h)       dres = a d
//   du = d * g * w_post     dx = (du - u mean(du u)) / rms(x)
//   dw_pre = sum_rows dy * t      dw_post = sum_rows d * g * u          dg = d * u * w_post (summed for a channel gate)
//
// Everything is 32-bit between the loads and the stores; y is formed from h before h is rounded, and the backward pass
// recomputes h from x and res, which it needs anyway, instead of reading the rounded h.
//
// Bound by memory: x, res (g) in and h, y out; dy, dh, x, res (g) in and dx, dres (dg) out. One group of threads owns a
// row and keeps it in registers: forward passes over a row once. The backward pass needs two row sums, the second of
// which depends on the first; it is split into
//   sum du u = sum g w_post u (dh + dt / rms(h)) - mean(dt t) / rms(h) * sum g w_post u t
// so that all three sums are taken together in one reduction. The sums over rows stay in registers while a block walks
// its rows, and one partial row per block goes to memory; a second kernel adds the partial rows in a fixed order, so
// results repeat bit for bit. For a channel gate (or none) both dw_post = g * A and dg = w_post * A follow from the one
// sum A = sum_rows d * u.
#include "common.cuh"
#include "vec_io.cuh"
#include "api.h"

namespace tdllm {
namespace sandwich {

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_FULL = 2 };

struct Args {
  const void *x, *res, *w_post, *w_pre, *gate;
  long long ldx, ldres, ldgate;   // row strides in elements
  int rows, H, gate_kind;
  float a, eps;
};

// sum of N values over the threads of a row (a warp, or the whole block); every thread gets the sums
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int tpr) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (tpr == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5;
  __syncthreads();   // the previous sums have been read
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < nw ? red[i * 32 + lane] : 0.f);
}

// tpr threads per row (32: a warp, several rows per block; else the whole block), NV vectors of V values per thread
template <class T, int V, int NV>
__global__ void __launch_bounds__(1024) fwd_kernel(const Args p, T* __restrict__ y, T* __restrict__ h,
                                                   float* __restrict__ rstd, int tpr) {
  __shared__ float red[32];
  const int rpb = blockDim.x / tpr;
  const long long row = (long long)blockIdx.x * rpb + threadIdx.x / tpr;
  const int t = threadIdx.x % tpr;
  if (row >= p.rows) return;   // (a whole warp, or the whole block)
  const T* x = (const T*)p.x + row * p.ldx;
  const T* res = (const T*)p.res + row * p.ldres;
  const T* wq = (const T*)p.w_post;
  const T* wp = (const T*)p.w_pre;
  const T* gate = (const T*)p.gate + (p.gate_kind == GATE_FULL ? row * p.ldgate : 0);
  float xv[NV][V], rv[NV][V];
  float ss[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * tpr) * V;
    if (c < p.H) {
      vio::load<T, V>(x + c, xv[i]);
      vio::load<T, V>(res + c, rv[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss[0] += xv[i][j] * xv[i][j];
    }
  }
  row_sum(ss, red, tpr);
  const float r1 = rsqrtf(ss[0] / (float)p.H + p.eps);
  ss[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * tpr) * V;
    if (c < p.H) {
      float w[V], g[V];
      vio::load<T, V>(wq + c, w);
      if (p.gate_kind) vio::load<T, V>(gate + c, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float b = xv[i][j] * r1 * w[j];
        if (p.gate_kind) b *= g[j];
        rv[i][j] = fmaf(p.a, rv[i][j], b);
        ss[0] += rv[i][j] * rv[i][j];
      }
      vio::store<T, V>(h + row * p.H + c, rv[i]);
    }
  }
  row_sum(ss, red, tpr);
  const float r2 = rsqrtf(ss[0] / (float)p.H + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * tpr) * V;
    if (c < p.H) {
      float w[V];
      vio::load<T, V>(wp + c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] *= rv[i][j] * r2;
      vio::store<T, V>(y + row * p.H + c, w);
    }
  }
  if (t == 0 && rstd) {
    rstd[row] = r1;
    rstd[p.rows + row] = r2;
  }
}

// part: [gridDim.x * rows per block][2][H]: the two row sums of each row walker
template <class T, int V, int NV>
__global__ void __launch_bounds__(1024) bwd_kernel(const Args p, const T* __restrict__ dy, const T* __restrict__ dh,
                                                   const float* __restrict__ rstd, T* __restrict__ dx,
                                                   T* __restrict__ dres, T* __restrict__ dgate,
                                                   float* __restrict__ part, int tpr) {
  __shared__ float red[3 * 32];
  const int rpb = blockDim.x / tpr;
  const long long walker = (long long)blockIdx.x * rpb + threadIdx.x / tpr;
  const long long walkers = (long long)gridDim.x * rpb;
  const int t = threadIdx.x % tpr;
  const T* wq = (const T*)p.w_post;
  const T* wp = (const T*)p.w_pre;
  const float inv_h = 1.f / (float)p.H;
  float sum_post[NV][V], sum_pre[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sum_post[i][j] = sum_pre[i][j] = 0.f;
  for (long long row = walker; row < p.rows; row += walkers) {
    const T* x = (const T*)p.x + row * p.ldx;
    const T* res = (const T*)p.res + row * p.ldres;
    const T* gate = (const T*)p.gate + (p.gate_kind == GATE_FULL ? row * p.ldgate : 0);
    const float r1 = rstd[row], r2 = rstd[p.rows + row];
    float u[NV][V], tt[NV][V], dt[NV][V], dd[NV][V], gw[NV][V];
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * V;
      if (c < p.H) {
        vio::load<T, V>(x + c, u[i]);
        vio::load<T, V>(res + c, tt[i]);
        vio::load<T, V>(wq + c, gw[i]);
        if (p.gate_kind) {
          float g[V];
          vio::load<T, V>(gate + c, g);
#pragma unroll
          for (int j = 0; j < V; ++j) gw[i][j] *= g[j];
        }
        if (dy) {
          float w[V];
          vio::load<T, V>(dy + row * p.H + c, dt[i]);
          vio::load<T, V>(wp + c, w);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            u[i][j] *= r1;
            tt[i][j] = r2 * fmaf(p.a, tt[i][j], u[i][j] * gw[i][j]);
            sum_pre[i][j] += dt[i][j] * tt[i][j];
            dt[i][j] *= w[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            u[i][j] *= r1;
            tt[i][j] = r2 * fmaf(p.a, tt[i][j], u[i][j] * gw[i][j]);
            dt[i][j] = 0.f;
          }
        }
        if (dh) {
          vio::load<T, V>(dh + row * p.H + c, dd[i]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) dd[i][j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dd[i][j] = fmaf(r2, dt[i][j], dd[i][j]);
          s[0] += dt[i][j] * tt[i][j];
          s[1] += gw[i][j] * u[i][j] * dd[i][j];
          s[2] += gw[i][j] * u[i][j] * tt[i][j];
        }
      }
    }
    row_sum(s, red, tpr);
    const float m1 = s[0] * inv_h * r2;
    const float m2 = (s[1] - m1 * s[2]) * inv_h;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * V;
      if (c < p.H) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dd[i][j] = fmaf(-tt[i][j], m1, dd[i][j]);
          o[j] = p.a * dd[i][j];
        }
        vio::store<T, V>(dres + row * p.H + c, o);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = r1 * fmaf(-u[i][j], m2, dd[i][j] * gw[i][j]);
        vio::store<T, V>(dx + row * p.H + c, o);
        if (p.gate_kind == GATE_FULL) {
          float w[V], g[V];
          vio::load<T, V>(wq + c, w);
          vio::load<T, V>(gate + c, g);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float du = dd[i][j] * u[i][j];
            o[j] = du * w[j];
            sum_post[i][j] += du * g[j];
          }
          vio::store<T, V>(dgate + row * p.H + c, o);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) sum_post[i][j] += dd[i][j] * u[i][j];
        }
      }
    }
  }
  float* mine = part + walker * 2 * p.H;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * tpr) * V;
    if (c < p.H) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        mine[c + j] = sum_post[i][j];
        mine[p.H + c + j] = sum_pre[i][j];
      }
    }
  }
}

struct Out {
  void* p;        // null: not wanted
  int fp32;       // else T
  int accumulate;
};
template <class T>
__device__ __forceinline__ void put(const Out& o, int c, float v) {
  if (!o.p) return;
  if (o.fp32) {
    float* q = (float*)o.p + c;
    *q = o.accumulate ? *q + v : v;
  } else {
    T* q = (T*)o.p + c;
    *q = vio::from_f<T>(o.accumulate ? vio::to_f(*q) + v : v);
  }
}

// Column sums of the partial rows: 32 columns x 8 row lanes per block.
template <class T>
__global__ void __launch_bounds__(256) finish_kernel(const float* __restrict__ part, int parts, const Args p, Out dw_post,
                                                     Out dw_pre, Out dgate) {
  __shared__ float sm[2][8][33];
  const int lane = threadIdx.x & 31, lanes = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s0 = 0.f, s1 = 0.f;
  if (c < p.H) {
    for (int r = lanes; r < parts; r += 8) {
      s0 += part[(size_t)r * 2 * p.H + c];
      s1 += part[(size_t)r * 2 * p.H + p.H + c];
    }
  }
  sm[0][lanes][lane] = s0;
  sm[1][lanes][lane] = s1;
  __syncthreads();
  if (lanes || c >= p.H) return;
  s0 = s1 = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s0 += sm[0][i][lane];
    s1 += sm[1][i][lane];
  }
  put<T>(dw_pre, c, s1);
  if (p.gate_kind == GATE_CHANNEL) {
    put<T>(dgate, c, s0 * vio::to_f(((const T*)p.w_post)[c]));
    s0 *= vio::to_f(((const T*)p.gate)[c]);
  }
  put<T>(dw_post, c, s0);
}

constexpr int MAX_H = 16384;

// threads per row and vectors per thread; a width that does not fill 16-byte vectors goes value by value
struct Shape {
  int v, nv, tpr;
};
static Shape shape_of(int H, int per16, bool vectors) {
  Shape s;
  s.v = vectors ? per16 : 1;
  const int units = (H + s.v - 1) / s.v;
  const int want = vectors ? 1 : 4;   // units per thread before the row gets more threads
  int tpr = 32;
  while (tpr < 1024 && tpr * want < units) tpr *= 2;
  s.tpr = tpr;
  int nv = 1;
  while (nv * tpr < units) nv *= 2;
  s.nv = nv;
  return s;
}

}  // namespace sandwich
}  // namespace tdllm

using namespace tdllm;

static bool sandwich_vectors(int elem, int H, const long long* lds, int nld, const void* const* ptrs, int n) {
  const int per16 = 16 / elem;
  if (H % per16) return false;
  for (int i = 0; i < nld; ++i)
    if (lds[i] % per16) return false;
  for (int i = 0; i < n; ++i)
    if ((uintptr_t)ptrs[i] % 16) return false;
  return true;
}

#define SANDWICH_NV(T, V, BODY)                         \
  switch (s.nv) {                                       \
    case 1: { constexpr int NV = 1; BODY(T, V, NV); break; }   \
    case 2: { constexpr int NV = 2; BODY(T, V, NV); break; }   \
    case 4: { constexpr int NV = 4; BODY(T, V, NV); break; }   \
    case 8: { constexpr int NV = 8; BODY(T, V, NV); break; }   \
    default: { constexpr int NV = 16; BODY(T, V, NV); break; } \
  }
#define SANDWICH_DISPATCH(BODY)                                                              \
  if (dtype == 0) {                                                                          \
    if (vec) { if (s.nv == 1) { BODY(__nv_bfloat16, 8, 1); } else { BODY(__nv_bfloat16, 8, 2); } } \
    else SANDWICH_NV(__nv_bfloat16, 1, BODY)                                                 \
  } else if (dtype == 1) {                                                                   \
    if (vec) { if (s.nv == 1) { BODY(__half, 8, 1); } else { BODY(__half, 8, 2); } }         \
    else SANDWICH_NV(__half, 1, BODY)                                                        \
  } else {                                                                                   \
    if (vec) { if (s.nv == 1) { BODY(float, 4, 1); } else if (s.nv == 2) { BODY(float, 4, 2); } else { BODY(float, 4, 4); } } \
    else SANDWICH_NV(float, 1, BODY)                                                         \
  }

static int sandwich_check(const char* who, int rows, int H, int gate_kind, int dtype) {
  if (rows < 0 || H < 1 || H > sandwich::MAX_H || gate_kind < 0 || gate_kind > 2 || dtype < 0 || dtype > 2) {
    tdllm_host::set_last_error("%s: widths 1..%d, gate kinds 0..2, types 0..2 (got H %d, gate %d, type %d)", who,
                               sandwich::MAX_H, H, gate_kind, dtype);
    return 1;
  }
  return 0;
}

// dtype: 0 bf16, 1 fp16, 2 fp32 (all tensors). gate_kind: 0 none, 1 [H], 2 [rows, H]. rstd: null or [2][rows] for backward.
extern "C" int tdllm_sandwich_norm_fwd(const void* x, const void* res, const void* w_post, const void* w_pre,
                                       const void* gate, void* y, void* h, float* rstd, long long ldx,
                                       long long ldres, long long ldgate, int rows, int H, int gate_kind, int dtype,
                                       float a, float eps, void* stream) {
  using namespace tdllm::sandwich;
  if (sandwich_check("sandwich_norm_fwd", rows, H, gate_kind, dtype)) return 1;
  if (rows == 0) return 0;
  const int elem = dtype == 2 ? 4 : 2;
  const long long lds[3] = {ldx, ldres, gate_kind == GATE_FULL ? ldgate : 0};
  const void* ptrs[7] = {x, res, w_post, w_pre, gate, y, h};
  const bool vec = sandwich_vectors(elem, H, lds, 3, ptrs, 7);
  const Shape s = shape_of(H, 16 / elem, vec);
  const Args p = {x, res, w_post, w_pre, gate, ldx, ldres, ldgate, rows, H, gate_kind, a, eps};
  const int rpb = s.tpr == 32 ? 4 : 1;
  const unsigned grid = (unsigned)(((long long)rows + rpb - 1) / rpb);
#define FWD(T, V, NV) fwd_kernel<T, V, NV><<<grid, s.tpr * rpb, 0, (cudaStream_t)stream>>>(p, (T*)y, (T*)h, rstd, s.tpr)
  SANDWICH_DISPATCH(FWD)
#undef FWD
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("sandwich_norm_fwd launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}

// rows of partial sums that tdllm_sandwich_norm_bwd writes: the caller's scratch holds parts * 2 * H floats
extern "C" int tdllm_sandwich_norm_parts(int rows) {
  const int most = 2 * tdllm_num_sms();
  return rows < most ? (rows + 3) / 4 * 4 : most * 4;
}

// dy / dh null: no gradient comes in there. dw_post, dw_pre, dgate_sum (a channel gate's gradient) may be null;
// *_fp32: fp32 output, else the tensors' type; *_acc: add to what is there. dgate: [rows, H] for a full gate.
extern "C" int tdllm_sandwich_norm_bwd(const void* x, const void* res, const void* w_post, const void* w_pre,
                                       const void* gate, const void* dy, const void* dh, const float* rstd, void* dx,
                                       void* dres, void* dgate, void* dw_post, void* dw_pre, void* dgate_sum,
                                       int post_fp32, int post_acc, int pre_fp32, int pre_acc, int gate_fp32,
                                       int gate_acc, float* scratch, long long ldx, long long ldres, long long ldgate,
                                       int rows, int H, int gate_kind, int dtype, float a, void* stream) {
  using namespace tdllm::sandwich;
  if (sandwich_check("sandwich_norm_bwd", rows, H, gate_kind, dtype)) return 1;
  const int elem = dtype == 2 ? 4 : 2;
  const long long lds[3] = {ldx, ldres, gate_kind == GATE_FULL ? ldgate : 0};
  const void* ptrs[10] = {x, res, w_post, w_pre, gate, dy, dh, dx, dres, dgate};
  const bool vec = sandwich_vectors(elem, H, lds, 3, ptrs, 10);
  const Shape s = shape_of(H, 16 / elem, vec);
  const Args p = {x, res, w_post, w_pre, gate, ldx, ldres, ldgate, rows, H, gate_kind, a, 0.f};
  const int rpb = s.tpr == 32 ? 4 : 1;
  const int most = 2 * tdllm_num_sms();
  int grid = (rows + rpb - 1) / rpb;
  if (grid > most) grid = most;
  cudaStream_t st = (cudaStream_t)stream;
  if (grid > 0) {
#define BWD(T, V, NV)                                                                                              \
  bwd_kernel<T, V, NV><<<grid, s.tpr * rpb, 0, st>>>(p, (const T*)dy, (const T*)dh, rstd, (T*)dx, (T*)dres, (T*)dgate, \
                                                     scratch, s.tpr)
    SANDWICH_DISPATCH(BWD)
#undef BWD
  }
  const Out op = {dw_post, post_fp32, post_acc}, oq = {dw_pre, pre_fp32, pre_acc}, og = {dgate_sum, gate_fp32, gate_acc};
  const int blocks = (H + 31) / 32, parts = grid * rpb;
  if (dtype == 0) finish_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(scratch, parts, p, op, oq, og);
  else if (dtype == 1) finish_kernel<__half><<<blocks, 256, 0, st>>>(scratch, parts, p, op, oq, og);
  else finish_kernel<float><<<blocks, 256, 0, st>>>(scratch, parts, p, op, oq, og);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("sandwich_norm_bwd launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}
