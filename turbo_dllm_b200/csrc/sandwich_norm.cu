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
// Bound by memory: x, res (g) in and h, y out; dy, dh, x, res (g) in and dx, dres (dg) out. A block owns rows that are
// gridDim.x apart and keeps a ring of them in shared memory, filled by bulk copies two or more rows ahead, so the copies
// run while a row's sums are joined and its results are stored; the passes over a row read shared memory. (Rows loaded
// into registers, one ahead, reached 3.4 TB/s forward and 2.9 TB/s backward at 16384 x 4096 bf16; the ring reaches 5.8 TB/s
// (92 us without a gate, 98 with one per channel) and 5.5 TB/s (147 us, both kernels).) The backward pass needs two row sums, the
// second of which depends on the first; it is split into
//   sum du u = sum g w_post u (dh + dt / rms(h)) - mean(dt t) / rms(h) * sum g w_post u t
// so that all three sums are taken together in one reduction. The sums over rows stay in registers, one partial row per
// block goes to memory, and a second kernel adds the partial rows in a fixed order, so results repeat bit for bit. For a
// channel gate (or none) both dw_post = g * A and dg = w_post * A follow from the one sum A = sum_rows d * u.
//
// Any width goes in 16-byte lines: with V values to a line, a row that starts s values behind a 16-byte boundary is cut
// into units [V c - s, V c - s + V). Its lines are bulk-copied as they are, the neighbours' values at both ends included,
// and what lies outside the row is masked off when a line is read; only at the tensors' last rows, behind which no neighbour
// may be, the last values come one by one. Ragged lines are stored value by value. The number of blocks is a multiple of V, so
// s is the same for all rows of a block. All row operands have to be shifted alike (the caller copies one that is not).
// 2999 x 1411 with a full gate, forward / backward: fp16 16 / 44 us, fp32 31 / 33 us. Backward, 16-bit rows have 376 blocks
// of three warps (the cap on partial rows), 11 % of an SM's warps, too few to cover one another's latency: they spend 23 % of
// their time on fixed latencies, 21 % on loads and copies, 13 % each on the block barriers of the row sums and on shared memory.
#include "common.cuh"
#include "vec_io.cuh"
#include "api.h"

namespace tdllm {
namespace sandwich {

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_FULL = 2 };
constexpr int KID = 14;
constexpr int MAX_H = 16384;
constexpr int MAX_THREADS = 512;
constexpr int MOST_THREADS = 544;   // a shifted row of the largest width has one unit more than 512 threads hold
constexpr int MAX_STAGES = 6;
constexpr int BUDGET = 227 * 1024;  // shared memory of a block at most
constexpr int HEADER = 512;         // barriers and the reduction's slots, in front of the ring

struct Args {
  const void *x, *res, *w_post, *w_pre, *gate;
  long long ldx, ldres, ldgate;   // row strides in elements
  int rows, H, gate_kind;
  float a, eps;
  int stages, line_bytes;         // ring: rows, bytes of one tensor's row
};

// sum of N values over the block; every thread gets the sums
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  const int nw = blockDim.x >> 5;
  if (nw == 1) {
    __syncwarp();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();   // the previous sums have been read
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < nw ? red[i * 32 + lane] : 0.f);
}

// The ring of rows of NB tensors. RING false (rows too wide for two stages, or no more than one row per block): rows are
// read from global memory in each pass; the second pass finds them in L2.
template <class T, int V, int NB, bool RING, bool SHIFT>
struct Ring {
  const T* base[NB];      // null: absent, reads as zeros (the slot was cleared)
  long long ld[NB];
  uint8_t* smem;          // [stage][tensor][line_bytes]
  uint32_t bars;
  int stages, line_bytes, H, shift;
  long long last;         // the tensors' last row
  __device__ __forceinline__ void setup(uint8_t* sm, const Args& p) {
    smem = sm + HEADER;
    bars = smem_u32(sm);
    stages = p.stages;
    line_bytes = p.line_bytes;
    H = p.H;
    // row r of every tensor starts (r * H) values behind a 16-byte boundary (strides differ from H by whole lines)
    shift = SHIFT ? (int)(((long long)blockIdx.x * p.H) % V) : 0;
    last = p.rows - 1;
    if (RING && threadIdx.x == 0) {
      for (int s = 0; s < stages; ++s) mbar_init(bars + 8 * s, 1);
      fence_mbar_init();
    }
  }
  __device__ __forceinline__ T* slot(int s, int b) const { return (T*)(smem + ((size_t)s * NB + b) * line_bytes); }
  // absent tensors read as zeros
  __device__ __forceinline__ void clear_absent() {
    if (!RING) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (!base[b])
        for (int s = 0; s < stages; ++s)
          for (int i = threadIdx.x; i < line_bytes / 16; i += blockDim.x)
            reinterpret_cast<uint4*>(slot(s, b))[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // rows whose last line may reach behind the tensor: a line holds up to V rows
  __device__ __forceinline__ bool near_end(long long row) const { return SHIFT && row > last - V; }
  // all threads: a row's lines into a stage (one thread copies; the last rows' last values go in by themselves, and the
  // caller puts a block barrier between this and their use)
  __device__ __forceinline__ void bring(int s, long long row) {
    if (!RING) return;
    const int tail = near_end(row) ? (H + shift) % V : 0;
    if (threadIdx.x == 0) {
      const int lines = SHIFT ? (tail ? (H + shift) / V : (H + shift + V - 1) / V) : H / V;
      uint32_t total = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (base[b]) total += lines * 16;
      mbar_expect_tx(bars + 8 * s, total);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (base[b] && lines)
          bulk_load_1d(smem_u32(slot(s, b)), base[b] + row * ld[b] - shift, lines * 16, bars + 8 * s);
    }
    if (tail && (int)threadIdx.x < tail) {
      const int e = H - tail + threadIdx.x;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (base[b] && e >= 0) slot(s, b)[shift + e] = base[b][row * ld[b] + e];
    }
  }
  // A wait gives up at once while another kernel's recorded error stands, but this block's copies are its own and land all the
  // same: each gets up to 0.2 ms more, so that no stage is filled again, and no block ends, under a copy on its way.
  __device__ __forceinline__ void wait(int s, uint32_t parity) const {
    if (!RING || mbar_wait(bars + 8 * s, parity, KID, s)) return;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(bars + 8 * s, parity) && globaltimer_ns() - t0 < 200000ull) __nanosleep(100);
  }
  // line c of a tensor's row (values e ..) as pairs, zeros outside the row; keep: the bits of the line that are the row's
  __device__ __forceinline__ void read(int s, int b, long long row, int c, int e, bool whole, const uint4& keep, uint64_t* f) const {
    if (RING) {
      vio::Raw<T, V> r = vio::load_raw<T, V>(slot(s, b) + c * V);
      if (SHIFT) {
        uint4* u = reinterpret_cast<uint4*>(&r);
        u->x &= keep.x;
        u->y &= keep.y;
        u->z &= keep.z;
        u->w &= keep.w;
      }
      vio::to_pairs<T, V>(r, f);
    } else {
      const T* at = base[b] ? base[b] + row * ld[b] : nullptr;
      if (at && whole) vio::to_pairs<T, V>(vio::load_raw<T, V>(at + e), f);
      else vio::load_pairs_each<T, V>(at, e, H, f);
    }
  }
};

// How a thread's units lie in its rows: unit i of NV covers the values from e[i] on, line c[i] of shared memory
template <int V, int NV, bool RING, bool SHIFT>
struct Units {
  int c[NV], e[NV];
  bool live[NV], whole[NV];
  uint4 keep[NV];
  __device__ __forceinline__ Units(int shift, int H) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      c[i] = threadIdx.x + i * blockDim.x;
      e[i] = c[i] * V - (SHIFT ? shift : 0);
      live[i] = e[i] < H && (!SHIFT || e[i] + V > 0);
      whole[i] = SHIFT ? e[i] >= 0 && e[i] + V <= H : live[i];
      if (RING && SHIFT) {
        uint32_t m[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          m[w] = 0u;
#pragma unroll
          for (int j = 0; j < V / 4; ++j) {   // one 32-bit value or two 16-bit values to a word
            const int at = e[i] + w * (V / 4) + j;
            if (at >= 0 && at < H) m[w] |= V == 4 ? 0xffffffffu : 0xffffu << (16 * j);
          }
        }
        keep[i] = make_uint4(m[0], m[1], m[2], m[3]);
      }
    }
  }
};
// values e .. e + V - 1 of a weight vector
template <class T, int V>
__device__ __forceinline__ void weight_unit(const T* w, int e, int H, uint64_t* f) {
  if (e >= 0 && e + V <= H && (uintptr_t)(w + e) % 16 == 0) vio::to_pairs<T, V>(vio::load_raw<T, V>(w + e), f);
  else vio::load_pairs_each<T, V>(w, e, H, f);
}
// a block's copies of the weights, shifted like its rows: [w_post, w_pre, channel gate][line_bytes]
template <class T>
__device__ __forceinline__ void copy_weights(T* sm, const T* post, const T* pre, const T* gate, int line, int shift, int H) {
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    const T* w = b == 0 ? post : b == 1 ? pre : gate;
    if (!w) continue;
#pragma unroll 8
    for (int i = threadIdx.x; i < line; i += blockDim.x) {
      const int c = i - shift;
      sm[b * line + i] = c >= 0 && c < H ? w[c] : vio::from_f<T>(0.f);
    }
  }
}
template <class T, int V, bool SHIFT>
__device__ __forceinline__ void store_unit(T* row, int e, bool whole, int H, const uint64_t* f) {
  if (!SHIFT || whole) *reinterpret_cast<vio::Raw<T, V>*>(row + e) = vio::from_pairs<T, V>(f);
  else vio::store_pairs_each<T, V>(row, e, H, f);
}

// The rows a block walks: row index of its n-th row is blockIdx.x + n * gridDim.x.
// SHIFT: the width may be no multiple of V, and the weights need no alignment. GATE: see Args. RING: see Ring.
template <class T, int V, int NV, bool RING, bool SHIFT, int GATE>
__global__ void __launch_bounds__(NV > 2 ? MOST_THREADS : MAX_THREADS, RING ? 2 : 1)
fwd_kernel(const Args p, T* __restrict__ y, T* __restrict__ h, float* __restrict__ rstd) {
  constexpr bool FULL = GATE == GATE_FULL;
  constexpr int NB = FULL ? 3 : 2;
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = (float*)(smem + 64);
  Ring<T, V, NB, RING, SHIFT> ring;
  ring.base[0] = (const T*)p.x;
  ring.base[1] = (const T*)p.res;
  ring.ld[0] = p.ldx;
  ring.ld[1] = p.ldres;
  if constexpr (FULL) {
    ring.base[2] = (const T*)p.gate;
    ring.ld[2] = p.ldgate;
  }
  ring.setup(smem, p);
  const Units<V, NV, RING, SHIFT> un(ring.shift, p.H);
  const T* gate = GATE == GATE_CHANNEL ? (const T*)p.gate : nullptr;
  const long long step = gridDim.x;
  const int n = (int)((p.rows - (long long)blockIdx.x + step - 1) / step);   // rows of this block
  const int S = p.stages;
  // weights: with one row per block in registers, loaded beside the row; of an aligned width straight from L1; else from a
  // copy behind the ring that is shifted like the rows
  constexpr bool HELD = !RING && NV == 2, COPIED = !HELD && SHIFT;
  constexpr int P = V / 2;
  T* s_w = (T*)(smem + HEADER + (RING ? (size_t)S * NB * p.line_bytes : 0));
  const int line = p.line_bytes / (int)sizeof(T);
  vio::Raw<T, V> held[3][HELD ? NV : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint64_t f[P];
      weight_unit<T, V>((const T*)p.w_post, un.e[i], p.H, f);
      held[0][i] = vio::from_pairs<T, V>(f);   // (exact: the values came as T)
      weight_unit<T, V>((const T*)p.w_pre, un.e[i], p.H, f);
      held[1][i] = vio::from_pairs<T, V>(f);
      if constexpr (GATE == GATE_CHANNEL) {
        weight_unit<T, V>(gate, un.e[i], p.H, f);
        held[2][i] = vio::from_pairs<T, V>(f);
      }
    }
  }
  auto weight = [&](int b, const T* w, int i, uint64_t* f) {
    if constexpr (HELD) vio::to_pairs<T, V>(held[b][i], f);
    else if constexpr (COPIED) vio::to_pairs<T, V>(vio::load_raw<T, V>(s_w + b * line + un.c[i] * V), f);
    else vio::to_pairs<T, V>(vio::load_raw<T, V>(w + un.e[i]), f);
  };
  __syncthreads();
  for (int k = 0; RING && k < S - 1 && k < n; ++k) {
    ring.bring(k, blockIdx.x + k * step);
  }
  if constexpr (COPIED) copy_weights<T>(s_w, (const T*)p.w_post, (const T*)p.w_pre, gate, line, ring.shift, p.H);
  __syncthreads();
  int s = 0;
  uint32_t parity = 0;
  for (int k = 0; k < n; ++k) {
    const long long row = blockIdx.x + k * step;
    ring.wait(s, parity);
    uint64_t hv[NV][P], sq = 0ull;
    float ss[1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (un.live[i]) {
        ring.read(s, 0, row, un.c[i], un.e[i], un.whole[i], un.keep[i], hv[i]);
#pragma unroll
        for (int j = 0; j < P; ++j) sq = fma_f32x2(hv[i][j], hv[i][j], sq);
      }
    }
    ss[0] = vio::sum_of(sq);
    row_sum(ss, red);
    // every thread is past the previous row: its stage takes the row S - 1 ahead
    const int sn = s ? s - 1 : S - 1;
    if (RING && k + S - 1 < n) ring.bring(sn, row + (S - 1) * step);
    const float r1 = rsqrtf(ss[0] / (float)p.H + p.eps);
    sq = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!un.live[i]) continue;
      uint64_t w[P], v[P];
      weight(0, (const T*)p.w_post, i, w);
      if constexpr (GATE != GATE_NONE) {
        if constexpr (FULL) ring.read(s, NB - 1, row, un.c[i], un.e[i], un.whole[i], un.keep[i], v);
        else weight(2, gate, i, v);
#pragma unroll
        for (int j = 0; j < P; ++j) w[j] = mul_f32x2(w[j], v[j]);
      }
      ring.read(s, 1, row, un.c[i], un.e[i], un.whole[i], un.keep[i], v);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint64_t b = mul_f32x2(mul_f32x2(hv[i][j], vio::twice(r1)), w[j]);
        hv[i][j] = fma_f32x2(vio::twice(p.a), v[j], b);
        sq = fma_f32x2(hv[i][j], hv[i][j], sq);
      }
      store_unit<T, V, SHIFT>(h + row * p.H, un.e[i], un.whole[i], p.H, hv[i]);
    }
    ss[0] = vio::sum_of(sq);
    row_sum(ss, red);
    const float r2 = rsqrtf(ss[0] / (float)p.H + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!un.live[i]) continue;
      uint64_t w[P];
      weight(1, (const T*)p.w_pre, i, w);
#pragma unroll
      for (int j = 0; j < P; ++j) w[j] = mul_f32x2(w[j], mul_f32x2(hv[i][j], vio::twice(r2)));
      store_unit<T, V, SHIFT>(y + row * p.H, un.e[i], un.whole[i], p.H, w);
    }
    if (threadIdx.x == 0 && rstd) {
      rstd[row] = r1;
      rstd[p.rows + row] = r2;
    }
    if (++s == S) {
      s = 0;
      parity ^= 1;
    }
  }
}

// part: [blocks][2][H]: the two row sums of each block
template <class T, int V, int NV, bool RING, bool SHIFT, int GATE>
__global__ void __launch_bounds__(NV > 2 ? MOST_THREADS : MAX_THREADS, 1)
bwd_kernel(const Args p, const T* __restrict__ dy, const T* __restrict__ dh, const float* __restrict__ rstd,
           T* __restrict__ dx, T* __restrict__ dres, T* __restrict__ dgate, float* __restrict__ part) {
  constexpr bool FULL = GATE == GATE_FULL;
  constexpr int NB = FULL ? 5 : 4;
  constexpr bool HELD = NV == 2;   // weights in registers
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = (float*)(smem + 64);
  Ring<T, V, NB, RING, SHIFT> ring;
  ring.base[0] = (const T*)p.x;
  ring.base[1] = (const T*)p.res;
  ring.base[2] = dy;
  ring.base[3] = dh;
  ring.ld[0] = p.ldx;
  ring.ld[1] = p.ldres;
  ring.ld[2] = ring.ld[3] = p.H;
  if constexpr (FULL) {
    ring.base[4] = (const T*)p.gate;
    ring.ld[4] = p.ldgate;
  }
  ring.setup(smem, p);
  const Units<V, NV, RING, SHIFT> un(ring.shift, p.H);
  const T* wq = (const T*)p.w_post;
  const T* wp = (const T*)p.w_pre;
  const T* gate = GATE == GATE_CHANNEL ? (const T*)p.gate : nullptr;
  const long long step = gridDim.x;
  const int n = (int)((p.rows - (long long)blockIdx.x + step - 1) / step);
  ring.clear_absent();
  __syncthreads();
  const int S = p.stages;
  for (int k = 0; RING && k < S - 1 && k < n; ++k) {
    ring.bring(k, blockIdx.x + k * step);
  }
  constexpr int P = V / 2;
  // held: g w_post (w_post alone for a full gate) as floats, w_pre as it came; wider rows read copies in shared memory
  uint64_t gwh[HELD ? NV : 1][P];
  vio::Raw<T, V> hp[HELD ? NV : 1];
  T* s_w = (T*)(smem + HEADER + (RING ? (size_t)S * NB * p.line_bytes : 0));
  const int line = p.line_bytes / (int)sizeof(T);
  if constexpr (!HELD) copy_weights<T>(s_w, wq, wp, gate, line, ring.shift, p.H);
  auto weight = [&](int b, const T* w, int i, uint64_t* f) {
    if constexpr (HELD) weight_unit<T, V>(w, un.e[i], p.H, f);
    else vio::to_pairs<T, V>(vio::load_raw<T, V>(s_w + b * line + un.c[i] * V), f);
  };
  auto gated = [&](int i, uint64_t* gw) {   // w_post, times a channel gate
    weight(0, wq, i, gw);
    if constexpr (GATE == GATE_CHANNEL) {
      uint64_t g[P];
      weight(2, gate, i, g);
#pragma unroll
      for (int j = 0; j < P; ++j) gw[j] = mul_f32x2(gw[j], g[j]);
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      gated(i, gwh[i]);
      uint64_t f[P];
      weight(1, wp, i, f);
      hp[i] = vio::from_pairs<T, V>(f);
    }
  }
  __syncthreads();
  const float inv_h = 1.f / (float)p.H;
  uint64_t sum_post[NV][P], sum_pre[NV][P];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < P; ++j) sum_post[i][j] = sum_pre[i][j] = 0ull;
  auto staged = [&](int s, long long row, int b, int i, uint64_t* f) {
    ring.read(s, b, row, un.c[i], un.e[i], un.whole[i], un.keep[i], f);
  };
  auto weights = [&](int i, int s, long long row, uint64_t* gw, uint64_t* q) {   // g w_post and w_pre
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < P; ++j) gw[j] = gwh[i][j];
      vio::to_pairs<T, V>(hp[i], q);
    } else {
      gated(i, gw);
      weight(1, wp, i, q);
    }
    if constexpr (FULL) {
      uint64_t g[P];
      staged(s, row, NB - 1, i, g);
#pragma unroll
      for (int j = 0; j < P; ++j) gw[j] = mul_f32x2(gw[j], g[j]);
    }
  };
  int s = 0;
  uint32_t parity = 0;
  float n1 = n > 0 ? rstd[blockIdx.x] : 0.f, n2 = n > 0 ? rstd[p.rows + blockIdx.x] : 0.f;
  for (int k = 0; k < n; ++k) {
    const long long row = blockIdx.x + k * step;
    const float r1 = n1, r2 = n2;
    if (k + 1 < n) {
      n1 = rstd[row + step];
      n2 = rstd[p.rows + row + step];
    }
    ring.wait(s, parity);
    uint64_t s0 = 0ull, s1 = 0ull, s2 = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!un.live[i]) continue;
      uint64_t gw[P], q[P], u[P], t[P], dt[P], d[P];
      weights(i, s, row, gw, q);
      staged(s, row, 0, i, u);
      staged(s, row, 1, i, t);
      staged(s, row, 2, i, dt);
      staged(s, row, 3, i, d);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint64_t b = mul_f32x2(mul_f32x2(u[j], vio::twice(r1)), gw[j]);
        t[j] = mul_f32x2(vio::twice(r2), fma_f32x2(vio::twice(p.a), t[j], b));
        sum_pre[i][j] = fma_f32x2(dt[j], t[j], sum_pre[i][j]);
        dt[j] = mul_f32x2(dt[j], q[j]);
        d[j] = fma_f32x2(vio::twice(r2), dt[j], d[j]);
        s0 = fma_f32x2(dt[j], t[j], s0);
        s1 = fma_f32x2(b, d[j], s1);
        s2 = fma_f32x2(b, t[j], s2);
      }
    }
    float sums[3] = {vio::sum_of(s0), vio::sum_of(s1), vio::sum_of(s2)};
    row_sum(sums, red);
    const int sn = s ? s - 1 : S - 1;
    if (RING && k + S - 1 < n) ring.bring(sn, row + (S - 1) * step);
    const float m1 = sums[0] * inv_h * r2;
    const float m2 = (sums[1] - m1 * sums[2]) * inv_h;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!un.live[i]) continue;
      uint64_t gw[P], q[P], u[P], t[P], d[P];
      weights(i, s, row, gw, q);
      staged(s, row, 2, i, t);
      staged(s, row, 3, i, d);
#pragma unroll
      for (int j = 0; j < P; ++j) d[j] = fma_f32x2(vio::twice(r2), mul_f32x2(t[j], q[j]), d[j]);
      staged(s, row, 0, i, u);
      staged(s, row, 1, i, t);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        u[j] = mul_f32x2(u[j], vio::twice(r1));
        t[j] = mul_f32x2(vio::twice(r2), fma_f32x2(vio::twice(p.a), t[j], mul_f32x2(u[j], gw[j])));
        d[j] = fma_f32x2(t[j], vio::twice(-m1), d[j]);
        q[j] = mul_f32x2(vio::twice(p.a), d[j]);
      }
      store_unit<T, V, SHIFT>(dres + row * p.H, un.e[i], un.whole[i], p.H, q);
#pragma unroll
      for (int j = 0; j < P; ++j)
        q[j] = mul_f32x2(vio::twice(r1), fma_f32x2(u[j], vio::twice(-m2), mul_f32x2(d[j], gw[j])));
      store_unit<T, V, SHIFT>(dx + row * p.H, un.e[i], un.whole[i], p.H, q);
      if constexpr (FULL) {
        uint64_t g[P];
        staged(s, row, NB - 1, i, g);
        if constexpr (HELD) {
#pragma unroll
          for (int j = 0; j < P; ++j) gw[j] = gwh[i][j];
        } else {
          gated(i, gw);
        }
#pragma unroll
        for (int j = 0; j < P; ++j) {
          u[j] = mul_f32x2(u[j], d[j]);
          q[j] = mul_f32x2(gw[j], u[j]);
          sum_post[i][j] = fma_f32x2(u[j], g[j], sum_post[i][j]);
        }
        store_unit<T, V, SHIFT>(dgate + row * p.H, un.e[i], un.whole[i], p.H, q);
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) sum_post[i][j] = fma_f32x2(u[j], d[j], sum_post[i][j]);
      }
    }
    // the block's last row has come in: values may have been put in by themselves, a barrier before they are read
    if (RING && SHIFT && k + S == n) __syncthreads();
    if (++s == S) {
      s = 0;
      parity ^= 1;
    }
  }
  float* mine = part + (long long)blockIdx.x * 2 * p.H;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = un.e[i] + j;
      float a[2], b[2];
      unpair_f32(sum_post[i][j / 2], a[0], a[1]);
      unpair_f32(sum_pre[i][j / 2], b[0], b[1]);
      if (c >= 0 && c < p.H) {
        mine[c] = a[j & 1];
        mine[p.H + c] = b[j & 1];
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

// Column sums of the partial rows: 32 columns x 32 row lanes per block. Launched while the partial sums are still being
// made; the dependency wait returns when they are complete and visible.
template <class T>
__global__ void __launch_bounds__(1024) finish_kernel(const float* __restrict__ part, int parts, const Args p, Out dw_post,
                                                      Out dw_pre, Out dgate) {
  __shared__ float sm[2][32][33];
  const int lane = threadIdx.x & 31, lanes = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s0 = 0.f, s1 = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c < p.H) {
#pragma unroll 4
    for (int r = lanes; r < parts; r += 32) {
      s0 += part[(size_t)r * 2 * p.H + c];
      s1 += part[(size_t)r * 2 * p.H + p.H + c];
    }
  }
  sm[0][lanes][lane] = s0;
  sm[1][lanes][lane] = s1;
  __syncthreads();
  if (lanes > 1) return;   // warp 0 joins the first sum, warp 1 the second
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += sm[lanes][i][lane];
  if (c >= p.H) return;
  if (lanes == 1) {
    put<T>(dw_pre, c, s);
    return;
  }
  if (p.gate_kind == GATE_CHANNEL) {
    put<T>(dgate, c, s * vio::to_f(((const T*)p.w_post)[c]));
    s *= vio::to_f(((const T*)p.gate)[c]);
  }
  put<T>(dw_post, c, s);
}

// Units per thread, threads, blocks and the ring. shift: rows or (forward) weights that lines of 16 bytes do not fit.
struct Shape {
  int nv, ring, shift, threads, stages, grid, line_bytes;
  size_t smem;
};
static Shape shape_of(int rows, int H, int elem, int tensors, bool backward, bool weights_fit = true) {
  Shape s;
  const int V = 16 / elem;
  s.shift = H % V != 0 || !weights_fit;
  const int units = H % V ? (H + V - 1 + V - 1) / V : H / V;   // room for any shift
  s.nv = 2;
  while (s.nv * MAX_THREADS < units && s.nv < 32 / V) s.nv *= 2;   // 32 values per thread at most
  s.threads = ((units + s.nv - 1) / s.nv + 31) / 32 * 32;
  s.line_bytes = units * 16;
  const int sms = tdllm_num_sms();
  int resident = (backward || s.nv > 2 ? 512 : 1024) / s.threads;   // by the kernels' registers
  if (resident < 1) resident = 1;
  if (resident > 16) resident = 16;
  const size_t row = (size_t)tensors * s.line_bytes;
  const size_t weights = (size_t)3 * s.line_bytes, budget = BUDGET;
  // a multiple of the values in a line: one shift per block
  auto blocks = [&](int most) { return most < rows ? (most + 7) / 8 * 8 : (rows + 7) / 8 * 8; };
  s.ring = s.nv == 2;
  if (s.ring) {
    const size_t extra = HEADER + (!backward && s.shift ? weights : 0);
    // three rows per block; fewer blocks on an SM where they would not fit (the widest ring has 80 KiB rows: two fit)
    while (resident > 1 && resident * (3 * row + extra + 1024) > budget) --resident;
    s.stages = (int)((budget / resident - extra - 1024) / row);
    if (s.stages > 4) s.stages = 4;
    s.smem = extra + s.stages * row;
    int most = sms * resident;
    // backward: a block's partial sums are two rows of floats; keep them under a sixth of what its own rows move
    if (backward && most > rows * elem / 16) most = rows * elem / 16 > sms ? rows * elem / 16 : sms;
    s.grid = blocks(most);
    if (s.grid >= rows) s.ring = 0;   // one row per block: nothing to bring in ahead
  }
  if (!s.ring) {
    s.stages = 1;
    s.smem = HEADER + (s.nv > 2 ? weights : 0);
    if (s.nv > 2) s.grid = blocks(sms);
  }
  return s;
}

}  // namespace sandwich
}  // namespace tdllm

using namespace tdllm;

// All row operands shifted alike: the same place in a 16-byte line and row strides that differ by whole lines.
static bool sandwich_alike(int elem, int H, const long long* lds, int nld, const void* const* ptrs, int n) {
  for (int i = 0; i < nld; ++i)
    if (((lds[i] - H) * elem) % 16) return false;
  for (int i = 0; i < n; ++i)
    if ((uintptr_t)ptrs[i] % 16) return false;
  return true;
}

// The limit is a property of the kernel and the device that all host threads share: it is set once, to the most that any width
// takes, so that no thread lowers it between another's setting and its launch. `done`: the instantiation's own flags.
template <class K>
static cudaError_t sandwich_smem(K kernel, size_t bytes, bool (&done)[64]) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sandwich::BUDGET);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

#define SANDWICH_GATE(T, V, NV, RING, SHIFT, BODY)                                   \
  if (gate_kind == GATE_NONE) { BODY(T, V, NV, RING, SHIFT, GATE_NONE); }            \
  else if (gate_kind == GATE_CHANNEL) { BODY(T, V, NV, RING, SHIFT, GATE_CHANNEL); } \
  else { BODY(T, V, NV, RING, SHIFT, GATE_FULL); }
// (without the ring: one form for aligned and shifted widths; the shifted form also serves aligned widths, with a shift of 0)
#define SANDWICH_TYPE(T, V, BODY)                                                     \
  if (s.ring && !s.shift) { SANDWICH_GATE(T, V, 2, true, false, BODY) }               \
  else if (s.ring) { SANDWICH_GATE(T, V, 2, true, true, BODY) }                       \
  else if (s.nv == 2) { SANDWICH_GATE(T, V, 2, false, true, BODY) }                   \
  else if (s.nv == 4) { SANDWICH_GATE(T, V, 4, false, true, BODY) }                   \
  else if constexpr (V == 4) { SANDWICH_GATE(T, V, 8, false, true, BODY) }
#define SANDWICH_DISPATCH(BODY)                                                \
  if (dtype == 0) { SANDWICH_TYPE(__nv_bfloat16, 8, BODY) }                    \
  else if (dtype == 1) { SANDWICH_TYPE(__half, 8, BODY) }                      \
  else { SANDWICH_TYPE(float, 4, BODY) }

// a ring of fewer than two rows would wait for a row that nobody brings
static int sandwich_ring(const char* who, const sandwich::Shape& s) {
  if (s.ring ? s.stages >= 2 && s.stages <= sandwich::MAX_STAGES : s.stages == 1) return 0;
  tdllm_host::set_last_error("%s: %d stages", who, s.stages);
  return 1;
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
  const long long lds[3] = {ldx, ldres, gate_kind == GATE_FULL ? ldgate : H};
  const void* ptrs[5] = {x, res, y, h, gate_kind == GATE_FULL ? gate : nullptr};
  if (!sandwich_alike(elem, H, lds, 3, ptrs, 5)) {
    tdllm_host::set_last_error("sandwich_norm_fwd: rows must start on 16 bytes and lie H values plus whole 16 bytes apart");
    return 1;
  }
  // weights that do not start on 16 bytes (a slice of a flat buffer) are copied value by value, as for widths of no whole lines
  const uintptr_t vectors = (uintptr_t)w_post | (uintptr_t)w_pre | (gate_kind == GATE_CHANNEL ? (uintptr_t)gate : 0);
  const Shape s = shape_of(rows, H, elem, gate_kind == GATE_FULL ? 3 : 2, false, vectors % 16 == 0);
  if (sandwich_ring("sandwich_norm_fwd", s)) return 1;
  const Args p = {x, res, w_post, w_pre, gate, ldx, ldres, ldgate, rows, H, gate_kind, a, eps, s.stages, s.line_bytes};
  cudaError_t e = cudaErrorInvalidValue;
#define FWD(T, V, NV, RING, SHIFT, GATE)                                                             \
  do {                                                                                  \
    static bool done[64] = {false};                                                     \
    auto k = fwd_kernel<T, V, NV, RING, SHIFT, GATE>;                                   \
    e = sandwich_smem(k, s.smem, done);                                                 \
    if (e == cudaSuccess)                                                               \
      k<<<s.grid, s.threads, s.smem, (cudaStream_t)stream>>>(p, (T*)y, (T*)h, rstd);    \
  } while (0)
  SANDWICH_DISPATCH(FWD)
#undef FWD
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("sandwich_norm_fwd launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}

// rows of partial sums that tdllm_sandwich_norm_bwd may write: the caller's scratch holds parts * 2 * H floats
extern "C" int tdllm_sandwich_norm_parts(int rows, int H) {
  using namespace tdllm::sandwich;
  if (rows <= 0 || H < 1) return 0;
  int most = 0;
  for (int elem = 2; elem <= 4; elem += 2)      // either type, either kind of gate
    for (int tensors = 4; tensors <= 5; ++tensors) {
      const Shape s = shape_of(rows, H, elem, tensors, true);
      if (s.grid > most) most = s.grid;
    }
  return most;
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
  const long long lds[3] = {ldx, ldres, gate_kind == GATE_FULL ? ldgate : H};
  const void* ptrs[8] = {x, res, dx, dres, dy, dh, gate_kind == GATE_FULL ? gate : nullptr, gate_kind == GATE_FULL ? dgate : nullptr};
  if (!sandwich_alike(elem, H, lds, 3, ptrs, 8)) {
    tdllm_host::set_last_error("sandwich_norm_bwd: rows must start on 16 bytes and lie H values plus whole 16 bytes apart");
    return 1;
  }
  const Shape s = shape_of(rows, H, elem, gate_kind == GATE_FULL ? 5 : 4, true);
  if (sandwich_ring("sandwich_norm_bwd", s)) return 1;
  const Args p = {x, res, w_post, w_pre, gate, ldx, ldres, ldgate, rows, H, gate_kind, a, 0.f, s.stages, s.line_bytes};
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (rows > 0) {
    e = cudaErrorInvalidValue;
#define BWD(T, V, NV, RING, SHIFT, GATE)                                                                                              \
  do {                                                                                                                   \
    static bool done[64] = {false};                                                                                      \
    auto k = bwd_kernel<T, V, NV, RING, SHIFT, GATE>;                                                                    \
    e = sandwich_smem(k, s.smem, done);                                                                                  \
    if (e == cudaSuccess)                                                                                                \
      k<<<s.grid, s.threads, s.smem, st>>>(p, (const T*)dy, (const T*)dh, rstd, (T*)dx, (T*)dres, (T*)dgate, scratch);   \
  } while (0)
    SANDWICH_DISPATCH(BWD)
#undef BWD
    if (e == cudaSuccess) e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    const Out op = {dw_post, post_fp32, post_acc}, oq = {dw_pre, pre_fp32, pre_acc}, og = {dgate_sum, gate_fp32, gate_acc};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((H + 31) / 32);
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = rows > 0 ? 1 : 0;
    const int parts = rows > 0 ? s.grid : 0;
    const float* sc = scratch;
    if (dtype == 0) e = cudaLaunchKernelEx(&cfg, finish_kernel<__nv_bfloat16>, sc, parts, p, op, oq, og);
    else if (dtype == 1) e = cudaLaunchKernelEx(&cfg, finish_kernel<__half>, sc, parts, p, op, oq, og);
    else e = cudaLaunchKernelEx(&cfg, finish_kernel<float>, sc, parts, p, op, oq, og);
  }
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("sandwich_norm_bwd launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}
