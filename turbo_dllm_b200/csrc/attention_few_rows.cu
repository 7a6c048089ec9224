// Attention of a few new rows (one token, one block of new tokens, a batch of either, a piece of a prompt) against a long
// cache, head width 128, with the score transforms and the declarative mask of the tile kernels. Forward only.
//
// A call reads K and V once and does little with them, so it is bound by memory as long as every SM pulls: the keys are
// split over CTAs. The G query heads of a KV head and the query rows are packed into one row axis (row r = query r / G,
// head r % G), so a KV head's keys are read once for all of them; up to 128 packed rows share a CTA.
//
//   warps 0-7   each 16 packed rows x a share of the tile's keys (WR warps along the rows, 8 / WR along the keys):
//               S = Q K^T with mma.m16n8k16 (Q fragments stay in registers), transform, mask, online softmax, O += P V.
//               The products are a few percent of what one tile's 64 KB of loads take, until the 128 rows of a CTA are
//               full, where both take about the same time.
//   warp 8      brings in the tiles: TMA for K and V (three stages of 64 KB), plain loads for the keys' codes
//
// Split s takes the key tiles s, s + S, s + 2 S, ...: a sequence of a batch, or a sliding window, is a run of tiles, and
// a stride spreads it evenly. Before the loop the warps test each of the CTA's tiles against the bounds of its rows'
// masks; tiles that no row can see are never loaded. Every warp keeps its own running maximum, sum and accumulator (32
// bits); they meet in shared memory at the end, and the splits' partial results (fp32, with their maximum and sum) in a
// second small kernel, in a fixed order.
//
// Measured with 8 KV heads of 4 query heads, scores capped, joining kernel included, calls replayed back to back in a graph
// (what L2 keeps of the call before helps): 1 token x 20000 keys 17.8 us (82 MB; with flushed caches 22.1 us at 3.8 TB/s and
// the join), 4 sequences x 32 tokens x 8192 keys 42.4 us (135 MB; flushed 43.4 and the join), 1 token x 300 keys 8.7 us. From
// 32 rows x 2048 keys (14.7 us) to 32 x 32768 (37.8) the bytes come at 5.4 TB/s, so what a call pays beside them are about
// 13 us of launches, first loads, the last tile's chain and the joining kernel.
//
// Probabilities are rounded to bf16 for the product with V (as in the tile kernels), sums use them unrounded. V rows of
// keys that none of a warp's 16 rows sees enter the product as zeros, whatever they hold.
#include "common.cuh"
#include "score_mod.cuh"
#include "api.h"

namespace tdllm {
namespace few {

constexpr int KID = 12;
constexpr int HD = 128;
constexpr int BK = 128;
constexpr int STAGES = 3;
constexpr int TILE_BYTES = BK * HD * 2;   // two halves of 64 columns: 128 rows x 128 bytes, swizzled
constexpr int HALF_BYTES = TILE_BYTES / 2;
constexpr int THREADS = 288;
constexpr int ROUND = 1024;               // own tiles per visibility round
constexpr int OFF_CODE = STAGES * 2 * TILE_BYTES;
constexpr int OFF_KPOS = OFF_CODE + STAGES * BK * 4;
constexpr int OFF_ML = OFF_KPOS + STAGES * BK * 4;          // [8 warps][16 rows] max, then sum
constexpr int OFF_BITS = OFF_ML + 2 * 8 * 16 * 4;
constexpr int OFF_BARS = OFF_BITS + ROUND / 8 + 32;
constexpr int SMEM_BYTES = OFF_BARS + 64 + 1024;
static_assert(8 * 16 * HD * 4 <= STAGES * 2 * TILE_BYTES, "the warps' accumulators reuse the stages");

struct Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  float* lse;
  float* part_o;    // [splits][nq * Hq][128]
  float* part_ml;   // [splits][nq * Hq][2]
  const int *q_lo, *q_hi, *q_grp, *k_code, *q_pos, *k_pos;
  const float* slopes;
  long long ldq, ldo, ld_lse;
  int nq, nk, Hq, Hkv, splits, row_tiles;
  float scale_log2;
  score::Mod mod;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool visible(int code, int lo, int hi, int grp) {
  return code >= 0 ? (code >= lo && code < hi) : (code == grp);
}

// The codes of a tile's keys, four per lane (e * 32 + lane); what lies behind the last key is dead.
struct Codes {
  int c[4];
  __device__ __forceinline__ void load(const Params& p, int k0, int lane) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + e * 32 + lane;
      c[e] = k < p.nk ? __ldg(p.k_code + k) : score::DEAD_KEY;
    }
  }
};
// Bounds over a CTA's rows, in shared memory: lo_min, hi_max (rows with a clean interval), grp_min, grp_max (noisy
// rows), and over all rows lo_max, hi_min.
struct Bounds {
  int v[6];
  __device__ __forceinline__ void clear() {
    v[0] = 2147483647; v[1] = -1; v[2] = 0; v[3] = score::DEAD_KEY; v[4] = -2147483647 - 1; v[5] = 2147483647;
  }
  __device__ __forceinline__ void add(int lo, int hi, int grp) {
    if (lo < hi) {
      atomicMin(v, lo);
      atomicMax(v + 1, hi);
    }
    if (grp < 0) {
      atomicMin(v + 2, grp);
      atomicMax(v + 3, grp);
    }
    atomicMax(v + 4, lo);
    atomicMin(v + 5, hi);
  }
  __device__ __forceinline__ bool may_see(int c) const {
    return c >= 0 ? (c >= v[0] && c < v[1]) : (c >= v[2] && c <= v[3] && c != score::DEAD_KEY);
  }
  __device__ __forceinline__ bool all_see(int c) const { return c >= 0 && c >= v[4] && c < v[5]; }
};

// a row's log-sum-exp from its maximum (log2 units) and sum: -inf for a row that sees nothing, NaN for one with NaN scores
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.f ? -INFINITY : top * 0.69314718055994531f + __logf(sum);
}

// writes one finished row value range: 4 values of row r (packed index) starting at column c
__device__ __forceinline__ void store_row4(const Params& p, int kvh, int G, int r, int c, const float* v) {
  const int i = r / G, h = kvh * G + r % G;
  uint2 w;
  w.x = pack_bf16x2(v[0], v[1]);
  w.y = pack_bf16x2(v[2], v[3]);
  *reinterpret_cast<uint2*>(p.o + (long long)i * p.ldo + h * HD + c) = w;
}

template <int WR, int MOD>
__global__ void __launch_bounds__(THREADS, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  constexpr int KW = 8 / WR;           // warps along the keys
  constexpr int SB = WR == 1 ? 1 : 2;  // 16-key blocks a warp takes at a time
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int* s_code = (int*)(smem + OFF_CODE);
  float* s_kpos = (float*)(smem + OFF_KPOS);
  float* s_ml = (float*)(smem + OFF_ML);
  uint32_t* s_bits = (uint32_t*)(smem + OFF_BITS);
  Bounds* s_bound = (Bounds*)(s_bits + ROUND / 32);
  const uint32_t bar_full = smem_u32(smem + OFF_BARS), bar_empty = bar_full + 8 * STAGES;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.Hq / p.Hkv;
  const int kvh = blockIdx.x % p.Hkv;
  const int rt = (blockIdx.x / p.Hkv) % p.row_tiles;
  const int split = blockIdx.x / (p.Hkv * p.row_tiles);
  const int rows = p.nq * G;             // packed rows of a KV head
  const int row0 = rt * 16 * WR;
  const int nkt = (p.nk + BK - 1) / BK;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int own = split < nkt ? (nkt - split + p.splits - 1) / p.splits : 0;

  if (tid == 256) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // on their way while the barriers are set up: the codes of this warp's first tile and this thread's row's mask
  Codes first;
  if (warp < own) first.load(p, (split + warp * p.splits) * BK, lane);
  const int i1 = min((row0 + 16 * WR - 1) / G, p.nq - 1), i_mine = row0 / G + tid;   // at most 128 query rows
  int mask_of[3] = {0, 0, 0};
  if (i_mine <= i1) {
    mask_of[0] = p.q_lo[i_mine];
    mask_of[1] = p.q_hi[i_mine];
    mask_of[2] = p.q_grp[i_mine];
  }
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 33);
      mbar_init(bar_empty + 8 * s, 8);
    }
    fence_mbar_init();
    s_bound->clear();
  }
  __syncthreads();
  if (i_mine <= i1) s_bound->add(mask_of[0], mask_of[1], mask_of[2]);

  // compute warps: rows and their metadata
  const int wr = warp % WR, kw = warp / WR;
  const int g = lane >> 2, t4 = lane & 3;
  const int ra = row0 + wr * 16 + g, rb = ra + 8;
  uint32_t qf[8][4];
  int lo[2] = {0, 0}, hi[2] = {0, 0}, grp[2] = {0, 0};
  [[maybe_unused]] float slope2[2] = {0.f, 0.f}, qpos[2] = {0.f, 0.f};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float acc[16][4];
  if (warp < 8) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = x ? rb : ra;
      if (r < rows) {
        const int i = r / G, h = kvh * G + r % G;
        lo[x] = p.q_lo[i];
        hi[x] = p.q_hi[i];
        grp[x] = p.q_grp[i];
        if constexpr ((MOD & score::BIAS) != 0) {
          slope2[x] = p.slopes[h] * 1.4426950408889634f;
          qpos[x] = score::position(p.q_pos[i]);
        }
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (long long)i * p.ldq + h * HD) + t4;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[k][x] = src[k * 8];
          qf[k][x + 2] = src[k * 8 + 4];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) qf[k][x] = qf[k][x + 2] = 0u;
      }
    }
  }

  int it = 0;        // tiles through the pipeline so far: stage it % STAGES
  bool ok = true;
  for (int base = 0; base < own; base += ROUND) {
    const int cnt = min(ROUND, own - base);
    __syncthreads();   // the previous round's bits have been read; the bounds are complete
    for (int i = tid; i < ROUND / 32; i += THREADS) s_bits[i] = 0u;
    __syncthreads();
    const Bounds bounds = *s_bound;
    for (int o = warp; o < cnt; o += THREADS / 32) {
      if (base + o != warp) first.load(p, (split + (base + o) * p.splits) * BK, lane);
      const bool any = bounds.may_see(first.c[0]) || bounds.may_see(first.c[1]) || bounds.may_see(first.c[2]) ||
                       bounds.may_see(first.c[3]);
      if (__any_sync(0xffffffffu, any) && lane == 0) atomicOr(s_bits + (o >> 5), 1u << (o & 31));
    }
    __syncthreads();
    int total = 0;
    for (int i = 0; i < (cnt + 31) / 32; ++i) total += __popc(s_bits[i]);
    if (warp == 8) {
      int j = 0;
      for (int w = 0; w < (cnt + 31) / 32 && ok; ++w) {
        uint32_t bits = s_bits[w];
        while (bits && ok) {
          const int o = w * 32 + __ffs(bits) - 1;
          bits &= bits - 1;
          const int k0 = (split + (base + o) * p.splits) * BK;
          const int s = (it + j) % STAGES;
          const uint32_t ph = ((it + j) / STAGES) & 1;
          int code[4];
          [[maybe_unused]] int kp[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = k0 + e * 32 + lane;
            code[e] = k < p.nk ? __ldg(p.k_code + k) : score::DEAD_KEY;
            if constexpr ((MOD & score::BIAS) != 0) kp[e] = k < p.nk ? __ldg(p.k_pos + k) : 0;
          }
          ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, KID, 10));
          if (!ok) break;
          if (lane == 0) {
            const uint32_t bar = bar_full + 8 * s;
            const uint32_t dst = smem_u32(smem + s * 2 * TILE_BYTES);
            mbar_expect_tx(bar, 2 * TILE_BYTES);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              tma_load_2d(dst + c * HALF_BYTES, &tm_k, bar, kvh * HD + c * 64, k0);
              tma_load_2d(dst + TILE_BYTES + c * HALF_BYTES, &tm_v, bar, kvh * HD + c * 64, k0);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s_code[s * BK + e * 32 + lane] = code[e];
            if constexpr ((MOD & score::BIAS) != 0) s_kpos[s * BK + e * 32 + lane] = score::position(kp[e]);
          }
          mbar_arrive(bar_full + 8 * s);
          ++j;
        }
      }
    } else {
      for (int j = 0; j < total && ok; ++j) {
        const int s = (it + j) % STAGES;
        const uint32_t ph = ((it + j) / STAGES) & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * s, ph, KID, 20));
        if (!ok) break;
        const uint32_t kb = smem_u32(smem + s * 2 * TILE_BYTES), vb = kb + TILE_BYTES;
        const int* codes = s_code + s * BK;
        const float* kpos = s_kpos + s * BK;
#pragma unroll 1
        for (int b0 = kw * SB; b0 < 8; b0 += KW * SB) {   // SB blocks of 16 keys
          float sc[SB * 2][4];
#pragma unroll
          for (int n = 0; n < SB * 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
#pragma unroll
            for (int b = 0; b < SB; ++b) {
              uint32_t kf[4];
              const int key = (b0 + b) * 16 + (lane >> 4) * 8 + (lane & 7);
              const int chunk = k * 2 + ((lane >> 3) & 1);
              ldsm4(kb + (chunk >> 3) * HALF_BYTES + sw128_offset(key, chunk & 7), kf);
              mma16816(sc[b * 2], qf[k], kf[0], kf[1]);
              mma16816(sc[b * 2 + 1], qf[k], kf[2], kf[3]);
            }
          }
          float mx[2] = {-INFINITY, -INFINITY};
          uint32_t live[SB * 2];   // bit 0, 1: a row of this warp sees key 2 t4 (+1) of the 8
          uint32_t seen = 0u;      // this thread's scores: bit 4 n + e
          uint32_t z[SB * 8];
#pragma unroll
          for (int n = 0; n < SB * 2; ++n) {
            const int key = b0 * 16 + n * 8 + t4 * 2;
            const int c0 = codes[key], c1 = codes[key + 1];
            live[n] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool v = visible((e & 1) ? c1 : c0, lo[e >> 1], hi[e >> 1], grp[e >> 1]);
              live[n] |= (uint32_t)v << (e & 1);
              seen |= (uint32_t)v << (n * 4 + e);
              z[n * 4 + e] = v ? __float_as_uint(sc[n][e]) : 0u;
            }
          }
          if constexpr ((MOD & score::CAP) != 0) score::cap_block<SB * 8>(z, p.mod);
#pragma unroll
          for (int n = 0; n < SB * 2; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int x = e >> 1;
              float v = __uint_as_float(z[n * 4 + e]);
              if constexpr ((MOD & score::CAP) == 0) v *= p.scale_log2;
              if constexpr ((MOD & score::BIAS) != 0)
                v = fmaf(-slope2[x], fabsf(qpos[x] - kpos[b0 * 16 + n * 8 + t4 * 2 + (e & 1)]), v);
              sc[n][e] = ((seen >> (n * 4 + e)) & 1u) ? v : -INFINITY;
              mx[x] = fmaxf(mx[x], sc[n][e]);
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
          }
#pragma unroll
          for (int n = 0; n < SB * 2; ++n) {
            live[n] |= __shfl_xor_sync(0xffffffffu, live[n], 4);
            live[n] |= __shfl_xor_sync(0xffffffffu, live[n], 8);
            live[n] |= __shfl_xor_sync(0xffffffffu, live[n], 16);
          }
          // the reference maximum moves only when the new one is 2^8 larger
          float alpha[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            alpha[x] = 1.f;
            if (mx[x] > -INFINITY && (m[x] == -INFINITY || mx[x] - m[x] > 8.f)) {
              alpha[x] = m[x] == -INFINITY ? 0.f : score::exp2_approx(m[x] - mx[x]);
              m[x] = mx[x];
            }
            l[x] *= alpha[x];
          }
          if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              acc[e][0] *= alpha[0];
              acc[e][1] *= alpha[0];
              acc[e][2] *= alpha[1];
              acc[e][3] *= alpha[1];
            }
          }
          const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
          for (int b = 0; b < SB; ++b) {
            uint32_t pf[4], keep[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {   // keys 0-7, 8-15 of the block
              float* w = sc[b * 2 + hh];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[e] = score::exp2_approx(w[e] - ref[e >> 1]);
                l[e >> 1] += w[e];
              }
              pf[hh * 2] = pack_bf16x2(w[0], w[1]);
              pf[hh * 2 + 1] = pack_bf16x2(w[2], w[3]);
              const uint32_t lv = live[b * 2 + hh];
              keep[hh] = ((lv & 1u) ? 0xffffu : 0u) | ((lv & 2u) ? 0xffff0000u : 0u);
            }
            const bool all = __all_sync(0xffffffffu, (keep[0] & keep[1]) == 0xffffffffu);
#pragma unroll
            for (int d = 0; d < 8; ++d) {   // 16 columns of V at a time
              uint32_t vf[4];
              const int key = (b0 + b) * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
              const int chunk = d * 2 + (lane >> 4);
              ldsm4t(vb + (chunk >> 3) * HALF_BYTES + sw128_offset(key, chunk & 7), vf);
              if (!all) {
                vf[0] &= keep[0];
                vf[1] &= keep[1];
                vf[2] &= keep[0];
                vf[3] &= keep[1];
              }
              mma16816(acc[d * 2], pf, vf[0], vf[1]);
              mma16816(acc[d * 2 + 1], pf, vf[2], vf[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + 8 * s);
      }
    }
    it += total;
  }

  // the warps' partial results meet in shared memory
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
  }
  if (__syncthreads_or(!ok)) {
    // a wait ran out: leave the results alone, give this CTA's own copies time to land
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
    return;
  }
  float* s_acc = (float*)smem;   // [warp][16][128]
  if (warp < 8) {
    float* mine = s_acc + warp * 16 * HD;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      *reinterpret_cast<float2*>(mine + g * HD + e * 8 + t4 * 2) = make_float2(acc[e][0], acc[e][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * HD + e * 8 + t4 * 2) = make_float2(acc[e][2], acc[e][3]);
    }
    if (t4 == 0) {
      s_ml[warp * 16 + g] = m[0];
      s_ml[warp * 16 + g + 8] = m[1];
      s_ml[128 + warp * 16 + g] = l[0];
      s_ml[128 + warp * 16 + g + 8] = l[1];
    }
  }
  __syncthreads();
  for (int i = tid; i < 16 * WR * (HD / 4); i += THREADS) {
    const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
    const int row = row0 + r;
    if (row >= rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; ++k) top = fmaxf(top, s_ml[(k * WR + r / 16) * 16 + r % 16]);
    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    const float ref = top > -INFINITY ? top : 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int w = k * WR + r / 16;
      const float f = score::exp2_approx(s_ml[w * 16 + r % 16] - ref);   // (-inf: 0; times NaN sums: NaN)
      sum += f * s_ml[128 + w * 16 + r % 16];
      const float4 a = *reinterpret_cast<const float4*>(s_acc + (w * 16 + r % 16) * HD + c);
      v[0] += f * a.x;
      v[1] += f * a.y;
      v[2] += f * a.z;
      v[3] += f * a.w;
    }
    const long long out_row = (long long)(row / G) * p.Hq + kvh * G + row % G;
    if (p.splits == 1) {
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= inv;
      store_row4(p, kvh, G, row, c, v);
      if (c == 0) p.lse[(long long)(kvh * G + row % G) * p.ld_lse + row / G] = lse_of(ref, sum);
    } else {
      const long long at = (long long)split * p.nq * p.Hq + out_row;
      *reinterpret_cast<float4*>(p.part_o + at * HD + c) = make_float4(v[0], v[1], v[2], v[3]);
      if (c == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(top, sum);
    }
  }
}

// ---------------------------------------------------------------------------
// The same for more packed rows (and group sizes that divide 128): tcgen05 products on a 128-row tile
// ---------------------------------------------------------------------------
// One CTA owns 128 packed rows of a KV head and one split of the keys. Its tiles alternate between two softmax
// pipelines of eight warps (two threads per row, 64 keys each) with their own scores and accumulator in TMEM, so that the
// exponentials of one tile overlap the products of the next; the two accumulators are joined at the end like two splits.
//   warps 0-15 softmax, warp 16 TMA (Q once: a 3-D box of 128 / G rows x G heads lands as packed rows; K and V, three
//   stages), warp 17 issues the MMAs.  TMEM: S0 [0,128) S1 [128,256) O0 [256,384) O1 [384,512), P over S as bf16.
// Tiles that every row sees whole skip the mask; in the others, V rows of keys that none of the CTA's rows sees are overwritten
// with zeros. The bounds' hull also holds unused cache slots between two sequences, so that takes the rows' own masks: each
// softmax warp leaves the OR over its rows, and warp 17, which has registers to spare, clears before it issues P V.
namespace fewt {

constexpr int KID = 13;
constexpr int STAGES = 3;
constexpr int THREADS = 576;
constexpr int OFF_STAGE = TILE_BYTES;                             // behind Q
constexpr int OFF_X = OFF_STAGE + STAGES * 2 * TILE_BYTES;        // row exchange [pipeline][half][128]
constexpr int OFF_BITS = OFF_X + 2048;                            // visible tiles, then fully visible tiles
constexpr int OFF_BOUND = OFF_BITS + 2 * ROUND / 8;
constexpr int OFF_BARS = OFF_BOUND + 32;
constexpr int OFF_SEEN = OFF_BARS + 256;                          // keys seen: [softmax warp][its 64 keys]
// no alignment slack: the kernel checks that its dynamic shared memory starts 1 KiB aligned
constexpr int SMEM_BYTES = OFF_SEEN + 2 * 4 * 16;
static_assert(SMEM_BYTES <= 232448, "shared memory budget of one CTA");

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// walks the set bits of a bit map in order
struct Walk {
  const uint32_t* words;
  int w;
  uint32_t bits;
  __device__ __forceinline__ explicit Walk(const uint32_t* b) : words(b), w(0), bits(b[0]) {}
  __device__ __forceinline__ int next() {   // only called while bits are left
    while (!bits) bits = words[++w];
    const int o = w * 32 + __ffs(bits) - 1;
    bits &= bits - 1;
    return o;
  }
};

template <int MOD>
__global__ void __launch_bounds__(THREADS, 1)
few_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {   // swizzled tiles need 1 KiB alignment; nothing has been set up yet
    if (threadIdx.x == 0) set_error(ERR_BAD_INDEX, KID, 1);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + OFF_STAGE;   // [stage][K | V]
  float* sX = (float*)(smem + OFF_X);
  uint32_t* s_vis = (uint32_t*)(smem + OFF_BITS);
  uint32_t* s_full = s_vis + ROUND / 32;
  Bounds* s_bound = (Bounds*)(smem + OFF_BOUND);
  const uint32_t b0 = smem_u32(smem + OFF_BARS);
  const uint32_t bar_q = b0, bar_kfull = b0 + 8, bar_vfull = b0 + 32, bar_empty = b0 + 56;   // [3] each
  const uint32_t bar_sfull = b0 + 80, bar_pfull = b0 + 96, bar_odone = b0 + 112;             // [2] each
  uint32_t* tmem_slot = (uint32_t*)(smem + OFF_BARS + 128);
  uint32_t* s_seen = (uint32_t*)(smem + OFF_SEEN);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.Hq / p.Hkv;
  const int kvh = blockIdx.x % p.Hkv;
  const int rt = (blockIdx.x / p.Hkv) % p.row_tiles;
  const int split = blockIdx.x / (p.Hkv * p.row_tiles);
  const int rows = p.nq * G;
  const int row0 = rt * 128;
  const int nkt = (p.nk + BK - 1) / BK;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int own = split < nkt ? (nkt - split + p.splits - 1) / p.splits : 0;   // at most ROUND (host)

  if (tid == 512) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // on their way while the barriers are set up: the codes of this warp's first tile and this thread's row's mask
  Codes first;
  if (warp < own) first.load(p, (split + warp * p.splits) * BK, lane);
  const int i1 = min((row0 + 127) / G, p.nq - 1), i_mine = row0 / G + tid;   // at most 128 query rows
  int mask_of[3] = {0, 0, 0};
  if (i_mine <= i1) {
    mask_of[0] = p.q_lo[i_mine];
    mask_of[1] = p.q_hi[i_mine];
    mask_of[2] = p.q_grp[i_mine];
  }
  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_kfull + 8 * s, 1);
      mbar_init(bar_vfull + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_pfull + 8 * s, 256);
      mbar_init(bar_odone + 8 * s, 1);
    }
    fence_mbar_init();
    s_bound->clear();
  }
  if (warp == 17) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  for (int i = tid; i < 2 * ROUND / 32; i += THREADS) s_vis[i] = 0u;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (i_mine <= i1) s_bound->add(mask_of[0], mask_of[1], mask_of[2]);
  if (warp == 16 && lane == 0) {   // Q is needed in any case (if no tile is visible, it still has to land before the end)
    mbar_expect_tx(bar_q, TILE_BYTES);
#pragma unroll
    for (int c = 0; c < 2; ++c) tma_load_3d(smem_u32(sQ + c * HALF_BYTES), &tm_q, bar_q, c * 64, kvh * G, row0 / G);
  }
  __syncthreads();
  {
    const Bounds bounds = *s_bound;
    for (int o = warp; o < own; o += THREADS / 32) {
      if (o != warp) first.load(p, (split + o * p.splits) * BK, lane);
      bool any = false, all = true;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        any |= bounds.may_see(first.c[e]);
        all &= bounds.all_see(first.c[e]);
      }
      any = __any_sync(0xffffffffu, any);
      all = __all_sync(0xffffffffu, all);
      if (lane == 0 && any) atomicOr(s_vis + (o >> 5), 1u << (o & 31));
      if (lane == 0 && all) atomicOr(s_full + (o >> 5), 1u << (o & 31));
    }
  }
  __syncthreads();
  int n = 0;
  for (int i = 0; i < (own + 31) / 32; ++i) n += __popc(s_vis[i]);

  if (warp == 16) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0 && n == 0) mbar_wait(bar_q, 0, KID, 11);
    if (lane == 0 && n > 0) {
      Walk walk(s_vis);
      for (int j = 0; j < n; ++j) {
        const int s = j % STAGES;
        const int k0 = (split + walk.next() * p.splits) * BK;
        const uint32_t dst = smem_u32(sKV + s * 2 * TILE_BYTES);
        if (!mbar_wait_spin(bar_empty + 8 * s, ((j / STAGES) & 1) ^ 1, KID, 10)) break;
        mbar_expect_tx(bar_kfull + 8 * s, TILE_BYTES);
#pragma unroll
        for (int c = 0; c < 2; ++c) tma_load_2d(dst + c * HALF_BYTES, &tm_k, bar_kfull + 8 * s, kvh * HD + c * 64, k0);
        mbar_expect_tx(bar_vfull + 8 * s, TILE_BYTES);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          tma_load_2d(dst + TILE_BYTES + c * HALF_BYTES, &tm_v, bar_vfull + 8 * s, kvh * HD + c * 64, k0);
      }
    }
  } else if (warp == 17) {
    // ------------------------------ MMA issuer (whole warp, one elected lane issues) ----
    if (n > 0) {
      const bool leader = elect_one();
      const uint32_t idesc_qk = make_idesc_bf16(128, BK, 0, 0);
      const uint32_t idesc_pv = make_idesc_bf16(128, HD, 0, 1);
      auto wait_all = [&](uint32_t bar, uint32_t parity, int detail) {
        return __all_sync(0xffffffffu, mbar_wait_spin(bar, parity, KID, detail));
      };
      auto issue_qk = [&](int j) {   // scores of tile j into pipeline j & 1
        const uint32_t qa = smem_u32(sQ), ka = smem_u32(sKV + (j % STAGES) * 2 * TILE_BYTES);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = (k >> 2) * HALF_BYTES + (k & 3) * 32;
          const uint64_t ad = make_smem_desc_sw128(qa + off, 16, 1024);
          const uint64_t bd = make_smem_desc_sw128(ka + off, 16, 1024);
          if (leader) tc_mma_ss(tmem_base + (j & 1) * 128, ad, bd, idesc_qk, k ? 1u : 0u);
        }
        if (leader) tc_commit(bar_sfull + 8 * (j & 1));
      };
      Walk walk(s_vis);
      bool ok = wait_all(bar_q, 0, 20);
      for (int j = 0; j < 2 && j < n && ok; ++j) {
        ok = wait_all(bar_kfull + 8 * j, 0, 21);
        if (ok) {
          tc_fence_after();
          issue_qk(j);
        }
      }
      for (int j = 0; j < n && ok; ++j) {
        const int i = j & 1, s = j % STAGES;
        const int o = walk.next();   // (before the waits, which it would lengthen)
        const bool masked = !((s_full[o >> 5] >> (o & 31)) & 1u);
        if (!wait_all(bar_vfull + 8 * s, (j / STAGES) & 1, 22)) break;
        if (!wait_all(bar_pfull + 8 * i, (j >> 1) & 1, 23)) break;
        tc_fence_after();
        if (masked) {   // V rows that no row of the CTA sees (behind the last key they are zeros)
          const uint4* seen = reinterpret_cast<const uint4*>(s_seen + i * 16);
          const uint4 a = seen[0], b = seen[1], c = seen[2], d = seen[3];   // two warps each: keys 0-63, then 64-127
          const uint32_t some[4] = {a.x | a.z | b.x | b.z, a.y | a.w | b.y | b.w, c.x | c.z | d.x | d.z, c.y | c.w | d.y | d.w};
          const int left = p.nk - (split + o * p.splits) * BK;
          bool any = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int key = w * 32 + lane;   // (pieces of a row in an order by key: no two lanes meet in a bank)
            if (((some[w] >> lane) & 1u) || key >= left) continue;
            any = true;
            uint8_t* vrow = sKV + s * 2 * TILE_BYTES + TILE_BYTES + key * 128;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              *reinterpret_cast<uint4*>(vrow + (e >> 3) * HALF_BYTES + ((e + lane) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          if (any) fence_proxy_async_smem();
          __syncwarp();
        }
        const uint32_t va = smem_u32(sKV + s * 2 * TILE_BYTES + TILE_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          const uint64_t bd = make_smem_desc_sw128(va + k * 2048, HALF_BYTES, 1024);
          if (leader) tc_mma_ts(tmem_base + 256 + i * 128, tmem_base + i * 128 + k * 8, bd, idesc_pv, (j > 1 || k) ? 1u : 0u);
        }
        if (leader) {
          tc_commit(bar_empty + 8 * s);
          if (j + 2 >= n) tc_commit(bar_odone + 8 * i);
        }
        if (j + 2 < n) {
          if (!wait_all(bar_kfull + 8 * ((j + 2) % STAGES), ((j + 2) / STAGES) & 1, 24)) break;
          tc_fence_after();
          issue_qk(j + 2);
        }
      }
      __syncwarp();
    }
  }
  // ------------------------------ softmax pipelines -------------------------------
  const int i = warp >> 3;          // pipeline
  const int sub = (warp >> 2) & 1;  // which 64 keys of a tile (and columns of the accumulator)
  const int qd = warp & 3;          // TMEM lane quarter
  const int row = qd * 32 + lane;
  const uint32_t t_s = tmem_base + ((uint32_t)(qd * 32) << 16) + i * 128;
  const uint32_t t_o = tmem_base + ((uint32_t)(qd * 32) << 16) + 256 + i * 128;
  float* xmine = sX + (i * 2 + sub) * 128 + row;
  const float* xother = sX + (i * 2 + (sub ^ 1)) * 128 + row;
  const float scl = (MOD & score::CAP) != 0 ? 1.f : p.scale_log2;   // capped scores already are in log2 units
  float m = -INFINITY, l = 0.f;
  bool ok = true;
  if (warp < 16) {
    const int prow = row0 + row;
    // (the row's mask is read where a tile needs it: held here it would push the scores out of registers)
    const int qi = prow < rows ? prow / G : -1;
    [[maybe_unused]] float slope = 0.f, qpos = 0.f;
    if (prow < rows) {
      if constexpr ((MOD & score::BIAS) != 0) {
        slope = p.slopes[kvh * G + prow % G] * 1.4426950408889634f / scl;
        qpos = score::position(p.q_pos[qi]);
      }
    }
    Walk walk(s_vis);
    uint32_t r[64];
    for (int j = 0; j < n; ++j) {
      const int o = walk.next();
      if ((j & 1) != i) continue;
      const int k0 = (split + o * p.splits) * BK + sub * 64;
      const bool masked = !((s_full[o >> 5] >> (o & 31)) & 1u);
      // positions of the 64 keys: two per lane, loaded while the scores are on their way, passed by shuffles
      [[maybe_unused]] float kpos[2] = {0.f, 0.f};
      if constexpr ((MOD & score::BIAS) != 0) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int k = k0 + x * 32 + lane;
          kpos[x] = k < p.nk ? score::position(__ldg(p.k_pos + k)) : 0.f;
        }
      }
      bool good = __all_sync(0xffffffffu, mbar_wait_spin(bar_sfull + 8 * i, (j >> 1) & 1, KID, 30));
      if (good) {
        tc_fence_after();
        tmem_ld32(t_s + sub * 64, r);
        tmem_ld32(t_s + sub * 64 + 32, r + 32);
        tmem_ld_wait();
        score::transform_row<MOD>(r, p.mod, slope, qpos, make_float2(kpos[0], kpos[1]), [&](int e) {
          const float kp = kpos[e >> 5];
          asm volatile("" ::: "memory");
          return make_float4(__shfl_sync(0xffffffffu, kp, e & 31), __shfl_sync(0xffffffffu, kp, (e + 1) & 31),
                             __shfl_sync(0xffffffffu, kp, (e + 2) & 31), __shfl_sync(0xffffffffu, kp, (e + 3) & 31));
        });
        if (masked) {
          // (a bit per key first, in a loop that holds one code at a time: the scores keep their registers)
          const score::RowMask mask(qi < 0 ? 0 : __ldg(p.q_lo + qi), qi < 0 ? 0 : __ldg(p.q_hi + qi), qi < 0 ? 0 : __ldg(p.q_grp + qi));
          uint32_t hidden[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int k = k0 + x * 32 + lane;
            const int code = k < p.nk ? __ldg(p.k_code + k) : score::DEAD_KEY;
            uint32_t h = 0u;
#pragma unroll 4
            for (int e = 0; e < 32; ++e) h |= (uint32_t)!mask.sees(__shfl_sync(0xffffffffu, code, e)) << e;
            hidden[x] = h;
          }
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if ((hidden[e >> 5] >> (e & 31)) & 1u) r[e] = 0xff800000u;   // -inf
          {
            const uint32_t s0 = ~__reduce_and_sync(0xffffffffu, hidden[0]), s1 = ~__reduce_and_sync(0xffffffffu, hidden[1]);
            if (lane == 0) *reinterpret_cast<uint2*>(s_seen + warp * 2) = make_uint2(s0, s1);
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 64; e += 2) mx = score::max3(mx, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
        *xmine = mx;
      }
      // the barrier also orders the P stores below after the partner's loads of its score columns
      if (!named_bar_all(1 + i, 256, good)) { ok = false; break; }
      const float mx = fmaxf(*xmine, *xother);
      float alpha = 1.f;   // the reference maximum moves only when the new one is 2^8 larger
      if (mx > -INFINITY && (m == -INFINITY || (mx - m) * scl > 8.f)) {
        alpha = m == -INFINITY ? 0.f : score::exp2_approx((m - mx) * scl);
        m = mx;
      }
      l *= alpha;
      if (__any_sync(0xffffffffu, alpha != 1.f) && j > 1) {
        uint32_t ro[16];
#pragma unroll 1
        for (int c = 4 * sub; c < 4 * sub + 4; ++c) {   // this thread's half of the accumulator columns
          tmem_ld16(t_o + c * 16, ro);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) ro[e] = __float_as_uint(__uint_as_float(ro[e]) * alpha);
          tmem_st16(t_o + c * 16, ro);
        }
      }
      const float ref = m == -INFINITY ? 0.f : m * scl;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = score::exp2_approx(fmaf(__uint_as_float(r[c * 16 + e]), scl, -ref));
          const float p1 = score::exp2_approx(fmaf(__uint_as_float(r[c * 16 + e + 1]), scl, -ref));
          l += p0 + p1;
          pk[e >> 1] = pack_bf16x2(p0, p1);
        }
        tmem_st8(t_s + sub * 32 + c * 8, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar_pfull + 8 * i);
      // (the exchange slots are rewritten only after this tile's products, which wait for all 256 arrivals above)
    }
    m *= scl;   // (log2 units from here on)
    if (ok && n > i) ok = mbar_wait_spin(bar_odone + 8 * i, 0, KID, 31);
  }
  // ------------------------------ joining the two pipelines ------------------------
  bool good = !__syncthreads_or(!ok || error_is_set());   // all products done, all tiles consumed: the stages are free
  float* s_acc = (float*)sKV;      // [128 rows][128 columns] fp32, 16-byte chunks swizzled by row
  float* s_ml = sX;                // [m1 | l1 of both halves]
  tc_fence_after();
  auto chunk_at = [&](int rr, int c) { return s_acc + rr * HD + ((c ^ (rr & 31)) << 2); };   // c: 16-byte chunk 0..31
  if (good && warp < 16 && i == 1) {
    uint32_t ro[32];
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      if (n > 1) {
        tmem_ld32(t_o + sub * 64 + h * 32, ro);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) ro[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        *reinterpret_cast<uint4*>(chunk_at(row, sub * 16 + h * 8 + e)) = make_uint4(ro[4 * e], ro[4 * e + 1], ro[4 * e + 2], ro[4 * e + 3]);
    }
    s_ml[256 + sub * 128 + row] = l;
    if (sub == 0) s_ml[row] = m;   // (pipeline 0's slots: its own exchange is over)
  }
  float m1 = -INFINITY, l1 = 0.f;
  __syncthreads();
  if (good && warp < 16 && i == 0) {
    m1 = s_ml[row];
    l1 = s_ml[256 + row] + s_ml[384 + row];
  }
  __syncthreads();
  if (good && warp < 16 && i == 0) s_ml[sub * 128 + row] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  if (good && warp < 16 && i == 0) {
    const float l0 = s_ml[row] + s_ml[128 + row];
    top = fmaxf(m, m1);
    const float f0 = m == -INFINITY ? 0.f : score::exp2_approx(m - top), f1 = m1 == -INFINITY ? 0.f : score::exp2_approx(m1 - top);
    sum = f0 * l0 + f1 * l1;
    const float norm = p.splits == 1 ? (sum > 0.f ? 1.f / sum : 0.f) : 1.f;
    const float g0 = f0 * norm, g1 = f1 * norm;
    uint32_t ro[32];
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      if (n > 0) {
        tmem_ld32(t_o + sub * 64 + h * 32, ro);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) ro[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float4* at = reinterpret_cast<float4*>(chunk_at(row, sub * 16 + h * 8 + e));
        float4 b = *at;
        b.x = fmaf(g0, __uint_as_float(ro[4 * e]), g1 * b.x);
        b.y = fmaf(g0, __uint_as_float(ro[4 * e + 1]), g1 * b.y);
        b.z = fmaf(g0, __uint_as_float(ro[4 * e + 2]), g1 * b.z);
        b.w = fmaf(g0, __uint_as_float(ro[4 * e + 3]), g1 * b.w);
        *at = b;
      }
    }
  }
  __syncthreads();
  if (good) {
    // whole rows go out 512 (256) bytes at a time
    for (int x = tid; x < 128 * (HD / 4); x += THREADS) {
      const int rr = x / (HD / 4), c = x % (HD / 4), prow = row0 + rr;
      if (prow >= rows) break;
      const float4 v = *reinterpret_cast<const float4*>(chunk_at(rr, c));
      if (p.splits == 1) {
        const float o4[4] = {v.x, v.y, v.z, v.w};
        store_row4(p, kvh, G, prow, c * 4, o4);
      } else {
        const long long at = ((long long)split * p.nq + prow / G) * p.Hq + kvh * G + prow % G;
        *reinterpret_cast<float4*>(p.part_o + at * HD + c * 4) = v;
      }
    }
    if (warp < 8 && sub == 0 && row0 + row < rows) {
      const int prow = row0 + row, qi = prow / G, h = kvh * G + prow % G;
      if (p.splits == 1)
        p.lse[(long long)h * p.ld_lse + qi] = lse_of(top, sum);
      else
        *reinterpret_cast<float2*>(p.part_ml + (((long long)split * p.nq + qi) * p.Hq + h) * 2) = make_float2(top, sum);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (error_is_set()) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 17) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int MOD>
static cudaError_t launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, cudaStream_t st) {
  static bool attr_set[64] = {false};   // a function attribute belongs to one device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(few_tiles_kernel<MOD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  few_tiles_kernel<MOD><<<p.Hkv * p.row_tiles * p.splits, THREADS, SMEM_BYTES, st>>>(tq, tk, tv, p);
  return cudaGetLastError();
}

}  // namespace fewt

// Joins the splits of a (query row, head), W warps to each. Launched while the splits still run; the dependency wait returns
// when that grid has ended and its results are visible. The sums run in a fixed order.
// Four warps to a row when there are more than 8 splits, whose loads one warp would take in several rounds (one token
// against 20000 keys, 18 splits: 17.9 us for both kernels against 18.8; 8 rows against 4000: 14.2 against 16.2), else one, and
// few blocks (128 rows against 1024 keys, 4 splits: 14.8 us against 19.7 with four warps to a row). Blocks of 256 threads cost
// another 1 us.
constexpr int JOIN_WARPS_FROM = 9;
constexpr int JOIN_THREADS = 128;
template <int W>
__global__ void __launch_bounds__(JOIN_THREADS) few_rows_join_kernel(const Params p) {
  constexpr int ROWS = JOIN_THREADS / 32 / W;
  __shared__ float4 s_v[W > 1 ? JOIN_THREADS : 1];
  __shared__ float s_sum[JOIN_THREADS / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n = (long long)p.nq * p.Hq;
  const long long mine = (long long)blockIdx.x * ROWS + warp / W, at = min(mine, n - 1);
  if (W == 1 && mine >= n) return;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, p.part_ml[(s * n + at) * 2]);
  top = warp_max(top);
  const float ref = top > -INFINITY ? top : 0.f;
  float sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = warp % W; s < p.splits; s += W) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * n + at) * 2);
    const float4 a = *reinterpret_cast<const float4*>(p.part_o + (s * n + at) * HD + lane * 4);
    const float f = score::exp2_approx(ml.x - ref);
    sum += f * ml.y;
    v.x += f * a.x;
    v.y += f * a.y;
    v.z += f * a.z;
    v.w += f * a.w;
  }
  if constexpr (W > 1) {
    s_v[threadIdx.x] = v;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp % W || mine >= n) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 a = s_v[threadIdx.x + w * 32];
      v.x += a.x;
      v.y += a.y;
      v.z += a.z;
      v.w += a.w;
      sum += s_sum[warp + w];
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  const int i = (int)(at / p.Hq), h = (int)(at % p.Hq);
  uint2 w;
  w.x = pack_bf16x2(v.x * inv, v.y * inv);
  w.y = pack_bf16x2(v.z * inv, v.w * inv);
  *reinterpret_cast<uint2*>(p.o + (long long)i * p.ldo + h * HD + lane * 4) = w;
  if (lane == 0) p.lse[(long long)h * p.ld_lse + i] = lse_of(ref, sum);
}

struct Plan {
  int wr, row_tiles, splits;
  bool tiles;   // tcgen05 on 128-row tiles
};
// Packed rows of a KV head from which the tcgen05 form is taken. B200, 8 KV heads of 4 query heads, capped, us (mma form against
// tcgen05 form): 64 rows x 2048 keys 15.6 / 12.8, 64 x 32768 65 / 35, 128 x 300 19.9 / 14.5, 128 x 2048 21.9 / 14.7,
// 128 x 32768 114 / 38; up to 32 rows the tcgen05 form computes at least four times what is asked for.
constexpr int TILE_ROWS_FROM = 33;
static Plan plan_of(int nq, int nk, int Hq, int Hkv) {
  Plan pl;
  const int rows = nq * (Hq / Hkv);
  pl.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8;
  pl.tiles = rows >= TILE_ROWS_FROM && 128 % (Hq / Hkv) == 0;
  if (pl.tiles) pl.wr = 8;
  pl.row_tiles = (rows + 16 * pl.wr - 1) / (16 * pl.wr);
  const int nkt = (nk + BK - 1) / BK;
  int s = tdllm_num_sms() / (Hkv * pl.row_tiles);
  if (s > nkt) s = nkt;
  if (s < 1) s = 1;
  if (pl.tiles && s < (nkt + ROUND - 1) / ROUND) s = (nkt + ROUND - 1) / ROUND;   // one visibility round per CTA
  pl.splits = s;
  return pl;
}

template <int WR, int MOD>
static cudaError_t launch(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, cudaStream_t st) {
  static bool attr_set[64] = {false};   // a function attribute belongs to one device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<WR, MOD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  few_rows_kernel<WR, MOD><<<p.Hkv * p.row_tiles * p.splits, THREADS, SMEM_BYTES, st>>>(tk, tv, p);
  return cudaGetLastError();
}
template <int MOD>
static cudaError_t launch_wr(int wr, const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, cudaStream_t st) {
  switch (wr) {
    case 1: return launch<1, MOD>(tk, tv, p, st);
    case 2: return launch<2, MOD>(tk, tv, p, st);
    case 4: return launch<4, MOD>(tk, tv, p, st);
    default: return launch<8, MOD>(tk, tv, p, st);
  }
}

}  // namespace few
}  // namespace tdllm

using namespace tdllm;

// floats of scratch that tdllm_attn_few_rows needs (0: the keys are not split)
extern "C" long long tdllm_attn_few_rows_scratch(int nq, int nk, int Hq, int Hkv) {
  if (nq <= 0 || nk <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv) return 0;
  const few::Plan pl = few::plan_of(nq, nk, Hq, Hkv);
  return pl.splits > 1 ? (long long)pl.splits * nq * Hq * (few::HD + 2) : 0;
}

// q [nq, Hq*128], k / v [nk, Hkv*128], o [nq, Hq*128] (row strides in elements), lse [Hq][ld_lse]. The mask's arrays are
// the layout's own (nothing padded, no tile lists); positions int32, slopes [Hq] (null: no bias).
extern "C" int tdllm_attn_few_rows(const void* q, const void* k, const void* v, void* o, float* lse, float* scratch,
                                   int nq, int nk, int Hq, int Hkv, long long ldq, long long ldk, long long ldv,
                                   long long ldo, long long ld_lse, const int* q_lo, const int* q_hi, const int* q_grp,
                                   const int* k_code, float scale, float softcap, const float* slopes, const int* q_pos,
                                   const int* k_pos, void* stream) {
  if (nq <= 0 || nk <= 0) return 0;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv) {
    tdllm_host::set_last_error("attn_few_rows: %d query heads do not divide over %d KV heads", Hq, Hkv);
    return 1;
  }
  const long long lds[4] = {ldq, ldk, ldv, ldo};
  const void* ptrs[4] = {q, k, v, o};
  for (int i = 0; i < 4; ++i)
    if ((lds[i] % 8) || ((uintptr_t)ptrs[i] % 16)) {
      tdllm_host::set_last_error("attn_few_rows: operand %d needs a 16-byte aligned base and row stride", i);
      return 1;
    }
  const few::Plan pl = few::plan_of(nq, nk, Hq, Hkv);
  CUtensorMap tk, tv;
  if (tdllm_host::encode_rows_tmap(&tk, k, (long long)Hkv * few::HD, nk, ldk, few::BK)) return 3;
  if (tdllm_host::encode_rows_tmap(&tv, v, (long long)Hkv * few::HD, nk, ldv, few::BK)) return 3;
  few::Params p;
  p.q = (const __nv_bfloat16*)q;
  p.o = (__nv_bfloat16*)o;
  p.lse = lse;
  p.part_o = scratch;
  p.part_ml = scratch ? scratch + (long long)pl.splits * nq * Hq * few::HD : nullptr;
  p.q_lo = q_lo; p.q_hi = q_hi; p.q_grp = q_grp; p.k_code = k_code; p.q_pos = q_pos; p.k_pos = k_pos;
  p.slopes = slopes;
  p.ldq = ldq; p.ldo = ldo; p.ld_lse = ld_lse;
  p.nq = nq; p.nk = nk; p.Hq = Hq; p.Hkv = Hkv; p.splits = pl.splits; p.row_tiles = pl.row_tiles;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mod = score_mod_of(scale, softcap, nullptr, nullptr, nullptr);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (pl.tiles) {
    const int G = Hq / Hkv;
    CUtensorMap tq;
    const uint64_t dims[3] = {(uint64_t)few::HD, (uint64_t)Hq, (uint64_t)nq};
    const uint64_t strides[2] = {(uint64_t)few::HD * 2, (uint64_t)ldq * 2};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)(128 / G)};
    if (tdllm_host::encode_tmap(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return 3;
    switch ((softcap > 0.f ? score::CAP : 0) | (slopes ? score::BIAS : 0)) {
      case 0: e = few::fewt::launch<0>(tq, tk, tv, p, st); break;
      case score::CAP: e = few::fewt::launch<score::CAP>(tq, tk, tv, p, st); break;
      case score::BIAS: e = few::fewt::launch<score::BIAS>(tq, tk, tv, p, st); break;
      default: e = few::fewt::launch<score::CAP | score::BIAS>(tq, tk, tv, p, st); break;
    }
  } else
  switch ((softcap > 0.f ? score::CAP : 0) | (slopes ? score::BIAS : 0)) {
    case 0: e = few::launch_wr<0>(pl.wr, tk, tv, p, st); break;
    case score::CAP: e = few::launch_wr<score::CAP>(pl.wr, tk, tv, p, st); break;
    case score::BIAS: e = few::launch_wr<score::BIAS>(pl.wr, tk, tv, p, st); break;
    default: e = few::launch_wr<score::CAP | score::BIAS>(pl.wr, tk, tv, p, st); break;
  }
  if (e == cudaSuccess && pl.splits > 1) {
    const long long n = (long long)nq * Hq;
    cudaLaunchConfig_t cfg = {};
    const bool many = pl.splits >= few::JOIN_WARPS_FROM;
    const int rows = few::JOIN_THREADS / 32 / (many ? 4 : 1);
    cfg.gridDim = dim3((unsigned)((n + rows - 1) / rows));
    cfg.blockDim = dim3(few::JOIN_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = many ? cudaLaunchKernelEx(&cfg, few::few_rows_join_kernel<4>, p)
             : cudaLaunchKernelEx(&cfg, few::few_rows_join_kernel<1>, p);
  }
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("attn_few_rows launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}
