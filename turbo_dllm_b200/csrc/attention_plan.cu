// Tile lists of a declarative mask, built on the device: which 128-key tiles each 128-row query tile has to visit
// (forward), and which query tiles of a chunk each key tile meets (backward). No host synchronisation and no size that
// only the device knows, so a plan can be built inside a captured graph.
//
// Rows that see no clean key get an empty interval behind every coordinate, so that they do not widen what their tile
// seems to see; keys that no row sees get the code DEAD_KEY. Per tile:
//   queries   lo_min, hi_max (rows with an interval), lo_max, hi_min (all rows), grp_min, grp_max (noisy rows)
//   keys      c_min, c_max (clean), n_min, n_max (noisy), all_clean
// A pair of tiles is visited if the clean or the noisy ranges meet, and needs no mask if every row's interval holds all
// of the keys. Lists are in tile order; `order` has the longest lists first (ties: lowest tile), so results and their
// launch order repeat. The work is a few comparisons per pair of tiles: the first pass on a new layout of 5000 rows takes
// 0.3 ms longer than the next one, most of it on the host (1.7 ms with lists built there).
#include "common.cuh"
#include "score_mod.cuh"
#include "api.h"

namespace tdllm {
namespace plan {

constexpr int TILE = 128;
constexpr int BIG = 2147483647;

struct QStat { int lo_min, hi_max, lo_max, hi_min, g_min, g_max; };
struct KStat { int c_min, c_max, n_min, n_max, all_clean, pad; };

struct Args {
  const int *q_lo, *q_hi, *q_grp, *k_code;   // the layout's own
  int nq, nk, nqt, nkt, chunk, nch;
  int *lo, *hi, *grp, *code;                 // padded to whole tiles
  QStat* qs;
  KStat* ks;
  int *f_ptr, *f_idx, *f_order;              // forward: [nqt + 1], [nqt * nkt], [nqt]
  int *w_ptr, *w_idx, *w_order;              // backward: items chunk * nkt + key tile; [items + 1], [nqt * nkt], [items]
  int *f_count, *w_count;
};

__device__ __forceinline__ int red_min(int v, int* sm) {
  for (int o = 16; o; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  return min(min(sm[0], sm[1]), min(sm[2], sm[3]));
}
__device__ __forceinline__ int red_max(int v, int* sm) { return ~red_min(~v, sm); }

// one block per query tile: padded copies and the tile's bounds
__global__ void __launch_bounds__(TILE) query_kernel(const Args a) {
  __shared__ int sm[4];
  const int at = blockIdx.x * TILE + threadIdx.x;
  const bool real = at < a.nq;
  int lo = real ? max(a.q_lo[at], 0) : 0, hi = real ? a.q_hi[at] : 0;
  const int grp = real ? a.q_grp[at] : 0;
  const bool sees = hi > lo;
  if (!sees) { lo = BIG; hi = 0; }
  a.lo[at] = lo;
  a.hi[at] = hi;
  a.grp[at] = grp;
  const int lo_min = red_min(sees ? lo : BIG, sm), hi_max = red_max(sees ? hi : -1, sm);
  const int lo_max = red_max(real ? lo : -BIG, sm), hi_min = red_min(real ? hi : BIG, sm);
  const int g_min = red_min(grp < 0 ? grp : 0, sm), g_max = red_max(grp < 0 ? grp : -BIG - 1, sm);
  if (threadIdx.x == 0) a.qs[blockIdx.x] = {lo_min, hi_max, lo_max, hi_min, g_min, g_max};
}

__device__ __forceinline__ bool meets(const QStat& q, const KStat& k) {
  return (k.c_min < q.hi_max && k.c_max >= q.lo_min) || (k.n_min <= q.g_max && k.n_max >= q.g_min);
}
__device__ __forceinline__ bool whole(const QStat& q, const KStat& k) {
  return k.all_clean && k.c_max < q.hi_min && k.c_min >= q.lo_max;
}

__device__ __forceinline__ KStat key_stat(int c, int* sm) {
  const bool clean = c >= 0, noisy = c < 0 && c != score::DEAD_KEY;
  KStat s;
  s.c_min = red_min(clean ? c : BIG, sm);
  s.c_max = red_max(clean ? c : -1, sm);
  s.n_min = red_min(noisy ? c : 0, sm);
  s.n_max = red_max(noisy ? c : -BIG - 1, sm);
  s.all_clean = red_min(clean ? 1 : 0, sm);
  s.pad = 0;
  return s;
}

// one block per key tile: the codes, those of keys that no row sees replaced by DEAD_KEY, and the tile's bounds. The rows of
// the query tiles that may see the tile are tried until every key has been seen (mostly in the first tile).
__global__ void __launch_bounds__(TILE) key_kernel(const Args a) {
  __shared__ int sm[4];
  __shared__ int4 rows[TILE];
  const int t = threadIdx.x, at = blockIdx.x * TILE + t;
  const int c = at < a.nk ? a.k_code[at] : score::DEAD_KEY;
  const KStat all = key_stat(c, sm);
  bool seen = false;
  for (int q = 0; q < a.nqt; ++q) {
    if (!meets(a.qs[q], all)) continue;
    if (__syncthreads_and(seen || c == score::DEAD_KEY)) break;
    rows[t] = make_int4(a.lo[q * TILE + t], a.hi[q * TILE + t], a.grp[q * TILE + t], 0);
    __syncthreads();
    for (int e = 0; e < TILE && !seen; ++e) {
      const int4 r = rows[e];
      seen = c >= 0 ? c >= r.x && c < r.y : c == r.z;
    }
  }
  const int code = seen ? c : score::DEAD_KEY;
  a.code[at] = code;
  const KStat s = key_stat(code, sm);
  if (t == 0) a.ks[blockIdx.x] = s;
}

// one warp per list, forward lists first: FILL false counts, FILL true writes the entries (tile * 2 + needs a mask)
template <bool FILL>
__global__ void __launch_bounds__(256) list_kernel(const Args a) {
  const int lane = threadIdx.x & 31;
  const int list = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int items = a.nch * a.nkt;
  if (list >= a.nqt + items) return;
  const bool forward = list < a.nqt;
  const int it = forward ? list : list - a.nqt;
  const int fixed = forward ? it : it % a.nkt;                       // the list's own tile
  const int from = forward ? 0 : (it / a.nkt) * a.chunk;             // the tiles it walks
  const int to = forward ? a.nkt : min(from + a.chunk, a.nqt);
  int* out = FILL ? (forward ? a.f_idx + a.f_ptr[it] : a.w_idx + a.w_ptr[it]) : nullptr;
  int n = 0;
  for (int base = from; base < to; base += 32) {
    const int t = base + lane;
    bool hit = false, full = false;
    if (t < to) {
      const QStat q = a.qs[forward ? fixed : t];
      const KStat k = a.ks[forward ? t : fixed];
      hit = meets(q, k);
      full = whole(q, k);
    }
    const unsigned m = __ballot_sync(0xffffffffu, hit);
    if (FILL && hit) out[n + __popc(m & ((1u << lane) - 1u))] = t * 2 + (full ? 0 : 1);
    n += __popc(m);
  }
  if (!FILL && lane == 0) (forward ? a.f_count : a.w_count)[it] = n;
}

// block 0 sums the forward counts, block 1 the backward ones (a running sum over pieces of 1024)
__global__ void __launch_bounds__(1024) scan_kernel(const Args a) {
  __shared__ int sm[32];
  const int n = blockIdx.x ? a.nch * a.nkt : a.nqt;
  const int* count = blockIdx.x ? a.w_count : a.f_count;
  int* ptr = blockIdx.x ? a.w_ptr : a.f_ptr;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int base = 0; base < n; base += 1024) {
    const int i = base + threadIdx.x;
    const int c = i < n ? count[i] : 0;
    int v = c;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = v;
    __syncthreads();
    if (warp == 0) {
      int w = sm[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
      }
      sm[lane] = w;
    }
    __syncthreads();
    const int upto = before + v + (warp ? sm[warp - 1] : 0);
    if (i < n) ptr[i] = upto - c;
    before += sm[31];
  }
  if (threadIdx.x == 0) ptr[n] = before;
}

// a list's place: how many lists of its group are longer, or as long and earlier. Groups: all forward lists; the key tiles
// of one chunk of 64 query tiles or more, whose dQ rows then stay in L2; all items of shorter chunks, which are there to
// fill the GPU (2000 rows, 16 / 8 heads, chunks of 6 tiles, forward and backward: 155 us against 166 chunk by chunk)
__global__ void __launch_bounds__(256) order_kernel(const Args a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int items = a.nch * a.nkt;
  if (i >= a.nqt + items) return;
  const bool forward = i < a.nqt;
  const int it = forward ? i : i - a.nqt;
  const bool by_chunk = a.chunk >= 64;
  const int group = forward || !by_chunk ? 0 : it / a.nkt * a.nkt, size = forward ? a.nqt : by_chunk ? a.nkt : items;
  const int* count = (forward ? a.f_count : a.w_count) + group;
  const int me = it - group, mine = count[me];
  int place = 0;
  for (int j = 0; j < size; ++j) place += count[j] > mine || (count[j] == mine && j < me);
  (forward ? a.f_order : a.w_order)[group + place] = it;
}

}  // namespace plan
}  // namespace tdllm

using namespace tdllm;

// ints of the buffer that tdllm_attn_plan fills, and where its parts begin (offsets[11]: lo, hi, grp, code, f_ptr, f_idx,
// f_order, w_ptr, w_idx, w_order, then the end of what the kernels read); -1: too many tiles for 32-bit entries
extern "C" long long tdllm_attn_plan_size(int nq, int nk, int chunk, long long* offsets) {
  const long long nqt = (nq + 127) / 128, nkt = (nk + 127) / 128, nch = (nqt + chunk - 1) / chunk, items = nch * nkt;
  if (nq <= 0 || nk <= 0 || chunk <= 0 || nqt * nkt >= (1LL << 30)) return -1;
  const long long part[10] = {nqt * 128, nqt * 128, nqt * 128, nkt * 128, nqt + 1, nqt * nkt, nqt, items + 1, nqt * nkt, items};
  long long at = 0;
  for (int i = 0; i < 10; ++i) {
    offsets[i] = at;
    at += (part[i] + 63) / 64 * 64;   // parts begin on 256 bytes
  }
  offsets[10] = at;
  return at + (nqt * 6 + 63) / 64 * 64 + (nkt * 6 + 63) / 64 * 64 + (nqt + 63) / 64 * 64 + (items + 63) / 64 * 64;
}

extern "C" int tdllm_attn_plan(const int* q_lo, const int* q_hi, const int* q_grp, const int* k_code, int nq, int nk,
                               int chunk, int* buf, void* stream) {
  long long off[11];
  if (tdllm_attn_plan_size(nq, nk, chunk, off) < 0) {
    tdllm_host::set_last_error("attn_plan: %d rows x %d keys have too many tiles", nq, nk);
    return 1;
  }
  plan::Args a;
  a.q_lo = q_lo; a.q_hi = q_hi; a.q_grp = q_grp; a.k_code = k_code;
  a.nq = nq; a.nk = nk;
  a.nqt = (nq + 127) / 128;
  a.nkt = (nk + 127) / 128;
  a.chunk = chunk;
  a.nch = (a.nqt + chunk - 1) / chunk;
  a.lo = buf + off[0]; a.hi = buf + off[1]; a.grp = buf + off[2]; a.code = buf + off[3];
  a.f_ptr = buf + off[4]; a.f_idx = buf + off[5]; a.f_order = buf + off[6];
  a.w_ptr = buf + off[7]; a.w_idx = buf + off[8]; a.w_order = buf + off[9];
  int* work = buf + off[10];
  a.qs = (plan::QStat*)work;
  work += (a.nqt * 6 + 63) / 64 * 64;
  a.ks = (plan::KStat*)work;
  work += (a.nkt * 6 + 63) / 64 * 64;
  a.f_count = work;
  a.w_count = work + (a.nqt + 63) / 64 * 64;
  cudaStream_t st = (cudaStream_t)stream;
  const int lists = a.nqt + a.nch * a.nkt;
  plan::query_kernel<<<a.nqt, 128, 0, st>>>(a);
  plan::key_kernel<<<a.nkt, 128, 0, st>>>(a);
  plan::list_kernel<false><<<(lists + 7) / 8, 256, 0, st>>>(a);
  plan::scan_kernel<<<2, 1024, 0, st>>>(a);
  plan::list_kernel<true><<<(lists + 7) / 8, 256, 0, st>>>(a);
  plan::order_kernel<<<(lists + 255) / 256, 256, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    tdllm_host::set_last_error("attn_plan launch: %s", cudaGetErrorString(e));
    return 4;
  }
  return 0;
}
