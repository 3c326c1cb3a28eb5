// Eviction from the paged int4 / k8v4 cache by the weight that its keys have received: per sequence and KV head the first
// `sinks` and last `recent` positions and, of the others, those of largest weight (the lowest position first among equal
// ones), `budget` in all; their cells go to new blocks in the order of their positions, with their weights.
//
// Weights are compared as integers of the same order. A workgroup per (sequence, KV head) finds the smallest weight that
// stays from three histograms in LDS, of the integers' upper 11, next 11 and last 10 bits, and counts what stays in each run
// of kRun positions; then a workgroup per run lists its survivors and moves their cells. Nothing is sorted, every cell is read
// and written once, and all counts are integers, so nothing depends on an order of atomics. Contexts of more than kDirect
// positions are too much for one workgroup per head: there the first histogram is made by many, which then put the weights of
// the bin that the threshold lies in, a few per cent, into lists, and only those are looked at by the one.
//
// What bounds it, measured: 16384 of 131072 positions of 4 heads of 256 (int4) take 5.3 us for the histogram, 9 for the
// lists, 8.8 for the threshold, 15 for the cells (35 MB at 2.3 TB/s): four launches, each a chain of few dependent loads.
// With more to move the cells' share grows: 16 contexts of up to 16384, 2048 kept, 8 heads of 128, int8 keys: 36 of 60 us, at
// 2.9 TB/s.
#include "qp_common.h"
#include "quantpack_ops.h"

namespace qp {

struct EvictParams {
  const uint8_t *kcodes;
  int64_t ks0, ks1, ks2;  // bytes
  const uint32_t *kwords;
  int64_t kws0, kws1, kws2;
  const uint8_t *vcodes;
  int64_t vs0, vs1, vs2;
  const uint32_t *vwords;
  int64_t vws0, vws1, vws2;
  const float *weights;
  int64_t w0, w1;
  const int32_t *used, *table, *new_table;
  int64_t table_stride, new_stride;
  int32_t *kept;
  int64_t k0, k1;
  float *new_weights;
  int64_t nw0, nw1;
  int32_t *new_used;
  uint2 *threshold;       // [sequence, KV head]: the smallest weight's integer, and how many of that weight stay
  int2 *base;             // [sequence, KV head, run]: survivors above the threshold, and weights at it, before the run
  uint32_t *hist;         // long contexts: [sequence, KV head, part, kBins],
  uint2 *lists;           // [sequence, KV head, part, kPart]: weights in the threshold's bin, and their runs,
  int *list_len;          // [sequence, KV head, part]
  int32_t num_blocks, block_size, num_kv_heads, max_keys, new_blocks, budget, sinks, recent, runs, parts;
  uint32_t bs_magic, bs_shift;
  int32_t key_units, value_units, cell_units;  // of the copies: 4 bytes, or 8 in whole cells
  uint32_t cell_magic, cell_shift;
};

constexpr int kRun = 256;            // positions of a run
// Positions that one workgroup takes alone, kPer in each thread's registers. A workgroup alone against the long path, us, 8
// heads of 128, a quarter kept: 4096 positions 15 / 22, 8192 20 / 24, 64 sequences of 8192 121 / 135.
constexpr int kDirect = 8192;
constexpr int kSelectThreads = 512;
constexpr int kPer = kDirect / kSelectThreads;
constexpr int kPart = 8192;          // positions of a workgroup of the long path
constexpr int kPartThreads = 1024;
constexpr int kPartPer = kPart / kPartThreads;
constexpr int kBins = 2048;
constexpr int kFirstShift = 21;      // the upper 11 bits

// An integer in the order of the weights; NaN below all others, -0 as 0.
__device__ __forceinline__ uint32_t weight_order(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// The positions [lo, hi) that are not kept in any case; all of them where everything stays (hi = lo: nothing to choose).
__device__ __forceinline__ void evict_range(const EvictParams &p, int n, int &lo, int &hi) {
  lo = min(p.sinks, n);
  hi = max(lo, n - p.recent);
}

__device__ __forceinline__ int evict_len(const EvictParams &p, int seq) { return max(0, min(p.used[seq], p.max_keys)); }

// The sum of v over the threads before this one (exclusive), and over all of them. sums: a word per wave in LDS.
template <int THREADS>
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t *sums, uint32_t &total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sums[w] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    const uint32_t y = sums[i];
    before += i < w ? y : 0;
    total += y;
  }
  return before + x - v;
}

// Adds one to bin `bin` of hist for every lane that is `in`. Equal weights would queue up at one counter: lanes that share
// the first one's bin add once.
__device__ __forceinline__ void count_bin(uint32_t *hist, uint32_t bin, bool in) {
  const uint64_t some = __ballot(in);
  if (!some) return;
  const int leader = (int)__builtin_ctzll(some);
  const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, leader);
  const uint64_t same = __ballot(in && bin == first);
  if (in && bin != first) atomicAdd(&hist[bin], 1u);
  if ((int)(threadIdx.x & 63) == leader) atomicAdd(&hist[first], (uint32_t)__builtin_popcountll(same));
}

// The bin in which the need-th entry from the top lies, and its number in there. counts(i): the entries of bin i.
template <int THREADS, int BINS, class Counts>
__device__ __forceinline__ uint32_t find_bin(const Counts &counts, uint32_t &need, uint32_t *sums, uint32_t *found) {
  constexpr int kEach = BINS / THREADS;
  uint32_t mine[kEach], all = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    mine[i] = counts(BINS - 1 - (kEach * (int)threadIdx.x + i));
    all += mine[i];
  }
  uint32_t above = block_before<THREADS>(all, sums, total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (above < need && need <= above + mine[i]) {
      found[0] = (uint32_t)(BINS - 1 - (kEach * (int)threadIdx.x + i));
      found[1] = need - above;
    }
    above += mine[i];
  }
  __syncthreads();
  need = found[1];
  return found[0];
}

// Of n keys' unprotected positions [lo, hi), how many stay; 0 also where everything does (`all`).
__device__ __forceinline__ uint32_t evict_need(const EvictParams &p, int n, int &lo, int &hi, bool &all) {
  evict_range(p, n, lo, hi);
  all = n <= p.budget;
  return all ? 0u : (uint32_t)max(0, min(p.budget - (n - (hi - lo)), hi - lo));
}

// The threshold where no weight has to be looked for: everything, or nothing of [lo, hi).
__device__ __forceinline__ uint2 evict_trivial(bool all) {
  return all ? make_uint2(0u, 0x7FFFFFFFu) : make_uint2(0xFFFFFFFFu, 0u);
}

// The runs' counts in base (survivors above the threshold, weights at it) become their sums before each run.
template <int THREADS>
__device__ __forceinline__ void sum_runs(int2 *base, int runs, uint32_t *sums) {
  uint32_t gt0 = 0, eq0 = 0;
  for (int c0 = 0; c0 < runs; c0 += THREADS) {
    const int c = c0 + threadIdx.x;
    int2 x = make_int2(0, 0);
    if (c < runs) {
      const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(base + c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      x = make_int2((int)(uint32_t)v, (int)(v >> 32));
    }
    uint32_t gts, eqs;
    const uint32_t g = block_before<THREADS>((uint32_t)x.x, sums, gts), e = block_before<THREADS>((uint32_t)x.y, sums, eqs);
    if (c < runs) base[c] = make_int2((int)(gt0 + g), (int)(eq0 + e));
    gt0 += gts;
    eq0 += eqs;
  }
}

// Short contexts: a workgroup per head, the weights in its registers.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t sums[kSelectThreads / 64], found[2];
  __shared__ int runs_gt[kDirect / kRun], runs_eq[kDirect / kRun];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kvh = blockIdx.x, seq = blockIdx.y;
  const int n = evict_len(p, seq);
  const float *weights = p.weights + (int64_t)seq * p.w0 + (int64_t)kvh * p.w1;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  int lo, hi;
  bool all;
  uint32_t need = evict_need(p, n, lo, hi, all);
  if (kvh == 0 && tid == 0) p.new_used[seq] = min(n, p.budget);
  uint32_t u[kPer];
  const int used = (n + kSelectThreads - 1) / kSelectThreads;  // (slots past it hold nothing, and are not looked at)
  {
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = i * kSelectThreads + tid < n ? weights[i * kSelectThreads + tid] : 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) u[i] = weight_order(x[i]);
  }
  uint2 at = evict_trivial(all);
  if (need > 0) {
    uint32_t prefix = 0, mask = 0;
#pragma unroll
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? kFirstShift : level == 1 ? 10 : 0;
      const uint32_t nb = level == 2 ? 1024 : kBins;
#pragma unroll
      for (int i = 0; i < kBins / kSelectThreads; ++i) hist[i * kSelectThreads + tid] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (i >= used) break;
        const int j = i * kSelectThreads + tid;
        count_bin(hist, (u[i] >> shift) & (nb - 1), j >= lo && j < hi && (u[i] & mask) == prefix);
      }
      __syncthreads();
      auto counts = [&](int i) { return hist[i]; };
      const uint32_t bin = level == 2 ? find_bin<kSelectThreads, 1024>(counts, need, sums, found)
                                      : find_bin<kSelectThreads, kBins>(counts, need, sums, found);
      prefix |= bin << shift;
      mask |= (nb - 1) << shift;
      __syncthreads();
    }
    at = make_uint2(prefix, need);
  }
  if (tid == 0) p.threshold[head] = at;
  // ---- survivors above the threshold and weights at it per run: a wave's 64 positions lie in one
  const int runs = (n + kRun - 1) / kRun;
  for (int c = tid; c < runs; c += kSelectThreads) runs_gt[c] = runs_eq[c] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i >= used) break;
    const int j = i * kSelectThreads + tid;
    const bool sure = j < lo || j >= hi;
    const int gt = __builtin_popcountll(__ballot(j < n && (sure || u[i] > at.x)));
    const int eq = __builtin_popcountll(__ballot(j < n && !sure && u[i] == at.x));
    if (lane == 0 && j < n) {
      atomicAdd(&runs_gt[j / kRun], gt);
      atomicAdd(&runs_eq[j / kRun], eq);
    }
  }
  __syncthreads();
  int2 *base = p.base + head * p.runs;
  if (tid < 64) {  // (at most kDirect / kRun = 32 runs)
    int g = tid < runs ? runs_gt[tid] : 0, e = tid < runs ? runs_eq[tid] : 0;
    const int g0 = g, e0 = e;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(g, o, 64), y = __shfl_up(e, o, 64);
      if (tid >= o) {
        g += x;
        e += y;
      }
    }
    if (tid < runs) base[tid] = make_int2(g - g0, e - e0);
  }
}

// ---- long contexts, first: the histogram of a part's upper bits
__global__ __launch_bounds__(kPartThreads) void evict_hist_kernel(const EvictParams p) {
  __shared__ uint32_t hist[kBins];
  const int tid = threadIdx.x, part = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int n = evict_len(p, seq);
  if (part == 0 && kvh == 0 && tid == 0) p.new_used[seq] = min(n, p.budget);
  if (part * kPart >= n) return;
  int lo, hi;
  bool all;
  if (evict_need(p, n, lo, hi, all) == 0) return;
  const float *weights = p.weights + (int64_t)seq * p.w0 + (int64_t)kvh * p.w1;
  float x[kPartPer];
#pragma unroll
  for (int i = 0; i < kPartPer; ++i) {
    const int j = part * kPart + i * kPartThreads + tid;
    x[i] = j >= lo && j < hi ? weights[j] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kBins / kPartThreads; ++i) hist[i * kPartThreads + tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPartPer; ++i) {
    const int j = part * kPart + i * kPartThreads + tid;
    count_bin(hist, weight_order(x[i]) >> kFirstShift, j >= lo && j < hi);
  }
  __syncthreads();
  uint32_t *out = p.hist + (((int64_t)seq * p.num_kv_heads + kvh) * p.parts + part) * kBins;
#pragma unroll
  for (int i = 0; i < kBins / kPartThreads; ++i) out[i * kPartThreads + tid] = hist[i * kPartThreads + tid];
}

// Second: the threshold's bin from all parts' histograms; the part's runs' counts of what lies above it, and its weights in
// the bin, with their runs, in the part's list.
__global__ __launch_bounds__(kPartThreads) void evict_list_kernel(const EvictParams p) {
  __shared__ uint32_t sums[kPartThreads / 64], found[2], listed;
  __shared__ int above[kPart / kRun];
  const int tid = threadIdx.x, lane = tid & 63, part = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int n = evict_len(p, seq);
  if (part * kPart >= n) return;
  const float *weights = p.weights + (int64_t)seq * p.w0 + (int64_t)kvh * p.w1;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  int lo, hi;
  bool all;
  uint32_t need = evict_need(p, n, lo, hi, all);
  float x[kPartPer];
#pragma unroll
  for (int i = 0; i < kPartPer; ++i) {
    const int j = part * kPart + i * kPartThreads + tid;
    x[i] = j < n ? weights[j] : 0.f;
  }
  if (tid < kPart / kRun) above[tid] = 0;
  if (tid == 0) listed = 0;
  uint32_t bin = all ? 0u : 0xFFFFFFFFu;  // (nothing to look for: every weight is above the bin, or none)
  if (need > 0) {
    const uint32_t *hist = p.hist + head * p.parts * kBins;
    const int parts = (n + kPart - 1) / kPart;
    uint2 c = make_uint2(0u, 0u);  // the thread's two bins, from the top
#pragma unroll 8
    for (int q = 0; q < parts; ++q) {
      const uint2 x = *reinterpret_cast<const uint2 *>(hist + (int64_t)q * kBins + kBins - 2 - 2 * tid);
      c.x += x.x;
      c.y += x.y;
    }
    bin = find_bin<kPartThreads, kBins>([&](int i) { return i & 1 ? c.y : c.x; }, need, sums, found);
    if (part == 0 && tid == 0) p.threshold[head] = make_uint2(bin, need);
  } else if (part == 0 && tid == 0) {
    p.threshold[head] = evict_trivial(all);
  }
  __syncthreads();
  uint2 *list = p.lists + (head * p.parts + part) * kPart;
#pragma unroll
  for (int i = 0; i < kPartPer; ++i) {
    const int j = part * kPart + i * kPartThreads + tid;
    const uint32_t u = weight_order(x[i]);
    const bool sure = j < lo || j >= hi, in = j < n && !sure && need > 0 && u >> kFirstShift == bin;
    const bool up = j < n && (sure || all || (need > 0 && u >> kFirstShift > bin));
    const int gt = __builtin_popcountll(__ballot(up));
    const uint64_t ins = __ballot(in);
    uint32_t to = 0;
    if (lane == 0) {
      if (gt) atomicAdd(&above[(i * kPartThreads + tid) / kRun], gt);
      if (ins) to = atomicAdd(&listed, (uint32_t)__builtin_popcountll(ins));
    }
    to = (uint32_t)__builtin_amdgcn_readfirstlane((int)to);
    if (in) list[to + __builtin_popcountll(ins & (((uint64_t)1 << lane) - 1))] = make_uint2(u, (uint32_t)(j / kRun));
  }
  __syncthreads();
  const int run = part * (kPart / kRun) + tid;
  if (tid < kPart / kRun && run * kRun < n) p.base[head * p.runs + run] = make_int2(above[tid], 0);
  if (tid == 0) p.list_len[head * p.parts + part] = (int)listed;
}

// Third: the threshold among the listed weights, and the runs' sums.
__global__ __launch_bounds__(kPartThreads) void evict_resolve_kernel(const EvictParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t sums[kPartThreads / 64], found[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, kvh = blockIdx.x, seq = blockIdx.y;
  const int n = evict_len(p, seq);
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  int2 *base = p.base + head * p.runs;
  const int runs = (n + kRun - 1) / kRun, parts = (n + kPart - 1) / kPart;
  int lo, hi;
  bool all;
  if (evict_need(p, n, lo, hi, all) > 0) {
    // Lists are taken in pieces of 256 entries, four per lane, a list by kShare waves; a wave's first piece stays in registers.
    constexpr int kWaves = kPartThreads / 64;
    const int share = parts >= kWaves ? 1 : kWaves / parts;  // waves per list
    const int q0 = w / share, i0 = (w - q0 * share) * 256, step = share * 256;
    auto length = [&](int q) { return q < parts ? p.list_len[head * p.parts + q] : 0; };
    auto load = [&](int q, int at, int len, uint2 (&x)[4]) {
      const uint2 *list = p.lists + (head * p.parts + q) * kPart;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = at + 64 * i + lane < len ? list[at + 64 * i + lane] : make_uint2(0u, 0u);
    };
    uint2 held[4];
    const int len0 = length(q0);
    load(q0, i0, len0, held);
    auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f(held[i], i0 + 64 * i + lane < len0);
      for (int q = q0; q < parts; q += kWaves) {
        const int len = q == q0 ? len0 : length(q);
        for (int at = q == q0 ? i0 + step : i0; at < len; at += step) {
          uint2 x[4];
          load(q, at, len, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) f(x[i], at + 64 * i + lane < len);
        }
      }
    };
    const uint2 first = p.threshold[head];
    uint32_t prefix = first.x << kFirstShift, need = first.y, mask = (uint32_t)(kBins - 1) << kFirstShift;
#pragma unroll
    for (int level = 1; level < 3; ++level) {
      const int shift = level == 1 ? 10 : 0;
      const uint32_t nb = level == 2 ? 1024 : kBins;
#pragma unroll
      for (int i = 0; i < kBins / kPartThreads; ++i) hist[i * kPartThreads + tid] = 0;
      __syncthreads();
      each([&](uint2 x, bool in) { count_bin(hist, (x.x >> shift) & (nb - 1), in && (x.x & mask) == prefix); });
      __syncthreads();
      auto counts = [&](int i) { return hist[i]; };
      const uint32_t bin = level == 2 ? find_bin<kPartThreads, 1024>(counts, need, sums, found)
                                      : find_bin<kPartThreads, kBins>(counts, need, sums, found);
      prefix |= bin << shift;
      mask |= (nb - 1) << shift;
      __syncthreads();
    }
    each([&](uint2 x, bool in) {
      if (in && x.x > prefix) atomicAdd(&base[x.y].x, 1);
      if (in && x.x == prefix) atomicAdd(&base[x.y].y, 1);
    });
    if (tid == 0) p.threshold[head] = make_uint2(prefix, need);
    wait_vmcnt<0>();  // (the atomics are done: sum_runs reads their results, past the vector cache)
    __syncthreads();
  }
  sum_runs<kPartThreads>(base, runs, sums);
}

// A run's survivors to their places: positions, weights and cells.
template <bool CELL>
__global__ __launch_bounds__(kRun) void evict_move_kernel(const EvictParams p) {
  __shared__ int list[kRun];        // the survivors
  __shared__ longlong2 places[kRun];  // CELL: byte offsets of the old and the new cell; else their slots. Negative: no page
  __shared__ int counts[kRun / 64][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int j = c * kRun + tid;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  // (a row of weights holds max_keys of them: loaded beside the length, not after it)
  const float x = j < p.max_keys ? p.weights[(int64_t)seq * p.w0 + (int64_t)kvh * p.w1 + j] : 0.f;
  const uint2 at = p.threshold[head];
  const int equals = (int)at.y;
  const int2 base = p.base[head * p.runs + c];
  const int n = evict_len(p, seq);
  if (c * kRun >= n) return;
  int lo, hi;
  evict_range(p, n, lo, hi);
  const uint32_t u = weight_order(x);
  const bool sure = j < lo || j >= hi;
  const uint64_t mg = __ballot(j < n && (sure || u > at.x)), me = __ballot(j < n && !sure && u == at.x);
  if (lane == 0) {
    counts[w][0] = __builtin_popcountll(mg);
    counts[w][1] = __builtin_popcountll(me);
  }
  __syncthreads();
  int gt = base.x, eq = base.y, gts = base.x, eqs = base.y;
#pragma unroll
  for (int i = 0; i < kRun / 64; ++i) {
    gt += i < w ? counts[i][0] : 0;
    eq += i < w ? counts[i][1] : 0;
    gts += counts[i][0];
    eqs += counts[i][1];
  }
  const int first = base.x + min(base.y, equals);  // where the run's survivors begin
  const int total = gts + min(eqs, equals) - first;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  gt += __builtin_popcountll(mg & below);
  eq += __builtin_popcountll(me & below);
  if (((mg >> lane) & 1) || (((me >> lane) & 1) && eq < equals)) {
    const int to = gt + min(eq, equals);
    list[to - first] = j;
    p.kept[(int64_t)seq * p.k0 + (int64_t)kvh * p.k1 + to] = j;
    p.new_weights[(int64_t)seq * p.nw0 + (int64_t)kvh * p.nw1 + to] = x;
  }
  __syncthreads();
  auto place = [&](const int32_t *row, int blocks, int pos) -> int64_t {
    const int b = p.block_size == 1 ? pos : fast_div(pos, p.bs_magic, p.bs_shift);
    const int blk = b < blocks ? row[b] : -1;
    if ((uint32_t)blk >= (uint32_t)p.num_blocks) return -1;
    const int slot = pos - b * p.block_size;
    return CELL ? blk * p.ks0 + slot * p.ks1 + kvh * p.ks2 : (int64_t)blk << 32 | slot;
  };
  if (tid < total)
    places[tid] = make_longlong2(place(p.table + (int64_t)seq * p.table_stride, 0x7FFFFFFF, list[tid]),
                                 place(p.new_table + (int64_t)seq * p.new_stride, p.new_blocks, first + tid));
  __syncthreads();

  // ---- the cells, unit by unit (whole cells: 8 bytes; else key codes, key word, value codes, value word, 4 bytes each). A
  // thread's loads are all issued before any is stored.
  constexpr int kBatch = 4;
  uint8_t *cells = const_cast<uint8_t *>(p.kcodes);
  const uint32_t units = (uint32_t)total * (uint32_t)p.cell_units;
  for (uint32_t u0 = 0; u0 < units; u0 += kBatch * kRun) {
    u32x2_t data[kBatch];
    uint8_t *to[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t u = u0 + i * kRun + tid;
      to[i] = nullptr;
      if (u >= units) continue;
      const uint32_t e = (uint32_t)fast_div((int)u, p.cell_magic, p.cell_shift), d = u - e * p.cell_units;
      const longlong2 pl = places[e];
      if (pl.x < 0 || pl.y < 0) continue;
      if constexpr (CELL) {
        data[i] = *reinterpret_cast<const u32x2_t *>(p.kcodes + pl.x + 8 * d);
        to[i] = cells + pl.y + 8 * d;
      } else {
        const int64_t sb = pl.x >> 32, ss = pl.x & 0x7FFFFFFF, db = pl.y >> 32, ds = pl.y & 0x7FFFFFFF;
        const uint8_t *from;
        if ((int)d < p.key_units) {
          from = p.kcodes + sb * p.ks0 + ss * p.ks1 + kvh * p.ks2 + 4 * d;
          to[i] = cells + db * p.ks0 + ds * p.ks1 + kvh * p.ks2 + 4 * d;
        } else if ((int)d == p.key_units) {
          from = reinterpret_cast<const uint8_t *>(p.kwords + sb * p.kws0 + ss * p.kws1 + kvh * p.kws2);
          to[i] = reinterpret_cast<uint8_t *>(const_cast<uint32_t *>(p.kwords) + db * p.kws0 + ds * p.kws1 + kvh * p.kws2);
        } else if ((int)d <= p.key_units + p.value_units) {
          const int64_t off = kvh * p.vs2 + 4 * (int64_t)(d - p.key_units - 1);
          from = p.vcodes + sb * p.vs0 + ss * p.vs1 + off;
          to[i] = const_cast<uint8_t *>(p.vcodes) + db * p.vs0 + ds * p.vs1 + off;
        } else {
          from = reinterpret_cast<const uint8_t *>(p.vwords + sb * p.vws0 + ss * p.vws1 + kvh * p.vws2);
          to[i] = reinterpret_cast<uint8_t *>(const_cast<uint32_t *>(p.vwords) + db * p.vws0 + ds * p.vws1 + kvh * p.vws2);
        }
        data[i][0] = *reinterpret_cast<const uint32_t *>(from);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (to[i]) {
        if constexpr (CELL) *reinterpret_cast<u32x2_t *>(to[i]) = data[i];
        else *reinterpret_cast<uint32_t *>(to[i]) = data[i][0];
      }
  }
}

// Places in the workspace: the runs' counts and thresholds, and for long contexts the parts' histograms, lists and lengths.
struct EvictPlan {
  int64_t runs, parts, threshold_at, hist_at, lists_at, len_at, bytes;
};

EvictPlan evict_plan(const qp_paged_cache *c, const qp_evict_args *a) {
  EvictPlan k;
  const int64_t heads = (int64_t)a->num_seqs * c->num_kv_heads;
  k.runs = ((int64_t)a->max_seqlen_k + kRun - 1) / kRun;
  k.parts = a->max_seqlen_k > kDirect ? ((int64_t)a->max_seqlen_k + kPart - 1) / kPart : 0;
  k.threshold_at = heads * k.runs * 8;
  k.hist_at = (k.threshold_at + heads * 8 + 255) / 256 * 256;
  k.lists_at = k.hist_at + heads * k.parts * kBins * 4;
  k.len_at = k.lists_at + heads * k.parts * kPart * 8;
  k.bytes = (k.len_at + heads * k.parts * 4 + 7) / 8 * 8;
  return k;
}

// Whole cells ([K codes | K word | V codes | V word] without gaps) whose places are all multiples of 8 bytes.
bool whole_cells(const qp_paged_cache *c) {
  const int hs = c->head_size;
  const int kb = c->key.format == QP_CODES_INT4 ? hs / 2 : hs;
  const uint8_t *k = static_cast<const uint8_t *>(c->key.codes);
  if (static_cast<const uint8_t *>(c->key.words) != k + kb || static_cast<const uint8_t *>(c->value.codes) != k + kb + 4 ||
      static_cast<const uint8_t *>(c->value.words) != k + kb + 4 + hs / 2 || !aligned(k, 8))
    return false;
  for (int i = 0; i < 3; ++i)
    if (c->key.code_stride[i] != c->value.code_stride[i] || c->key.word_stride[i] * 4 != c->key.code_stride[i] ||
        c->value.word_stride[i] * 4 != c->key.code_stride[i] || c->key.code_stride[i] % 8)
      return false;
  return true;
}

int check_evict(const qp_paged_cache *c, const qp_evict_args *a) {
  QP_REQUIRE(c && a, "qp_evict: null argument");
  QP_SUPPORTED(c->head_size == 64 || c->head_size == 128 || c->head_size == 256 || c->head_size == 512,
               "qp_evict: head size must be 64, 128, 256 or 512");
  QP_REQUIRE((c->key.format == QP_CODES_INT4 || c->key.format == QP_CODES_INT8) && c->value.format == QP_CODES_INT4,
             "qp_evict: keys must be int4 or int8, values int4");
  QP_REQUIRE(c->num_kv_heads > 0 && c->num_blocks >= 0 && c->block_size > 0, "qp_evict: bad cache sizes");
  QP_SUPPORTED((int64_t)c->num_blocks * c->block_size < (int64_t(1) << 31), "qp_evict: at most 2^31 - 1 cache slots");
  QP_REQUIRE(a->num_seqs >= 0 && a->max_seqlen_k >= 0 && a->max_blocks >= 0 && a->new_max_blocks >= 0, "qp_evict: bad sizes");
  QP_SUPPORTED(a->num_seqs < 65536 && c->num_kv_heads < 65536, "qp_evict: at most 65535 sequences and KV heads");
  QP_SUPPORTED(a->max_seqlen_k <= 1 << 30, "qp_evict: at most 2^30 positions");
  QP_REQUIRE(a->budget > 0 && a->sinks >= 0 && a->recent >= 0 && (int64_t)a->sinks + a->recent <= a->budget,
             "qp_evict: the budget must be positive and hold the first `sinks` and the last `recent` positions");
  return QP_OK;
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_evict_workspace_size(const qp_paged_cache *cache, const qp_evict_args *a) {
  if (check_evict(cache, a) != QP_OK) return 0;
  return evict_plan(cache, a).bytes;
}

extern "C" int qp_evict(const qp_paged_cache *cache, const qp_evict_args *a, qp_stream_t stream) {
  const int st = check_evict(cache, a);
  if (st != QP_OK) return st;
  if (a->num_seqs == 0) return QP_OK;
  const int64_t held = (int64_t)a->max_blocks * cache->block_size, room = (int64_t)a->new_max_blocks * cache->block_size;
  const int64_t keys = held < a->max_seqlen_k ? held : a->max_seqlen_k;
  QP_REQUIRE(a->seqused_k && a->new_seqused_k, "qp_evict: null tensor");
  QP_REQUIRE(keys == 0 || (cache->key.codes && cache->key.words && cache->value.codes && cache->value.words),
             "qp_evict: null cache view");
  QP_REQUIRE(keys == 0 || (a->weights && a->block_table && a->new_block_table && a->kept && a->new_weights),
             "qp_evict: null tensor");
  for (int i = 0; i < 3; ++i)
    QP_REQUIRE(cache->key.code_stride[i] % 4 == 0 && cache->value.code_stride[i] % 4 == 0,
               "qp_evict: code strides must be multiples of 4 bytes");
  QP_REQUIRE(aligned(cache->key.codes, 4) && aligned(cache->value.codes, 4) && aligned(cache->key.words, 4) &&
                 aligned(cache->value.words, 4),
             "qp_evict: cache views must be 4-byte aligned");
  QP_REQUIRE(room >= (keys < a->budget ? keys : a->budget), "qp_evict: the new block table has no room for the budget");
  const EvictPlan k = evict_plan(cache, a);
  QP_REQUIRE(a->workspace && a->workspace_bytes >= k.bytes && aligned(a->workspace, 8),
             "qp_evict: needs an 8-byte aligned workspace of qp_evict_workspace_size bytes");
  const int hs = cache->head_size;
  const int kb = cache->key.format == QP_CODES_INT4 ? hs / 2 : hs;
  const bool cells = whole_cells(cache);
  EvictParams p;
  p.kcodes = static_cast<const uint8_t *>(cache->key.codes);
  p.ks0 = cache->key.code_stride[0];
  p.ks1 = cache->key.code_stride[1];
  p.ks2 = cache->key.code_stride[2];
  p.kwords = static_cast<const uint32_t *>(cache->key.words);
  p.kws0 = cache->key.word_stride[0];
  p.kws1 = cache->key.word_stride[1];
  p.kws2 = cache->key.word_stride[2];
  p.vcodes = static_cast<const uint8_t *>(cache->value.codes);
  p.vs0 = cache->value.code_stride[0];
  p.vs1 = cache->value.code_stride[1];
  p.vs2 = cache->value.code_stride[2];
  p.vwords = static_cast<const uint32_t *>(cache->value.words);
  p.vws0 = cache->value.word_stride[0];
  p.vws1 = cache->value.word_stride[1];
  p.vws2 = cache->value.word_stride[2];
  p.weights = a->weights;
  p.w0 = a->weights_stride[0];
  p.w1 = a->weights_stride[1];
  p.used = a->seqused_k;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.new_table = a->new_block_table;
  p.new_stride = a->new_block_table_stride;
  p.kept = a->kept;
  p.k0 = a->kept_stride[0];
  p.k1 = a->kept_stride[1];
  p.new_weights = a->new_weights;
  p.nw0 = a->new_weights_stride[0];
  p.nw1 = a->new_weights_stride[1];
  p.new_used = a->new_seqused_k;
  uint8_t *space = static_cast<uint8_t *>(a->workspace);
  p.base = reinterpret_cast<int2 *>(space);
  p.threshold = reinterpret_cast<uint2 *>(space + k.threshold_at);
  p.hist = reinterpret_cast<uint32_t *>(space + k.hist_at);
  p.lists = reinterpret_cast<uint2 *>(space + k.lists_at);
  p.list_len = reinterpret_cast<int *>(space + k.len_at);
  p.runs = (int32_t)k.runs;
  p.parts = (int32_t)k.parts;
  p.num_blocks = cache->num_blocks;
  p.block_size = cache->block_size;
  p.num_kv_heads = cache->num_kv_heads;
  p.max_keys = (int32_t)keys;
  p.new_blocks = a->new_max_blocks;
  p.budget = a->budget;
  p.sinks = a->sinks;
  p.recent = a->recent;
  p.bs_magic = p.bs_shift = 0;
  if (cache->block_size > 1) div_magic((uint32_t)cache->block_size, &p.bs_magic, &p.bs_shift);
  p.key_units = kb / 4;
  p.value_units = hs / 8;
  p.cell_units = cells ? (kb + hs / 2 + 8) / 8 : kb / 4 + hs / 8 + 2;
  div_magic((uint32_t)p.cell_units, &p.cell_magic, &p.cell_shift);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (k.parts == 0) {
    evict_select_kernel<<<dim3(cache->num_kv_heads, a->num_seqs), kSelectThreads, 0, s>>>(p);
  } else {
    const dim3 grid(p.parts, cache->num_kv_heads, a->num_seqs);
    evict_hist_kernel<<<grid, kPartThreads, 0, s>>>(p);
    evict_list_kernel<<<grid, kPartThreads, 0, s>>>(p);
    evict_resolve_kernel<<<dim3(cache->num_kv_heads, a->num_seqs), kPartThreads, 0, s>>>(p);
  }
  if (keys > 0) {
    const dim3 grid(p.runs, cache->num_kv_heads, a->num_seqs);
    if (cells) evict_move_kernel<true><<<grid, kRun, 0, s>>>(p);
    else evict_move_kernel<false><<<grid, kRun, 0, s>>>(p);
  }
  return launch_status();
}
