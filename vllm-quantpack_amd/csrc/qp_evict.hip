// Eviction from the paged int4 / k8v4 cache by the weight that its keys have received: per sequence and KV head the first
// `sinks` and last `recent` positions and, of the others, those of largest weight (the lowest position first among equal
// ones), `budget` in all; their cells go to new blocks in the order of their positions, with their weights.
//
// Two launches. A workgroup per (sequence, KV head) finds the smallest weight that stays, bit by bit from the top of its
// order-preserving integer (three histograms of 11, 11 and 10 bits in LDS), and counts what stays in each run of kChunk
// positions. Then a workgroup per run knows where its survivors go, lists them and moves their cells: every cell is read
// once and written once, and nothing is sorted. All counts are integers, so nothing depends on an order of atomics.
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
  uint32_t *threshold;    // [sequence, KV head, 2]: the smallest weight's integer, and how many of that weight stay
  int2 *base;             // [sequence, KV head, run]: survivors above the threshold, and weights at it, before the run
  int32_t num_blocks, block_size, num_kv_heads, max_keys, new_blocks, budget, sinks, recent, chunks;
  uint32_t bs_magic, bs_shift;
  int32_t key_units, value_units, cell_units;  // of the copies: 4 bytes, or 8 in whole cells
  uint32_t cell_magic, cell_shift;
};

constexpr int kEvictChunk = 1024;    // positions of a run
constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;

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
  for (int i = 0; i < (int)blockDim.x / 64; ++i) {
    before += i < w ? sums[i] : 0;
    total += sums[i];
  }
  return before + x - v;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t sums[kSelectThreads / 64], found[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int kvh = blockIdx.x, seq = blockIdx.y;
  const int n = evict_len(p, seq);
  const float *weights = p.weights + (int64_t)seq * p.w0 + (int64_t)kvh * p.w1;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  int lo, hi;
  evict_range(p, n, lo, hi);
  uint32_t need = (uint32_t)max(0, min(p.budget - (n - (hi - lo)), hi - lo));  // how many of [lo, hi) stay
  if (kvh == 0 && tid == 0) p.new_used[seq] = min(n, p.budget);
  const bool all = n <= p.budget;
  uint32_t prefix = 0, mask = 0;  // the threshold's bits so far
  if (!all && need > 0) {
    const int shifts[3] = {21, 10, 0}, bins[3] = {2048, 2048, 1024};
#pragma unroll
    for (int level = 0; level < 3; ++level) {
      const int shift = shifts[level], nb = bins[level];
      for (int i = tid; i < nb; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      constexpr int kBatch = 8;
      for (int j0 = lo; j0 < hi; j0 += kBatch * kSelectThreads) {
        float x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int j = j0 + i * kSelectThreads + tid;
          x[i] = j < hi ? weights[j] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int j = j0 + i * kSelectThreads + tid;
          const uint32_t u = weight_order(x[i]);
          const bool in = j < hi && (u & mask) == prefix;
          const uint32_t bin = (u >> shift) & (nb - 1);
          const uint64_t some = __ballot(in);
          if (!some) continue;
          // (equal weights would queue up at one counter: lanes that share the first one's bin add once)
          const uint32_t first = __shfl(bin, (int)__builtin_ctzll(some), 64);
          const uint64_t same = __ballot(in && bin == first);
          if (in && bin != first) atomicAdd(&hist[bin], 1u);
          if (lane == (int)__builtin_ctzll(same)) atomicAdd(&hist[first], (uint32_t)__builtin_popcountll(same));
        }
      }
      __syncthreads();
      // the bin in which the need-th largest lies: counts from the top (thread t: bins nb - 1 - 2 t and below)
      const int per = nb / kSelectThreads;  // 2 or 1
      uint32_t mine[2] = {0, 0};
      for (int i = 0; i < per; ++i) mine[i] = hist[nb - 1 - (per * tid + i)];
      uint32_t total;
      uint32_t above = block_before(mine[0] + mine[1], sums, total);
      for (int i = 0; i < per; ++i) {
        if (above < need && need <= above + mine[i]) {
          found[0] = (uint32_t)(nb - 1 - (per * tid + i));
          found[1] = need - above;
        }
        above += mine[i];
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= (uint32_t)(nb - 1) << shift;
      need = found[1];
      __syncthreads();
    }
  }
  // threshold and the number of its equals that stay; everything or nothing of [lo, hi) stays without one
  const uint32_t at = all ? 0u : mask ? prefix : 0xFFFFFFFFu;
  const uint32_t equals = all ? 0x7FFFFFFFu : mask ? need : 0u;
  if (tid == 0) {
    p.threshold[2 * head] = at;
    p.threshold[2 * head + 1] = equals;
  }
  // ---- survivors above the threshold and weights at it per run of positions, and their sums before each run
  int2 *base = p.base + head * p.chunks;
  const int runs = (n + kEvictChunk - 1) / kEvictChunk;
  for (int c = w; c < runs; c += kSelectThreads / 64) {
    float x[kEvictChunk / 64];
#pragma unroll
    for (int i = 0; i < kEvictChunk / 64; ++i) {
      const int j = c * kEvictChunk + 64 * i + lane;
      x[i] = j < n ? weights[j] : 0.f;
    }
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < kEvictChunk / 64; ++i) {
      const int j = c * kEvictChunk + 64 * i + lane;
      const uint32_t u = weight_order(x[i]);
      const bool sure = j < lo || j >= hi;
      gt += __builtin_popcountll(__ballot(j < n && (sure || u > at)));
      eq += __builtin_popcountll(__ballot(j < n && !sure && u == at));
    }
    if (lane == 0) base[c] = make_int2(gt, eq);
  }
  __syncthreads();
  uint32_t gt0 = 0, eq0 = 0;
  for (int c0 = 0; c0 < runs; c0 += kSelectThreads) {
    const int c = c0 + tid;
    const int2 x = c < runs ? base[c] : make_int2(0, 0);
    uint32_t gts, eqs;
    const uint32_t g = block_before((uint32_t)x.x, sums, gts), e = block_before((uint32_t)x.y, sums, eqs);
    if (c < runs) base[c] = make_int2((int)(gt0 + g), (int)(eq0 + e));
    gt0 += gts;
    eq0 += eqs;
  }
}

template <bool CELL>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictParams p) {
  __shared__ int list[kEvictChunk];   // the run's survivors
  __shared__ int2 places[kEvictChunk];  // old and new (block * block size + slot), negative: not on a page that exists
  __shared__ int counts[kMoveThreads / 64][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int n = evict_len(p, seq);
  if (c * kEvictChunk >= n) return;
  const float *weights = p.weights + (int64_t)seq * p.w0 + (int64_t)kvh * p.w1;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  const uint32_t at = p.threshold[2 * head];
  const int equals = (int)p.threshold[2 * head + 1];
  const int2 base = p.base[head * p.chunks + c];
  int lo, hi;
  evict_range(p, n, lo, hi);
  // ---- a wave takes kEvictChunk / 4 consecutive positions, 64 at a time
  constexpr int kSlabs = kEvictChunk / kMoveThreads;
  const int j0 = c * kEvictChunk + w * 64 * kSlabs + lane;
  float x[kSlabs];
  uint64_t mg[kSlabs], me[kSlabs];
  int gt = 0, eq = 0;
#pragma unroll
  for (int i = 0; i < kSlabs; ++i) x[i] = j0 + 64 * i < n ? weights[j0 + 64 * i] : 0.f;
#pragma unroll
  for (int i = 0; i < kSlabs; ++i) {
    const int j = j0 + 64 * i;
    const uint32_t u = weight_order(x[i]);
    const bool sure = j < lo || j >= hi;
    mg[i] = __ballot(j < n && (sure || u > at));
    me[i] = __ballot(j < n && !sure && u == at);
    gt += __builtin_popcountll(mg[i]);
    eq += __builtin_popcountll(me[i]);
  }
  if (lane == 0) {
    counts[w][0] = gt;
    counts[w][1] = eq;
  }
  __syncthreads();
  gt = base.x;
  eq = base.y;
  for (int i = 0; i < w; ++i) {
    gt += counts[i][0];
    eq += counts[i][1];
  }
  const int first = base.x + min(base.y, equals);  // where the run's survivors begin
  int gts = base.x, eqs = base.y;
  for (int i = 0; i < kMoveThreads / 64; ++i) {
    gts += counts[i][0];
    eqs += counts[i][1];
  }
  const int total = gts + min(eqs, equals) - first;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int i = 0; i < kSlabs; ++i) {
    const int j = j0 + 64 * i;
    const int g = gt + __builtin_popcountll(mg[i] & below), e = eq + __builtin_popcountll(me[i] & below);
    const bool stays = ((mg[i] >> lane) & 1) || (((me[i] >> lane) & 1) && e < equals);
    if (stays) {
      const int to = g + min(e, equals);
      list[to - first] = j;
      p.kept[(int64_t)seq * p.k0 + (int64_t)kvh * p.k1 + to] = j;
      p.new_weights[(int64_t)seq * p.nw0 + (int64_t)kvh * p.nw1 + to] = x[i];
    }
    gt += __builtin_popcountll(mg[i]);
    eq += __builtin_popcountll(me[i]);
  }
  __syncthreads();
  const int32_t *trow = p.table + (int64_t)seq * p.table_stride, *nrow = p.new_table + (int64_t)seq * p.new_stride;
  auto place = [&](const int32_t *row, int blocks, int pos) {
    const int b = p.block_size == 1 ? pos : fast_div(pos, p.bs_magic, p.bs_shift);
    const int blk = b < blocks ? row[b] : -1;
    return (uint32_t)blk < (uint32_t)p.num_blocks ? blk * p.block_size + (pos - b * p.block_size) : -1;
  };
  for (int i = tid; i < total; i += kMoveThreads)
    places[i] = make_int2(place(trow, 0x7FFFFFFF, list[i]), place(nrow, p.new_blocks, first + i));
  __syncthreads();

  // ---- the cells, unit by unit: key codes, key word, value codes, value word. A thread's loads are all issued before any
  // is stored.
  constexpr int kBatch = 4;
  const uint32_t units = (uint32_t)total * (uint32_t)p.cell_units;
  for (uint32_t u0 = 0; u0 < units; u0 += kBatch * kMoveThreads) {
    u32x2_t data[kBatch];
    uint8_t *to[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t u = u0 + i * kMoveThreads + tid;
      to[i] = nullptr;
      if (u >= units) continue;
      const uint32_t e = (uint32_t)fast_div((int)u, p.cell_magic, p.cell_shift), d = u - e * p.cell_units;
      const int2 pl = places[e];
      if (pl.x < 0 || pl.y < 0) continue;
      auto split = [&](int at, int64_t &blk, int64_t &slot) {
        blk = p.block_size == 1 ? at : fast_div(at, p.bs_magic, p.bs_shift);
        slot = at - blk * p.block_size;
      };
      int64_t sb, ss, db, ds;
      split(pl.x, sb, ss);
      split(pl.y, db, ds);
      if constexpr (CELL) {
        const int64_t off = (int64_t)kvh * p.ks2 + 8 * d;
        data[i] = *reinterpret_cast<const u32x2_t *>(p.kcodes + sb * p.ks0 + ss * p.ks1 + off);
        to[i] = const_cast<uint8_t *>(p.kcodes) + db * p.ks0 + ds * p.ks1 + off;
      } else {
        const uint8_t *from;
        if ((int)d < p.key_units) {
          from = p.kcodes + sb * p.ks0 + ss * p.ks1 + kvh * p.ks2 + 4 * d;
          to[i] = const_cast<uint8_t *>(p.kcodes) + db * p.ks0 + ds * p.ks1 + kvh * p.ks2 + 4 * d;
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

int evict_chunks(const qp_evict_args *a) { return (int)(((int64_t)a->max_seqlen_k + kEvictChunk - 1) / kEvictChunk); }

int64_t evict_bytes(const qp_paged_cache *c, const qp_evict_args *a) {
  return (int64_t)a->num_seqs * c->num_kv_heads * ((int64_t)evict_chunks(a) * 8 + 8);
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
  QP_REQUIRE(a->budget > 0 && a->sinks >= 0 && a->recent >= 0 && (int64_t)a->sinks + a->recent <= a->budget,
             "qp_evict: the budget must be positive and hold the first `sinks` and the last `recent` positions");
  return QP_OK;
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_evict_workspace_size(const qp_paged_cache *cache, const qp_evict_args *a) {
  if (check_evict(cache, a) != QP_OK) return 0;
  return evict_bytes(cache, a);
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
  const int64_t need = evict_bytes(cache, a);
  QP_REQUIRE(a->workspace && a->workspace_bytes >= need && aligned(a->workspace, 8),
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
  p.base = static_cast<int2 *>(a->workspace);
  p.chunks = evict_chunks(a);
  p.threshold = reinterpret_cast<uint32_t *>(p.base + (int64_t)a->num_seqs * cache->num_kv_heads * p.chunks);
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
  evict_select_kernel<<<dim3(cache->num_kv_heads, a->num_seqs), kSelectThreads, 0, s>>>(p);
  if (keys > 0) {
    const dim3 grid(p.chunks, cache->num_kv_heads, a->num_seqs);
    if (cells) evict_move_kernel<true><<<grid, kMoveThreads, 0, s>>>(p);
    else evict_move_kernel<false><<<grid, kMoveThreads, 0, s>>>(p);
  }
  return launch_status();
}
