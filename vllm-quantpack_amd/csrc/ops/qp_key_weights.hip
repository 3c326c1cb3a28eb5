// The attention weight that each cached key receives from a set of query rows, per KV head:
//
//   w[s, g, j] = decay w_prev[s, g, j] + sum_t sum_{h in g} p_{t,h,j},   p_{t,h,j} = e^(a_thj - lse_th),   a = scale q . k
//
// over the dequantised keys of the paged int4 / k8v4 cache, t over the sequence's query tokens (the last of its positions,
// causal), h over the query heads of KV head g. Only the key half of the cache is read.
//
// Every weight has one owner, so no order of additions varies. With few query rows (a decode step) the scores are made once
// and kept between the passes; with many (the last tokens of a prompt) they are made twice, from keys unpacked in registers.
//
// What bounds it, measured: one token, 24 / 4 heads of 256, over 131072 int4 keys takes 30 us for the scores and 9.7 for the
// sums. A cell's key half lies beside its value half, so that nearly all lines of the cache are fetched: 135 MB for 66 of key
// codes, at 4.5 TB/s. 64 tokens over 32768 keys, 64 / 8 heads of 128: 62 us for the statistics and 49 for the weights, 550
// and 700 TFLOP/s, and 10 for rows and statistics. In the two passes the matrix pipes are busy for 33 and 38 % of the cycles and
// the vector pipes for 65 and 56: exponentials and scaling run beside the products only in part.
//
// Precision: codes enter the product as code - 8 (int4) or as they are (int8), exact in bf16 and centred, so that the zero
// point's share, sum(q) (zp - 8), takes away little; scores meet the row's maximum in one fused multiply-add.
#include "qp_common.h"
#include "quantpack_ops.h"

namespace qp {

struct KeyWeightParams {
  const uint8_t *codes;
  int64_t cs0, cs1, cs2;  // bytes
  const uint32_t *words;
  int64_t ws0, ws1, ws2;  // words
  const uint16_t *q;
  int64_t qs0, qs1;
  const int32_t *cu_q, *used_k, *table;
  int64_t table_stride;
  const float *signs;     // rotation of the query rows as they load (null: none)
  const float *prev;      // null: no earlier weights
  int64_t ps0, ps1;
  float *out;
  int64_t os0, os1;
  float2 *part;           // [sequence, KV head, segment, row]: maximum (log2 units) and sum of a row over a segment
  float2 *stat;           // many rows: [sequence, KV head, row_cap]: maximum and 1 / sum
  float *scores;          // few rows: [sequence, KV head, row, score_stride] in log2 units
  int64_t score_stride;
  int32_t num_tokens, num_q_heads, num_kv_heads, num_blocks, block_size, max_blocks, max_keys, max_rows, segments, subs;
  int32_t seg_keys;       // keys of a segment
  u32x4_t *rows, *sums;   // many rows: [sequence, KV head, row_cap] rows and their sum operands
  int32_t row_cap;
  uint32_t bs_magic, bs_shift;
  float scale_log2, decay;
};

constexpr int kKwWaves = 4;
constexpr int kKwThreads = kKwWaves * 64;
constexpr int kKwSubs = 4;              // 32-key tiles of a wave at most
constexpr int kKwBlocks = 8;           // blocks of keys of a workgroup at most (many rows)
constexpr float kKwNone = -1e30f;       // the maximum of a row that has seen no key

typedef uint32_t u32x4_words_t __attribute__((ext_vector_type(4), aligned(4)));

// 8 codes as bf16 pairs, channels in order: int4 code - 8 (over 16: the conversion's own unit), or int8.
__device__ __forceinline__ u32x4_t kw_int4(uint32_t x) {
  const uint32_t lo = x ^ 0x88888888u, hi = lo >> 4;
  u32x4_t y;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    y[j] = __builtin_amdgcn_perm(__float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(hi >> (8 * j))),
                                 __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(lo >> (8 * j))), 0x07060302u);
  return y;
}
__device__ __forceinline__ u32x4_t kw_int8(uint32_t x0, uint32_t x1) {
  u32x4_t y;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = (j < 2 ? x0 : x1) >> (16 * (j & 1));
    y[j] = __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)(x >> 8)), __float_as_uint((float)(int8_t)x), 0x07060302u);
  }
  return y;
}

__device__ __forceinline__ f32x16_t kw_mfma(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

template <int HS, int FMT>
struct KwShape {
  static constexpr int kSteps = HS / 16;                                  // MFMA steps
  static constexpr int kRaw = FMT == QP_CODES_INT4 ? HS / 16 : HS / 8;    // dwords of codes per lane: half a row
  static constexpr int kRowBytes = HS * 2;
  static constexpr int kGroup = HS / 8;                                   // lanes that load a row
  // The halves of a wave take a key's codes by turns of 16 bytes (adjacent lanes' loads then share their cache lines); the
  // 8-channel unit of a query row that step i of half h goes with:
  static __host__ __device__ constexpr int unit(int h, int i) {
    return FMT == QP_CODES_INT4 ? 8 * (i / 4) + 4 * h + i % 4 : 4 * (i / 2) + 2 * h + i % 2;
  }
  static __host__ __device__ constexpr int swz(int r, int c) { return HS == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); }
};

// Channels 8 gl .. of row rr (gl: the lane's number in its row's group) of a sequence and KV head, rotated when asked (and
// then rounded to bf16 once), and the row's sum; zeros when it is not there.
template <int HS>
__device__ __forceinline__ u32x4_t load_row(const KeyWeightParams &p, int q0, int kvh, int rr, bool there, float &sum) {
  constexpr int kGroup = HS / 8;
  const int gl = threadIdx.x % kGroup, G = p.num_q_heads / p.num_kv_heads, tok = rr / G;
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (there)
    v = *reinterpret_cast<const u32x4_t *>(p.q + (int64_t)(q0 + tok) * p.qs0 + (int64_t)(kvh * G + rr - tok * G) * p.qs1 + 8 * gl);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(v[i]);
    x[2 * i + 1] = bf16_hi(v[i]);
  }
  if (p.signs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= p.signs[8 * gl + i];
    fwht_groups<8, kGroup>(x, threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      x[2 * i] = bf16_lo(v[i]);
      x[2 * i + 1] = bf16_hi(v[i]);
    }
  }
  sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
  for (int o = 1; o < kGroup; o <<= 1) sum += shfl_xor_f(sum, o);
  return v;
}

// A key's entry of the block table (-1: past the context), and whether that is a page of the cache.
__device__ __forceinline__ int key_entry(const KeyWeightParams &p, const int32_t *trow, int key, int n, int &slot) {
  const int b = p.block_size == 1 ? key : fast_div(key, p.bs_magic, p.bs_shift);
  slot = key - b * p.block_size;
  return key < n ? trow[b] : -1;
}
__device__ __forceinline__ int as_page(const KeyWeightParams &p, int blk) {
  return (uint32_t)blk < (uint32_t)p.num_blocks ? blk : -1;
}

// The lane's half h of a key's codes, and its word; zeros for page -1.
template <int HS, int FMT>
__device__ __forceinline__ void load_key(const KeyWeightParams &p, int blk, int slot, int kvh, int h,
                                         uint32_t (&raw)[KwShape<HS, FMT>::kRaw], uint32_t &word) {
  using Sh = KwShape<HS, FMT>;
  word = 0;
#pragma unroll
  for (int i = 0; i < Sh::kRaw; ++i) raw[i] = 0;
  if (blk < 0) return;
  const uint8_t *src = p.codes + blk * p.cs0 + slot * p.cs1 + kvh * p.cs2 + 16 * h;
#pragma unroll
  for (int i = 0; i < Sh::kRaw / 4; ++i) {
    const u32x4_words_t x = *reinterpret_cast<const u32x4_words_t *>(src + 32 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[4 * i + j] = x[j];
  }
  word = p.words[blk * p.ws0 + slot * p.ws1 + kvh * p.ws2];
}

// A word's scale (log2 units; of code - 8 over 16) and zero point.
template <int FMT>
__device__ __forceinline__ float word_scale(const KeyWeightParams &p, uint32_t word) {
  return FMT == QP_CODES_INT4 ? __uint_as_float(word & 0xFFFFFFF0u) * (16.f * p.scale_log2) : __uint_as_float(word) * p.scale_log2;
}
template <int FMT>
__device__ __forceinline__ float word_zero(uint32_t word) {
  return FMT == QP_CODES_INT4 ? ((float)(word & 0xFu) - 8.f) * 0.0625f : 0.f;
}

// Step i's 8 channels of the codes.
template <int HS, int FMT>
__device__ __forceinline__ u32x4_t key_operand(const uint32_t (&raw)[KwShape<HS, FMT>::kRaw], int i) {
  if constexpr (FMT == QP_CODES_INT4) return kw_int4(raw[i]);
  else return kw_int8(raw[2 * i], raw[2 * i + 1]);
}

// ------------------------------------------------------------------------------------------------ few rows
//
// A decode step has up to 24 rows per KV head. The scores themselves are then few beside the codes they come from, and are
// kept in the workspace between the passes: the keys are read and unpacked once.

// Scores of a segment's keys, with the rows' maxima and sums over it: the lanes hold keys, the registers rows
// (NR of them: rows 8 (i / 4) + 4 h + i % 4), so a lane runs its own maximum and sum over its keys.
template <int HS, int FMT, int NR>
__global__ __launch_bounds__(kKwThreads) void key_scores_kernel(const KeyWeightParams p) {
  using Sh = KwShape<HS, FMT>;
  __shared__ __attribute__((aligned(16))) uint8_t qrows[32 * Sh::kRowBytes];
  __shared__ float rsum[32];
  __shared__ int rpos[32];
  __shared__ float2 state[kKwWaves][32];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int segment = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int n = max(0, min(p.used_k[seq], p.max_keys));
  const int k0 = segment * p.subs * kKwWaves * 32;
  if (k0 >= n) return;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int nrows = min(qlen * G, p.max_rows);
  const int32_t *trow = p.table + (int64_t)seq * p.table_stride;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  // the pages of all the wave's keys, then its first codes, before the rows
  int blk[kKwSubs], slot[kKwSubs];
#pragma unroll
  for (int s = 0; s < kKwSubs; ++s)
    blk[s] = s < p.subs ? as_page(p, key_entry(p, trow, k0 + 32 * (s * kKwWaves + w) + col, n, slot[s])) : -1;
  constexpr int kBuf = HS == 512 ? 1 : 2;
  uint32_t raw[kBuf][Sh::kRaw], word[kBuf];
  load_key<HS, FMT>(p, blk[0], slot[0], kvh, h, raw[0], word[0]);
  for (int r = tid / Sh::kGroup; r < 32; r += kKwThreads / Sh::kGroup) {
    float x;
    *reinterpret_cast<u32x4_t *>(qrows + r * Sh::kRowBytes + 16 * Sh::swz(r, tid % Sh::kGroup)) =
        load_row<HS>(p, q0, kvh, r, r < nrows, x);
    if (tid % Sh::kGroup == 0) {
      rsum[r] = x;
      rpos[r] = r < nrows ? n - qlen + r / G : -1;
    }
  }
  __syncthreads();
  float m[NR], l[NR], sum[NR];
  int pos[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = 8 * (i >> 2) + 4 * h + (i & 3);
    m[i] = kKwNone;
    l[i] = 0.f;
    sum[i] = FMT == QP_CODES_INT4 ? rsum[r] : 0.f;
    pos[i] = rpos[r];
  }
  float *scores = p.scores + head * p.max_rows * p.score_stride;
  const uint8_t *qlane = qrows + col * Sh::kRowBytes;
#pragma unroll
  for (int s = 0; s < kKwSubs; ++s) {
    const int kw = k0 + 32 * (s * kKwWaves + w);
    if (s >= p.subs || kw >= n) break;
    const int cur = s % kBuf;
    if (kBuf == 2 && s + 1 < kKwSubs) load_key<HS, FMT>(p, blk[s + 1], slot[s + 1], kvh, h, raw[(s + 1) % kBuf], word[(s + 1) % kBuf]);
    if (kBuf == 1 && s > 0) load_key<HS, FMT>(p, blk[s], slot[s], kvh, h, raw[0], word[0]);
    const float a = word_scale<FMT>(p, word[cur]), z = word_zero<FMT>(word[cur]);
    f32x16_t d = {};
#pragma unroll
    for (int i = 0; i < Sh::kSteps; ++i)
      d = kw_mfma(*reinterpret_cast<const u32x4_t *>(qlane + 16 * Sh::swz(col, Sh::unit(h, i))),
                  key_operand<HS, FMT>(raw[cur], i), d);
    const int key = kw + col;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = 8 * (i >> 2) + 4 * h + (i & 3);
      float x = (FMT == QP_CODES_INT4 ? fmaf(-sum[i], z, d[i]) : d[i]) * a;
      if (key > pos[i] || blk[s] < 0) x = -INFINITY;
      if (r < nrows && key < n) scores[r * p.score_stride + key] = x;
      const float to = fmaxf(m[i], x);
      l[i] = fmaf(l[i], __builtin_amdgcn_exp2f(m[i] - to), __builtin_amdgcn_exp2f(x - to));
      m[i] = to;
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    float to = m[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) to = fmaxf(to, shfl_xor_f(to, o));
    float x = l[i] * __builtin_amdgcn_exp2f(m[i] - to);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) x += shfl_xor_f(x, o);
    if (col == 0) state[w][8 * (i >> 2) + 4 * h + (i & 3)] = make_float2(to, x);
  }
  __syncthreads();
  if (tid < nrows) {
    float to = kKwNone, x = 0.f;
#pragma unroll
    for (int i = 0; i < kKwWaves; ++i) to = fmaxf(to, state[i][tid].x);
#pragma unroll
    for (int i = 0; i < kKwWaves; ++i) x = fmaf(state[i][tid].y, __builtin_amdgcn_exp2f(state[i][tid].x - to), x);
    p.part[(head * p.segments + segment) * p.max_rows + tid] = make_float2(to, x);
  }
}

// A row's maximum and sum over the segments that a context has, in every one of a group of LANES lanes.
template <int LANES>
__device__ __forceinline__ float2 join_row(const float2 *part, int64_t stride, int used) {
  float top = kKwNone, l = 0.f;
  for (int s = threadIdx.x % LANES; s < used; s += LANES) {
    const float2 x = part[s * stride];
    const float to = fmaxf(top, x.x);
    l = fmaf(l, __builtin_amdgcn_exp2f(top - to), x.y * __builtin_amdgcn_exp2f(x.x - to));
    top = to;
  }
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    const float ot = shfl_xor_f(top, o), ol = shfl_xor_f(l, o);
    const float to = fmaxf(top, ot);
    l = l * __builtin_amdgcn_exp2f(top - to) + ol * __builtin_amdgcn_exp2f(ot - to);
    top = to;
  }
  // (a row that sees no key has no share; a sum that is no number stays none)
  return make_float2(top, l != 0.f ? 1.f / l : 0.f);
}

// The weights from the scores: the rows' statistics joined by each workgroup for itself, then kSumKeys keys.
constexpr int kSumKeys = 1024;

__global__ __launch_bounds__(256) void key_weights_sum_kernel(const KeyWeightParams p) {
  __shared__ float2 stat[32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int n = max(0, min(p.used_k[seq], p.max_keys));
  const int k0 = blockIdx.x * kSumKeys;
  if (k0 >= n) return;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int nrows = min(qlen * G, p.max_rows);
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  const int used = (n + p.seg_keys - 1) / p.seg_keys;
  constexpr int kPer = kSumKeys / 256, kBatch = 4;
  const float *scores = p.scores + head * p.max_rows * p.score_stride + k0 + tid;
  float x[kBatch][kPer], acc[kPer] = {};
  auto load = [&](int r0) {
#pragma unroll
    for (int r = 0; r < kBatch; ++r)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[r][i] = r0 + r < nrows && k0 + tid + 256 * i < n ? scores[(r0 + r) * p.score_stride + 256 * i] : -INFINITY;
  };
  load(0);  // (in flight while the statistics are joined)
  for (int r = tid >> 6; r < nrows; r += 4) {
    const float2 st = join_row<64>(p.part + head * p.segments * p.max_rows + r, p.max_rows, used);
    if (lane == 0) stat[r] = st;
  }
  __syncthreads();
  for (int r0 = 0; r0 < nrows; r0 += kBatch) {
    if (r0) load(r0);
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      if (r0 + r >= nrows) break;
      const float2 st = stat[r0 + r];
#pragma unroll
      for (int i = 0; i < kPer; ++i)  // (a key out of sight adds nothing, not even of a row whose sum is no number)
        if (x[r][i] != -INFINITY) acc[i] = fmaf(__builtin_amdgcn_exp2f(x[r][i] - st.x), st.y, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int key = k0 + tid + 256 * i;
    if (key >= n) continue;
    float v = acc[i];
    if (p.prev) v = fmaf(p.decay, p.prev[(int64_t)seq * p.ps0 + (int64_t)kvh * p.ps1 + key], v);
    p.out[(int64_t)seq * p.os0 + (int64_t)kvh * p.os1 + key] = v;
  }
}

// ----------------------------------------------------------------------------------------------- many rows
//
// The last tokens of a prompt: hundreds of rows. The scores are made twice, by waves that hold their keys unpacked in
// registers and let all rows go by: the rows, rotated once into the workspace, stream through LDS.

// The query sum's part in a score, -sum (zp - 8), as one more step of the product: the sum in three bf16 (24 bits) against
// the zero point's three times.
__device__ __forceinline__ u32x4_t sum_operand(float sum) {
  float r = -sum;
  uint32_t b[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    b[i] = f32_to_bf16_bits(r);
    r -= __uint_as_float(b[i] << 16);
  }
  return u32x4_t{b[0] | b[1] << 16, b[2], 0u, 0u};
}
__device__ __forceinline__ u32x4_t zero_operand(float z, int h) {
  const uint32_t b = h == 0 ? __float_as_uint(z) >> 16 : 0u;  // (sixteenths up to 7: exact)
  return u32x4_t{b | b << 16, b, 0u, 0u};
}

// A sequence and KV head's rows, rotated when asked, to the workspace, with their sum operands; zeros up to row_cap.
template <int HS, int FMT>
__global__ __launch_bounds__(kKwThreads) void key_weights_rows_kernel(const KeyWeightParams p) {
  using Sh = KwShape<HS, FMT>;
  const int kvh = blockIdx.y, seq = blockIdx.z, G = p.num_q_heads / p.num_kv_heads;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int nrows = min(qlen * G, p.max_rows);
  const int64_t at = ((int64_t)seq * p.num_kv_heads + kvh) * p.row_cap;
  const int gl = threadIdx.x % Sh::kGroup, rr = blockIdx.x * (kKwThreads / Sh::kGroup) + threadIdx.x / Sh::kGroup;
  if (rr >= p.row_cap) return;  // (whole groups)
  float sum;
  const u32x4_t v = load_row<HS>(p, q0, kvh, rr, rr < nrows, sum);
  p.rows[(at + rr) * Sh::kGroup + gl] = v;
  if (FMT == QP_CODES_INT4 && gl == 0) p.sums[at + rr] = sum_operand(sum);
}

template <int HS, int FMT>
struct KwMany {
  using Sh = KwShape<HS, FMT>;
  static constexpr int kAt = HS <= 128 ? 2 : 1;        // 32-key tiles of a wave: each query operand serves them all
  static constexpr int kKeys = kAt * kKwWaves * 32;    // keys of a workgroup
  // Whether a block's codes come during the one before: where the registers hold both (41 sequences of 4096 int4 keys, 64
  // rows, head 128: 156 us so, 172 without; int8 at 128 would spill, and at 512 leave one wave per SIMD).
  static constexpr bool kAhead = kAt * (Sh::kRaw + 4 * Sh::kSteps) <= 80;
  static constexpr int kStageRows = HS == 512 ? 32 : 64;
  static constexpr int kSumsAt = kStageRows * Sh::kRowBytes;
  static constexpr int kStage = kSumsAt + kStageRows * 16;
  static constexpr int kCopies = kStageRows * Sh::kRowBytes / 1024 / kKwWaves;  // of rows, per wave
};

template <int HS, int FMT, int PASS>
__global__ __launch_bounds__(kKwThreads, 2) void key_weights_kernel(const KeyWeightParams p) {
  using Sh = KwShape<HS, FMT>;
  using Mn = KwMany<HS, FMT>;
  constexpr int kAt = Mn::kAt, kTiles = Mn::kStageRows / 32;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * Mn::kStage];
  __shared__ float kscale[kKwWaves][kAt * 32];                       // (first pass) the waves' keys
  // of three stages: (first pass) the waves' statistics, (second pass) the rows'
  __shared__ __attribute__((aligned(16))) float2 state[3][PASS == 1 ? kKwWaves : 1][Mn::kStageRows];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int segment = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int n = max(0, min(p.used_k[seq], p.max_keys));
  const int blocks = min(p.subs, (n + Mn::kKeys - 1) / Mn::kKeys - segment * p.subs);  // blocks of kKeys keys
  if (blocks <= 0) return;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int nrows = min(qlen * G, p.max_rows), before = n - qlen;  // row r's token sees the keys up to before + r / G
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  const int32_t *trow = p.table + (int64_t)seq * p.table_stride;
  // The rows go by in stages, once for each block of keys: step g is stage g % stages for block g / stages. Up to two stages
  // stay where they are. A stage comes by HBM -> LDS copies: copy i of a wave fills units 64 (w + 4 i) .., the swizzle in
  // the source.
  const int stages = (nrows + Mn::kStageRows - 1) / Mn::kStageRows, ntiles = (nrows + 31) / 32;
  const bool stay = stages <= 2;
  const int steps = blocks * stages;
  const uint32_t lds0 = lds_addr(smem);
  const uint8_t *rows = reinterpret_cast<const uint8_t *>(p.rows) + head * p.row_cap * Sh::kRowBytes;
  const uint8_t *sums = reinterpret_cast<const uint8_t *>(p.sums) + head * p.row_cap * 16;
  const uint8_t *stats = reinterpret_cast<const uint8_t *>(p.stat) + head * p.row_cap * 8;
  auto copy = [&](int g) {
    if (g >= steps || (stay && g >= stages)) return;
    const int st = g % stages;
    const uint32_t dst = lds0 + (uint32_t)((g & 1) * Mn::kStage);
#pragma unroll
    for (int i = 0; i < Mn::kCopies; ++i) {
      const int at = 64 * (w + kKwWaves * i), d = at + lane, r = d / Sh::kGroup, c = d % Sh::kGroup;
      dma16_saddr<false>(rows + (int64_t)st * Mn::kStageRows * Sh::kRowBytes, (uint32_t)(r * Sh::kRowBytes + 16 * Sh::swz(r, c)),
                         dst + 16 * at);
    }
    if (FMT == QP_CODES_INT4 && w == 0 && lane < Mn::kStageRows)
      dma16_saddr<false>(sums + (int64_t)st * Mn::kStageRows * 16, 16u * lane, dst + Mn::kSumsAt);
    if (PASS == 2 && w == 1 && lane < Mn::kStageRows / 2)
      dma16_saddr<false>(stats + (int64_t)st * Mn::kStageRows * 8, 16u * lane, lds_addr(&state[g % 3][0][0]));
  };
  copy(0);
  // the lane's keys, half h of their channels: a block's codes are loaded while the one before is at work, its table entries
  // one block earlier. A key past the context, or on a page that does not exist, is not seen.
  int entry[kAt], slot[kAt];
  uint32_t raw[kAt][Sh::kRaw], word[kAt];
  uint32_t there = 0;
  const int first = segment * p.subs * Mn::kKeys + 32 * kAt * w;  // the wave's keys of a block: first + kKeys block ..
  auto entries = [&](int blk) {
#pragma unroll
    for (int k = 0; k < kAt; ++k)
      entry[k] = blk < blocks ? key_entry(p, trow, first + Mn::kKeys * blk + 32 * k + col, n, slot[k]) : -1;
  };
  auto codes = [&]() {
    there = 0;
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int page = as_page(p, entry[k]);
      there |= page >= 0 ? 1u << k : 0u;
      load_key<HS, FMT>(p, page, slot[k], kvh, h, raw[k], word[k]);
    }
  };
  entries(0);
  if (Mn::kAhead) {
    codes();
    entries(1);
  }

  u32x4_t kop[kAt][Sh::kSteps], kz[kAt];
  float a[kAt], sum[kAt];
  int first_row[kAt];                          // (second pass) the first row whose token sees the lane's key
  f32x4_t av[PASS == 1 ? kAt : 1][4];          // (first pass) the scales of the lane's keys 8 q + 4 h .. of each tile
  f32x16_t d[kAt], dn[kAt];
  // (first pass) a step's statistics of the four waves, joined when all of them are there
  auto join = [&](int g) {
    if (g < 0) return;
    const int r = g % stages * Mn::kStageRows + tid;
    if (tid >= Mn::kStageRows || r >= nrows) return;
    float to = kKwNone, l = 0.f;
#pragma unroll
    for (int i = 0; i < kKwWaves; ++i) to = fmaxf(to, state[g % 3][i][tid].x);
#pragma unroll
    for (int i = 0; i < kKwWaves; ++i) l = fmaf(state[g % 3][i][tid].y, __builtin_amdgcn_exp2f(state[g % 3][i][tid].x - to), l);
    p.part[(head * p.segments + segment * p.subs + g / stages) * p.max_rows + r] = make_float2(to, l);
  };
  for (int blk = 0; blk < blocks; ++blk) {
    const int kw = first + Mn::kKeys * blk, g0 = blk * stages;
    bool ok[kAt];
    if (!Mn::kAhead) codes();
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      ok[k] = there >> k & 1;
      a[k] = word_scale<FMT>(p, word[k]);
      kz[k] = zero_operand(word_zero<FMT>(word[k]), h);
#pragma unroll
      for (int i = 0; i < Sh::kSteps; ++i) kop[k][i] = key_operand<HS, FMT>(raw[k], i);
      // (a key that is not there has the scale NaN, which the store never writes: its scales are at least 1e-6)
      if (PASS == 1 && h == 0) kscale[w][32 * k + col] = ok[k] ? a[k] : __builtin_nanf("");
      sum[k] = 0.f;
      first_row[k] = max(0, kw + 32 * k + col - before) * G;
    }
    const bool all = __all(there == (1u << kAt) - 1);
    const uint32_t shown = there;
    if constexpr (PASS == 1) {
      wave_sync();
#pragma unroll
      for (int k = 0; k < kAt; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) av[k][q] = *reinterpret_cast<const f32x4_t *>(&kscale[w][32 * k + 8 * q + 4 * h]);
      wave_sync();
    }
    if (blk == 0) {
      wait_vmcnt<0>();
      __syncthreads();
      copy(1);
    }
    if (Mn::kAhead) codes();
    entries(blk + (Mn::kAhead ? 2 : 1));
    auto scores = [&](int tile, f32x16_t (&d)[kAt]) {
      const int st = tile / kTiles, t = tile % kTiles;
      const uint8_t *stage = smem + ((stay ? st : g0 + st) & 1) * Mn::kStage;
#pragma unroll
      for (int k = 0; k < kAt; ++k) d[k] = f32x16_t{};
      if constexpr (FMT == QP_CODES_INT4) {
        const u32x4_t q = *reinterpret_cast<const u32x4_t *>(stage + Mn::kSumsAt + 16 * (32 * t + col));
#pragma unroll
        for (int k = 0; k < kAt; ++k) d[k] = PASS == 1 ? kw_mfma(kz[k], q, d[k]) : kw_mfma(q, kz[k], d[k]);
      }
#pragma unroll
      for (int i = 0; i < Sh::kSteps; ++i) {
        const u32x4_t q = *reinterpret_cast<const u32x4_t *>(stage + (32 * t + col) * Sh::kRowBytes + 16 * Sh::swz(col, Sh::unit(h, i)));
#pragma unroll
        for (int k = 0; k < kAt; ++k) d[k] = PASS == 1 ? kw_mfma(kop[k][i], q, d[k]) : kw_mfma(q, kop[k][i], d[k]);
      }
    };
    // a tile's scores to statistics, or weights. MASK: some row does not see all of the wave's keys, or some are not there
    auto process = [&](int tile, f32x16_t (&d)[kAt], auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      const int t = tile % kTiles, r0 = 32 * tile, at = PASS == 2 && stay ? tile / kTiles : (g0 + tile / kTiles) % 3;
      if constexpr (PASS == 1) {
        // lane: row r0 + col, keys 8 (i / 4) + 4 h + i % 4 of each tile
        float top = kKwNone, l = 0.f;
        const int pos = MASK ? before + (r0 + col) / G : 0;
#pragma unroll
        for (int k = 0; k < kAt; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float sc = av[k][i >> 2][i & 3];
            d[k][i] *= sc;
            if (MASK && (kw + 32 * k + 8 * (i >> 2) + 4 * h + (i & 3) > pos || sc != sc)) d[k][i] = -INFINITY;
            top = fmaxf(top, d[k][i]);
          }
        {
          const uint32_t b = __float_as_uint(top);
          const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
          top = fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
        }
#pragma unroll
        for (int k = 0; k < kAt; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(d[k][i] - top);
        {
          const uint32_t b = __float_as_uint(l);
          const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
          l = __uint_as_float(q[0]) + __uint_as_float(q[1]);
        }
        if (h == 0) state[at][w][32 * t + col] = make_float2(top, l);
      } else {
        // lane: key col of each tile, rows r0 + 8 q + 4 h + j
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4_t *sp = reinterpret_cast<const f32x4_t *>(&state[at][0][32 * t + 8 * q + 4 * h]);
          const f32x4_t s0 = sp[0], s1 = sp[1];
          const float mx[4] = {s0[0], s0[2], s1[0], s1[2]}, iv[4] = {s0[1], s0[3], s1[1], s1[3]};
#pragma unroll
          for (int k = 0; k < kAt; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float e = __builtin_amdgcn_exp2f(fmaf(d[k][4 * q + j], a[k], -mx[j]));
              // (a row that does not see the key adds nothing, not even where its sum is no number)
              if (!MASK || r0 + 8 * q + 4 * h + j >= first_row[k]) sum[k] = fmaf(e, iv[j], sum[k]);
            }
        }
      }
    };

    // ---- the walk over the rows' tiles: one's scores are made beside the one before's exponentials. Before a stage's last
    // tile the waves meet: the next stage has landed, every wave is past this one's rows, and the one after takes their place.
    auto meet = [&](int tile) {
      if (tile != ntiles - 1 && tile % kTiles != kTiles - 1) return;
      const int g = g0 + tile / kTiles;
      if (g + 1 < steps) {
        wait_vmcnt<0>();
        __syncthreads();
        copy(g + 2);
        if (PASS == 1) join(g - 1);
      }
    };
    // later rows see more: from `whole` on every row of a tile sees all of the wave's keys
    const int64_t ahead = (int64_t)max(0, kw + 32 * kAt - 1 - before) * G;
    const int whole = uniform(all ? (int)min((int64_t)ntiles, (ahead + 31) / 32) : ntiles);
    if (ntiles > 0) scores(0, d);
    auto step = [&](int tile, auto mask_tag) {
      meet(tile);
      scores(tile + 1, dn);
      process(tile, d, mask_tag);
#pragma unroll
      for (int k = 0; k < kAt; ++k) d[k] = dn[k];
    };
    int tile = 0;
    for (; tile < min(whole, ntiles - 1); ++tile) step(tile, std::true_type{});
    for (; tile < ntiles - 1; ++tile) step(tile, std::false_type{});
    if (ntiles > 0) {
      meet(tile);
      if (tile < whole) process(tile, d, std::true_type{});
      else process(tile, d, std::false_type{});
    }
    if constexpr (PASS == 2) {
#pragma unroll
      for (int k = 0; k < kAt; ++k) {
        const int key = kw + 32 * k + col;
        const float x = sum[k] + shfl_xor_f(sum[k], 32);
        if (h == 0 && key < n) {
          float v = shown >> k & 1 ? x : 0.f;
          if (p.prev) v = fmaf(p.decay, p.prev[(int64_t)seq * p.ps0 + (int64_t)kvh * p.ps1 + key], v);
          p.out[(int64_t)seq * p.os0 + (int64_t)kvh * p.os1 + key] = v;
        }
      }
    }
  }
  if (PASS == 1 && steps > 0) {
    __syncthreads();
    join(steps - 2);
    join(steps - 1);
  }
}

// A row's maximum and sum over all segments, LANES lanes per row.
template <int LANES>
__global__ __launch_bounds__(256) void key_weights_join_kernel(const KeyWeightParams p) {
  const int row = (blockIdx.x * 256 + threadIdx.x) / LANES, kvh = blockIdx.y, seq = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int n = max(0, min(p.used_k[seq], p.max_keys)), used = (n + p.seg_keys - 1) / p.seg_keys;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  if (row >= p.row_cap) return;  // (whole groups)
  float2 st = make_float2(0.f, 0.f);  // (a row that pads a stage has no share)
  if (row < min(qlen * G, p.max_rows)) st = join_row<LANES>(p.part + head * p.segments * p.max_rows + row, p.max_rows, used);
  if (threadIdx.x % LANES == 0) p.stat[head * p.row_cap + row] = st;
}

struct KwPlan {
  int subs, segments, seg_keys, row_cap;
  bool few;               // few rows: the scores are kept between the passes
  int64_t max_rows, score_stride, part_bytes, stat_bytes, sum_bytes, bytes;
};

int many_keys(int hs) {
  return hs == 64 ? KwMany<64, QP_CODES_INT4>::kKeys : hs == 128 ? KwMany<128, QP_CODES_INT4>::kKeys :
         hs == 256 ? KwMany<256, QP_CODES_INT4>::kKeys : KwMany<512, QP_CODES_INT4>::kKeys;
}

KwPlan kw_plan(const qp_key_weights_args *a) {
  KwPlan k = {};
  const int64_t heads = (int64_t)a->num_seqs * a->num_kv_heads, cus = device_cus();
  const int64_t keys = a->max_seqlen_k;
  k.max_rows = (int64_t)a->max_query_len * (a->num_q_heads / a->num_kv_heads);
  k.score_stride = (keys + 3) / 4 * 4;
  const int64_t score_bytes = heads * k.max_rows * k.score_stride * 4;
  // Few rows: their scores are kept (in up to 1 GiB) between the passes, instead of made twice. Kept against made twice, us,
  // one sequence of 65536 int4 keys: heads of 64 (32 / 8), 16 rows 33 / 38, 32 rows 53 / 39; 128 (32 / 8), 16 rows 38 / 47,
  // 32 rows 66 / 47; 256 (24 / 4), 24 rows 43 / 44; 512 (16 / 2), 16 rows 33 / 42, 32 rows 48 / 42.
  k.few = k.max_rows > 0 && k.max_rows <= 16 + std::min(a->head_size, 256) / 32 && score_bytes <= (int64_t(1) << 30);
  if (k.few) {
    k.subs = kKwSubs;  // long segments, unless they are too few to fill the GPU
    while (k.subs > 1 && heads * ((keys + 128 * k.subs - 1) / (128 * k.subs)) < 2 * cus) k.subs >>= 1;
    k.seg_keys = 128 * k.subs;
  } else {
    k.seg_keys = many_keys(a->head_size);
    k.row_cap = (int)((k.max_rows + 63) / 64 * 64);
    const int64_t blocks = (keys + k.seg_keys - 1) / k.seg_keys;
    k.subs = kKwBlocks;  // several blocks, as long as two workgroups per CU are there
    while (k.subs > 1 && heads * ((blocks + k.subs - 1) / k.subs) < 2 * cus) k.subs >>= 1;
  }
  k.segments = (int)((keys + k.seg_keys - 1) / k.seg_keys);
  k.part_bytes = (heads * k.segments * k.max_rows * 8 + 255) / 256 * 256;
  if (k.few) {
    k.bytes = k.part_bytes + score_bytes;
  } else {
    k.stat_bytes = heads * k.row_cap * 8;  // (multiples of 256, as row_cap is of 64)
    k.sum_bytes = heads * k.row_cap * 16;
    k.bytes = k.part_bytes + k.stat_bytes + k.sum_bytes + heads * k.row_cap * a->head_size * 2;
  }
  return k;
}

template <int HS, int FMT>
void launch_key_weights(KeyWeightParams &p, int seqs, hipStream_t s) {
  const dim3 grid(p.scores ? p.segments : (p.segments + p.subs - 1) / p.subs, p.num_kv_heads, seqs);
  if (p.scores) {
    if (p.max_rows <= 8) key_scores_kernel<HS, FMT, 4><<<grid, kKwThreads, 0, s>>>(p);
    else if (p.max_rows <= 16) key_scores_kernel<HS, FMT, 8><<<grid, kKwThreads, 0, s>>>(p);
    else key_scores_kernel<HS, FMT, 16><<<grid, kKwThreads, 0, s>>>(p);
    key_weights_sum_kernel<<<dim3((p.max_keys + kSumKeys - 1) / kSumKeys, p.num_kv_heads, seqs), 256, 0, s>>>(p);
    return;
  }
  if (p.row_cap > 0) {
    const int per = kKwThreads / KwShape<HS, FMT>::kGroup;
    key_weights_rows_kernel<HS, FMT><<<dim3(p.row_cap / per, p.num_kv_heads, seqs), kKwThreads, 0, s>>>(p);
    key_weights_kernel<HS, FMT, 1><<<grid, kKwThreads, 0, s>>>(p);
    // (lanes by the segments: 8 of them, 480 heads of 256 rows: 5 us with 4 lanes, 33 with 64)
    if (p.segments > 32) key_weights_join_kernel<64><<<dim3(p.row_cap / 4, p.num_kv_heads, seqs), 256, 0, s>>>(p);
    else key_weights_join_kernel<4><<<dim3(p.row_cap / 64, p.num_kv_heads, seqs), 256, 0, s>>>(p);
  }
  key_weights_kernel<HS, FMT, 2><<<grid, kKwThreads, 0, s>>>(p);
}

int check_key_weights(const qp_key_weights_args *a) {
  QP_REQUIRE(a, "qp_key_weights: null argument");
  QP_SUPPORTED(a->head_size == 64 || a->head_size == 128 || a->head_size == 256 || a->head_size == 512,
               "qp_key_weights: head size must be 64, 128, 256 or 512");
  QP_REQUIRE(a->key.format == QP_CODES_INT4 || a->key.format == QP_CODES_INT8, "qp_key_weights: unknown code format");
  QP_REQUIRE(a->num_kv_heads > 0 && a->num_q_heads > 0 && a->num_q_heads % a->num_kv_heads == 0,
             "qp_key_weights: query heads must be a multiple of KV heads");
  QP_REQUIRE(a->num_seqs >= 0 && a->num_tokens >= 0 && a->max_query_len >= 0 && a->max_seqlen_k >= 0 && a->num_blocks >= 0 &&
                 a->block_size > 0 && a->max_blocks >= 0,
             "qp_key_weights: bad sizes");
  QP_SUPPORTED(a->num_seqs < 65536 && a->num_kv_heads < 65536, "qp_key_weights: at most 65535 sequences and KV heads");
  const int64_t group = a->num_q_heads / a->num_kv_heads;
  QP_SUPPORTED(a->max_query_len * group < (int64_t(1) << 25) && a->num_tokens * group < (int64_t(1) << 31),
               "qp_key_weights: too many query rows");  // (up to 64 threads for each of a sequence's)
  QP_SUPPORTED(a->max_seqlen_k <= 1 << 30, "qp_key_weights: at most 2^30 positions");
  QP_REQUIRE(a->softmax_scale > 0.f && a->softmax_scale < INFINITY, "qp_key_weights: the softmax scale must be positive");
  return QP_OK;
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_key_weights_workspace_size(const qp_key_weights_args *a) {
  if (check_key_weights(a) != QP_OK) return 0;
  return kw_plan(a).bytes;
}

extern "C" int qp_key_weights(const qp_key_weights_args *a, qp_stream_t stream) {
  const int st = check_key_weights(a);
  if (st != QP_OK) return st;
  if (a->num_seqs == 0 || a->max_seqlen_k == 0 || a->max_blocks == 0) return QP_OK;  // (no position, or none with a page)
  QP_REQUIRE(a->key.codes && a->key.words && a->cu_seqlens_q && a->seqused_k && a->block_table && a->out,
             "qp_key_weights: null tensor");
  QP_REQUIRE(a->query || a->num_tokens == 0, "qp_key_weights: null tensor");
  for (int i = 0; i < 3; ++i)
    QP_REQUIRE(a->key.code_stride[i] % 4 == 0, "qp_key_weights: code strides must be multiples of 4 bytes");
  QP_REQUIRE(aligned(a->key.codes, 4) && aligned(a->key.words, 4), "qp_key_weights: cache views must be 4-byte aligned");
  QP_REQUIRE(aligned(a->query, 16) && a->query_stride[0] % 8 == 0 && a->query_stride[1] % 8 == 0,
             "qp_key_weights: query rows must be 16-byte aligned");
  const KwPlan k = kw_plan(a);
  QP_REQUIRE(k.bytes == 0 || (a->workspace && a->workspace_bytes >= k.bytes && aligned(a->workspace, 16)),
             "qp_key_weights: needs a 16-byte aligned workspace of qp_key_weights_workspace_size bytes");
  KeyWeightParams p;
  p.codes = static_cast<const uint8_t *>(a->key.codes);
  p.cs0 = a->key.code_stride[0];
  p.cs1 = a->key.code_stride[1];
  p.cs2 = a->key.code_stride[2];
  p.words = static_cast<const uint32_t *>(a->key.words);
  p.ws0 = a->key.word_stride[0];
  p.ws1 = a->key.word_stride[1];
  p.ws2 = a->key.word_stride[2];
  p.q = static_cast<const uint16_t *>(a->query);
  p.qs0 = a->query_stride[0];
  p.qs1 = a->query_stride[1];
  p.cu_q = a->cu_seqlens_q;
  p.used_k = a->seqused_k;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.signs = a->query_signs;
  p.prev = a->decay != 0.f ? a->previous : nullptr;
  p.ps0 = a->previous_stride[0];
  p.ps1 = a->previous_stride[1];
  p.out = a->out;
  p.os0 = a->out_stride[0];
  p.os1 = a->out_stride[1];
  uint8_t *space = static_cast<uint8_t *>(a->workspace);
  p.part = reinterpret_cast<float2 *>(space);
  space += k.part_bytes;
  p.scores = k.few ? reinterpret_cast<float *>(space) : nullptr;
  p.score_stride = k.score_stride;
  p.stat = reinterpret_cast<float2 *>(space);
  p.sums = reinterpret_cast<u32x4_t *>(space + k.stat_bytes);
  p.rows = reinterpret_cast<u32x4_t *>(space + k.stat_bytes + k.sum_bytes);
  p.row_cap = k.row_cap;
  p.num_tokens = a->num_tokens;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.max_blocks = a->max_blocks;
  const int64_t held = (int64_t)a->max_blocks * a->block_size;  // positions that a row of the block table has room for
  p.max_keys = (int32_t)(held < a->max_seqlen_k ? held : a->max_seqlen_k);
  p.max_rows = (int32_t)k.max_rows;
  p.segments = k.segments;
  p.subs = k.subs;
  p.seg_keys = k.seg_keys;
  p.bs_magic = p.bs_shift = 0;
  if (a->block_size > 1) div_magic((uint32_t)a->block_size, &p.bs_magic, &p.bs_shift);
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.decay = a->decay;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool i4 = a->key.format == QP_CODES_INT4;
  switch (a->head_size) {
    case 64: i4 ? launch_key_weights<64, QP_CODES_INT4>(p, a->num_seqs, s) : launch_key_weights<64, QP_CODES_INT8>(p, a->num_seqs, s); break;
    case 128: i4 ? launch_key_weights<128, QP_CODES_INT4>(p, a->num_seqs, s) : launch_key_weights<128, QP_CODES_INT8>(p, a->num_seqs, s); break;
    case 256: i4 ? launch_key_weights<256, QP_CODES_INT4>(p, a->num_seqs, s) : launch_key_weights<256, QP_CODES_INT8>(p, a->num_seqs, s); break;
    default: i4 ? launch_key_weights<512, QP_CODES_INT4>(p, a->num_seqs, s) : launch_key_weights<512, QP_CODES_INT8>(p, a->num_seqs, s); break;
  }
  return launch_status();
}
