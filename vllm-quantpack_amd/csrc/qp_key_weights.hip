// The attention weight that each cached key receives from a set of query rows, per KV head:
//
//   w[s, g, j] = decay w_prev[s, g, j] + sum_t sum_{h in g} p_{t,h,j},   p_{t,h,j} = e^(a_thj - lse_th),   a = scale q . k
//
// over the dequantised keys of the paged int4 / k8v4 cache, t over the sequence's query tokens (the last of its positions,
// causal), h over the query heads of KV head g. Only the key half of the cache is read.
//
// Two passes over the keys, which a workgroup takes in segments: the first leaves each row's maximum and sum over the
// segment, a small kernel joins them, and the second makes the probabilities and adds them up over the rows. A wave holds
// 32 keys unpacked in registers and goes over all the rows, which lie in LDS; the first pass puts the rows in the lanes
// (K Q^T, so that a lane's values belong to one row), the second the keys (Q K^T, so that they belong to one key): the same
// registers with the operands of the MFMA exchanged. Every weight has one owner, so no order of additions varies.
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
  float2 *stat;           // [sequence, KV head, row]: maximum and 1 / sum
  int32_t num_tokens, num_q_heads, num_kv_heads, num_blocks, block_size, max_blocks, max_keys, max_rows, segments, subs;
  int32_t chunk;          // rows in LDS at once
  uint32_t bs_magic, bs_shift;
  float scale_log2, decay;
};

constexpr int kKwWaves = 4;
constexpr int kKwThreads = kKwWaves * 64;
constexpr int kKwSubs = 4;              // 32-key tiles of a wave at most
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
  static constexpr int kChunk = 32768 / kRowBytes;                        // rows in LDS at most
  static constexpr int kGroup = HS / 8;                                   // lanes that load a row
  static __host__ __device__ constexpr int swz(int r, int c) { return HS == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); }
  // LDS of a chunk of `rows` rows: the rows, four scalars each, and in the first pass the waves' row states and key scalars
  static __host__ __device__ constexpr int lds(int rows, int pass) {
    return rows * kRowBytes + rows * 16 + (pass == 1 ? kKwWaves * 2 * rows * 8 + kKwWaves * 32 * 8 : 0);
  }
};

template <int HS, int FMT, int PASS>
__global__ __launch_bounds__(kKwThreads) void key_weights_kernel(const KeyWeightParams p) {
  using Sh = KwShape<HS, FMT>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int segment = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int n = max(0, min(p.used_k[seq], p.max_keys));
  const int seg_keys = p.subs * kKwWaves * 32;
  const int k0 = segment * seg_keys;
  if (k0 >= n) return;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  const int nrows = min(qlen * G, p.max_rows);
  const int chunk = p.chunk;
  uint8_t *qrows = smem;
  float *rsum = reinterpret_cast<float *>(smem + chunk * Sh::kRowBytes);  // a row's query sum,
  int *rpos = reinterpret_cast<int *>(rsum + chunk);                      // last visible position,
  float *rmax = reinterpret_cast<float *>(rpos + chunk);                  // (second pass) maximum
  float *rinv = rmax + chunk;                                             // and 1 / sum
  float2 *state = reinterpret_cast<float2 *>(rinv + chunk);               // (first pass) [wave, half, row]: maximum and sum
  float2 *kscal = state + kKwWaves * 2 * chunk + 32 * w;                  // (first pass) the wave's keys: scale, zero point
  const int32_t *trow = p.table + (int64_t)seq * p.table_stride;
  const int64_t row_base = ((int64_t)seq * p.num_kv_heads + kvh) * p.max_rows;

  float acc[kKwSubs];
#pragma unroll
  for (int s = 0; s < kKwSubs; ++s) acc[s] = 0.f;

  for (int rc = 0; rc < nrows; rc += chunk) {
    const int count = min(chunk, nrows - rc), tiles = (count + 31) / 32;
    if (rc) __syncthreads();
    // ---- the chunk's rows to LDS, rotated when asked (and then rounded to bf16 once), with their sums
    {
      const int gl = tid % Sh::kGroup;
      float sg[8];
      if (p.signs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sg[i] = p.signs[8 * gl + i];
      }
      for (int r = tid / Sh::kGroup; r < 32 * tiles; r += kKwThreads / Sh::kGroup) {
        const int rr = rc + r, tok = rr / G;
        const bool ok = r < count;
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (ok)
          v = *reinterpret_cast<const u32x4_t *>(p.q + (int64_t)(q0 + tok) * p.qs0 + (int64_t)(kvh * G + rr - tok * G) * p.qs1 +
                                                 8 * gl);
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = bf16_lo(v[i]);
          x[2 * i + 1] = bf16_hi(v[i]);
        }
        if (p.signs) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= sg[i];
          fwht_groups<8, Sh::kGroup>(x, lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16_lo(v[i]);
            x[2 * i + 1] = bf16_hi(v[i]);
          }
        }
        *reinterpret_cast<u32x4_t *>(qrows + r * Sh::kRowBytes + 16 * Sh::swz(r, gl)) = v;
        if constexpr (FMT == QP_CODES_INT4) {
          float s = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
          for (int o = 1; o < Sh::kGroup; o <<= 1) s += shfl_xor_f(s, o);
          if (gl == 0) rsum[r] = s;
        }
        if (gl == 0) {
          rpos[r] = ok ? n - qlen + tok : -1;
          if constexpr (PASS == 2) {
            const float2 st = ok ? p.stat[row_base + rr] : make_float2(0.f, 0.f);
            rmax[r] = st.x;
            rinv[r] = st.y;
          }
        }
      }
    }
    __syncthreads();

#pragma unroll
    for (int s = 0; s < kKwSubs; ++s) {
      const int kw = k0 + 32 * (s * kKwWaves + w);  // the wave's keys kw ..
      if (s >= p.subs || kw >= n) break;
      // ---- the lane's key, half h of its channels; a key past the context, or on a page that does not exist, is not seen
      const int key = kw + col;
      const int b = p.block_size == 1 ? key : fast_div(key, p.bs_magic, p.bs_shift);
      const int blk = key < n ? trow[b] : -1;
      const bool ok = (uint32_t)blk < (uint32_t)p.num_blocks;
      uint32_t raw[Sh::kRaw];
      float a = 0.f, z = 0.f;
#pragma unroll
      for (int i = 0; i < Sh::kRaw; ++i) raw[i] = 0;
      if (ok) {
        const int64_t slot = key - b * p.block_size;
        const uint8_t *src = p.codes + blk * p.cs0 + slot * p.cs1 + kvh * p.cs2 + 4 * Sh::kRaw * h;
#pragma unroll
        for (int i = 0; i < Sh::kRaw / 4; ++i) {
          const u32x4_words_t x = *reinterpret_cast<const u32x4_words_t *>(src + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[4 * i + j] = x[j];
        }
        const uint32_t word = p.words[blk * p.ws0 + slot * p.ws1 + kvh * p.ws2];
        if constexpr (FMT == QP_CODES_INT4) {
          a = __uint_as_float(word & 0xFFFFFFF0u) * (16.f * p.scale_log2);  // (the product is over code - 8, over 16)
          z = ((float)(word & 0xFu) - 8.f) * 0.0625f;
        } else {
          a = __uint_as_float(word) * p.scale_log2;
        }
      }
      u32x4_t kop[Sh::kSteps];
#pragma unroll
      for (int i = 0; i < Sh::kSteps; ++i) {
        if constexpr (FMT == QP_CODES_INT4) kop[i] = kw_int4(raw[i]);
        else kop[i] = kw_int8(raw[2 * i], raw[2 * i + 1]);
      }
      const uint8_t *qlane = qrows + col * Sh::kRowBytes;
      auto q_op = [&](int t, int i) {
        return *reinterpret_cast<const u32x4_t *>(qlane + t * 32 * Sh::kRowBytes + 16 * Sh::swz(col, Sh::kSteps * h + i));
      };
      if constexpr (PASS == 1) {
        wave_sync();
        // (a key that is not there: scale NaN stands for it, no stored scale has it)
        if (h == 0) kscal[col] = make_float2(ok ? a : __builtin_nanf(""), z);
        wave_sync();
        for (int t = 0; t < tiles; ++t) {
          f32x16_t d = {};
#pragma unroll
          for (int i = 0; i < Sh::kSteps; ++i) d = kw_mfma(kop[i], q_op(t, i), d);
          // lane: row 32 t + col, keys 8 (i / 4) + 4 h + i % 4
          const float sum = FMT == QP_CODES_INT4 ? rsum[32 * t + col] : 0.f;
          const int pos = rpos[32 * t + col];
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int kk = 8 * (i >> 2) + 4 * h + (i & 3);
            const float2 sc = kscal[kk];
            d[i] = (FMT == QP_CODES_INT4 ? fmaf(-sum, sc.y, d[i]) : d[i]) * sc.x;
            if (kw + kk > pos || sc.x != sc.x) d[i] = -INFINITY;
            top = fmaxf(top, d[i]);
          }
          float2 *st = state + (2 * w + h) * chunk + 32 * t + col;
          const float2 was = s == 0 ? make_float2(kKwNone, 0.f) : *st;
          const float to = fmaxf(was.x, top);
          float l = was.y * __builtin_amdgcn_exp2f(was.x - to);
#pragma unroll
          for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(d[i] - to);
          *st = make_float2(to, l);
        }
      } else {
        float sum = 0.f;
        for (int t = 0; t < tiles; ++t) {
          f32x16_t d = {};
#pragma unroll
          for (int i = 0; i < Sh::kSteps; ++i) d = kw_mfma(q_op(t, i), kop[i], d);
          // lane: key kw + col, rows 32 t + 8 (i / 4) + 4 h + i % 4
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
            const float v = FMT == QP_CODES_INT4 ? fmaf(-rsum[r], z, d[i]) : d[i];
            const float e = __builtin_amdgcn_exp2f(fmaf(v, a, -rmax[r]));
            sum = fmaf(key <= rpos[r] ? e : 0.f, rinv[r], sum);
          }
        }
        acc[s] += ok ? sum : 0.f;
      }
    }
    if constexpr (PASS == 1) {
      __syncthreads();
      for (int r = tid; r < count; r += kKwThreads) {
        float top = kKwNone, l = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * kKwWaves; ++i)
          if (k0 + 32 * (i >> 1) < n) top = fmaxf(top, state[i * chunk + r].x);
#pragma unroll
        for (int i = 0; i < 2 * kKwWaves; ++i)
          if (k0 + 32 * (i >> 1) < n) {
            const float2 st = state[i * chunk + r];
            l = fmaf(st.y, __builtin_amdgcn_exp2f(st.x - top), l);
          }
        p.part[(((int64_t)seq * p.num_kv_heads + kvh) * p.segments + segment) * p.max_rows + rc + r] = make_float2(top, l);
      }
    }
  }
  if constexpr (PASS == 2) {
#pragma unroll
    for (int s = 0; s < kKwSubs; ++s) {
      const int key = k0 + 32 * (s * kKwWaves + w) + col;
      if (s >= p.subs) break;
      const float sum = acc[s] + shfl_xor_f(acc[s], 32);
      if (h == 0 && key < n) {
        float v = sum;
        if (p.prev) v = fmaf(p.decay, p.prev[(int64_t)seq * p.ps0 + (int64_t)kvh * p.ps1 + key], v);
        p.out[(int64_t)seq * p.os0 + (int64_t)kvh * p.os1 + key] = v;
      }
    }
  }
}

// A row's maximum and sum over all segments, a wave per row.
__global__ __launch_bounds__(256) void key_weights_join_kernel(const KeyWeightParams p) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), kvh = blockIdx.y, seq = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int q0 = max(0, p.cu_q[seq]), qlen = max(0, min(p.cu_q[seq + 1], p.num_tokens) - q0);
  if (row >= min(qlen * G, p.max_rows)) return;
  const int n = max(0, min(p.used_k[seq], p.max_keys));
  const int seg_keys = p.subs * kKwWaves * 32, used = (n + seg_keys - 1) / seg_keys;
  const int64_t head = (int64_t)seq * p.num_kv_heads + kvh;
  const float2 *part = p.part + head * p.segments * p.max_rows + row;
  float top = kKwNone, l = 0.f;
  for (int s = lane; s < used; s += 64) {
    const float2 x = part[(int64_t)s * p.max_rows];
    const float to = fmaxf(top, x.x);
    l = fmaf(l, __builtin_amdgcn_exp2f(top - to), x.y * __builtin_amdgcn_exp2f(x.x - to));
    top = to;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float ot = shfl_xor_f(top, o), ol = shfl_xor_f(l, o);
    const float to = fmaxf(top, ot);
    l = l * __builtin_amdgcn_exp2f(top - to) + ol * __builtin_amdgcn_exp2f(ot - to);
    top = to;
  }
  // (a row that sees no key has no share; a sum that is no number stays none)
  if (lane == 0) p.stat[head * p.max_rows + row] = make_float2(top, l != 0.f ? 1.f / l : 0.f);
}

struct KwPlan {
  int subs, segments;
  int64_t max_rows, part_bytes, bytes;
};

KwPlan kw_plan(const qp_key_weights_args *a) {
  KwPlan k;
  const int64_t heads = (int64_t)a->num_seqs * a->num_kv_heads, cus = device_cus();
  const int64_t keys = a->max_seqlen_k;
  k.subs = kKwSubs;  // long segments, unless they are too few to fill the GPU
  while (k.subs > 1 && heads * ((keys + 128 * k.subs - 1) / (128 * k.subs)) < 2 * cus) k.subs >>= 1;
  k.segments = (int)((keys + 128 * k.subs - 1) / (128 * k.subs));
  k.max_rows = (int64_t)a->max_query_len * (a->num_q_heads / a->num_kv_heads);
  k.part_bytes = heads * k.segments * k.max_rows * 8;
  k.bytes = k.part_bytes + heads * k.max_rows * 8;
  return k;
}

template <int HS, int FMT>
void launch_key_weights(KeyWeightParams &p, int seqs, hipStream_t s) {
  using Sh = KwShape<HS, FMT>;
  const int rows = (p.max_rows + 31) / 32 * 32;
  p.chunk = rows < Sh::kChunk ? (rows < 32 ? 32 : rows) : Sh::kChunk;
  const dim3 grid(p.segments, p.num_kv_heads, seqs);
  if (p.max_rows > 0) {
    key_weights_kernel<HS, FMT, 1><<<grid, kKwThreads, Sh::lds(p.chunk, 1), s>>>(p);
    key_weights_join_kernel<<<dim3((p.max_rows + 3) / 4, p.num_kv_heads, seqs), 256, 0, s>>>(p);
  }
  key_weights_kernel<HS, FMT, 2><<<grid, kKwThreads, Sh::lds(p.chunk, 2), s>>>(p);
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
  QP_SUPPORTED((int64_t)a->max_query_len * (a->num_q_heads / a->num_kv_heads) < (int64_t(1) << 30),
               "qp_key_weights: too many query rows");
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
  if (a->num_seqs == 0 || a->max_seqlen_k == 0) return QP_OK;
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
  p.part = static_cast<float2 *>(a->workspace);
  p.stat = reinterpret_cast<float2 *>(static_cast<uint8_t *>(a->workspace) + k.part_bytes);
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
