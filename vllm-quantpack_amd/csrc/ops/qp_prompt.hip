// Attention over a prompt's own keys and values: packed sequences of different lengths, grouped heads, bf16 or fp16, heads
// of 64, 128, 256 and 512.
//
//   a_tj = scale q_t . k_j,   out_t = sum_j e^(a_tj - m_t) v_j / l_t,   l_t = sum_j e^(a_tj - m_t),   lse_t = m_t + ln l_t
//
// over the keys j <= t + keys - tokens of the row's sequence (all of them without causal). A row that sees no key gives
// zeros and an lse of -inf.
//
// A workgroup owns the rows, (token, query head) pairs of one KV head and sequence, of its waves' 32-row tiles, and walks
// the keys once in tiles, with the running maximum and sum of a softmax. S^T = K Q^T and O^T += V^T P^T run on 32x32x16
// MFMAs, so that a lane holds keys of one row: row maxima need no exchange but the one between the two halves of a wave,
// and the packed probabilities are the B operand of the second product as they are. K and V tiles are copied to LDS as they
// lie in memory, a tile ahead of their use; the V^T operand comes from the LDS's transposing reads (ds_read_b64_tr_b16).
//
// What bounds it, measured: 16384 tokens, 32 / 8 heads of 128, take 1.94 to 2.02 ms = 1090 to 1130 TFLOP/s. MFMAs keep the
// matrix pipes busy for 57 % of the cycles at 1.9 GHz and the vector pipes are busy for 54 %; the same kernel's MFMAs alone take
// 1.61 ms, without the exponentials it takes 1.87, without the reads of K and V from LDS 1.84. At head 256 (4096 tokens, 24 / 4
// heads, 257 us) the two are busy for 33 and 28 %. A token over 65536 keys, 64 / 8 heads of 128: 57 us for the walk = 4.7 TB/s,
// and 4.9 for the merge. Small batches are bound by the blocks with the most keys and by each block's start, 3 to 4 us.
#include "qp_common.h"
#include "quantpack_ops.h"

#include <algorithm>

namespace qp {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

struct PromptParams {
  const uint16_t *q;
  int64_t qs0, qs1;
  const uint16_t *k;
  int64_t ks0, ks1;
  const uint16_t *v;
  int64_t vs0, vs1;
  const int32_t *cu_q, *cu_k;
  uint16_t *out;
  int64_t os0, os1;
  float *lse;  // null: not asked for
  int64_t ls0, ls1;
  float *so, *smax, *ssum;  // split partials: [token, head, split, HS], [token, head, split]
  int32_t num_seqs, num_tokens, num_keys, num_q_heads, num_kv_heads, num_splits, min_keys, causal;
  int32_t group_keys;  // the longest context, where a block's keys may be halved between groups of waves (else 0)
  int32_t step;  // the row blocks of all sequences are taken in the order of their keys, in steps of so many (0: they are not)
  float scale_log2;
};

// The kernels' one argument, loaded where this is called: what only a kernel's end needs would take scalar registers all the
// way to it.
__device__ __forceinline__ PromptParams late_params() {
  auto at = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  PromptParams p;
  __builtin_memcpy(&p, (const void *)at, sizeof p);
  return p;
}

constexpr float kPromptNone = -1e30f;  // a row's reference before it has seen a key
// A row's scores are taken relative to a reference m (log2 units), its running maximum less prompt_below. It is raised when a
// score exceeds it by kPromptHeadroom more than that, so the largest probability lies between 2^below and 2^(below + headroom),
// and the row's sum above 2^below. bf16 has the exponents of fp32. fp16 loses bits below 2^-14 and has nothing below 2^-25, while
// the sum takes unrounded probabilities: with the largest at 2^7 or more, and at most 2^15, a key loses 2^-32 of the sum at
// most. Relative to the maximum itself, 65536 keys 17 nats below another's came out 43 % wrong, and 18 nats below as nothing; a
// call takes up to 1.3 % longer.
template <bool F16>
constexpr float prompt_below = F16 ? 7.f : 0.f;
constexpr float kPromptHeadroom = 8.f;
constexpr int kPromptWideRows = 64;       // rows of a workgroup at head 512

template <bool F16>
__device__ __forceinline__ f32x16_t mfma_prompt(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// Two fp32 as a pair of the input type, to nearest even.
template <bool F16>
__device__ __forceinline__ uint32_t pack_prompt(float lo, float hi) {
  if constexpr (F16) {
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

template <bool F16>
__device__ __forceinline__ float from_bits(uint16_t x) {
  return F16 ? (float)__builtin_bit_cast(_Float16, x) : __uint_as_float((uint32_t)x << 16);
}

// Maximum over the two lanes l, l ^ 32, both receiving it.
__device__ __forceinline__ float other_half_max(float v) {
  const uint32_t b = __float_as_uint(v);
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// log2 of the XCDs that share a (KV head, split) pair's row blocks: 8 over the largest power of two in the pairs.
__host__ __device__ __forceinline__ uint32_t prompt_share(uint32_t pairs) {
  return (pairs & 7) == 0 ? 0 : (pairs & 3) == 0 ? 1 : (pairs & 1) == 0 ? 2 : 3;
}

// ------------------------------------------------------------------------------------ what the kernels share

// A workgroup's part of the work: rows r0 .. of sequence `seq`'s (token, query head) rows of KV head kvh, keys [kb, ke) of
// its n. False: none.
struct PromptBlock {
  int kvh, q0, qlen, k0, n, nrows, r0, kb, ke, split;
};

// The row block of rank `rank` among those of all sequences (at most 64), the ones with most keys first: a long sequence's
// last blocks would otherwise begin late, and beside others of its length. Lengths are told apart in 64 steps of `step` keys:
// block j of a sequence is of step T where (step T - earlier keys) G / ROWS <= j, for the largest such T, and each lane counts
// the blocks of its step or more. False: there are fewer blocks.
template <int ROWS>
__device__ __forceinline__ bool block_by_length(const PromptParams &p, int rank, PromptBlock &b) {
  constexpr int kLog = __builtin_ctz(ROWS);
  const int G = p.num_q_heads / p.num_kv_heads, lane = threadIdx.x & 63, seqs = p.num_seqs;
  const int i = min(lane, seqs - 1);
  const int q0 = max(0, p.cu_q[i]), k0 = max(0, p.cu_k[i]);
  const int qlen = max(0, min(p.cu_q[i + 1], p.num_tokens) - q0), n = max(0, min(p.cu_k[i + 1], p.num_keys) - k0);
  const int blocks = lane < seqs ? (qlen * G + ROWS - 1) >> kLog : 0, before = (n - qlen) * G;
  auto at_least = [&](int T, int blocks, int before) {  // blocks of step T or more
    return T > 0 ? max(0, blocks - max(0, (p.step * T * G - before) >> kLog)) : blocks;
  };
  int count = 0;
  for (int s = 0; s < seqs; ++s)
    count += at_least(lane, __builtin_amdgcn_readlane(blocks, s), __builtin_amdgcn_readlane(before, s));
  const int above = __builtin_popcountll(__ballot(count > rank)), T = above - 1;
  if (above == 0) return false;
  const int longer = above < 64 ? __builtin_amdgcn_readlane(count, above) : 0;
  const int here = at_least(T, blocks, before), equal = here - (above < 64 ? at_least(T + 1, blocks, before) : 0);
  int left = rank - longer, s = 0;
  for (; s < seqs - 1; ++s) {
    const int e = __builtin_amdgcn_readlane(equal, s);
    if (left < e) break;
    left -= e;
  }
  b.q0 = __builtin_amdgcn_readlane(q0, s);
  b.qlen = __builtin_amdgcn_readlane(qlen, s);
  b.k0 = __builtin_amdgcn_readlane(k0, s);
  b.n = __builtin_amdgcn_readlane(n, s);
  b.r0 = (__builtin_amdgcn_readlane(blocks, s) - __builtin_amdgcn_readlane(here, s) + left) * ROWS;
  return true;
}

// The row block of number `blk`: sequence s's rows own blocks [cu_q[s] G / ROWS + s, ...). 63 sequences are looked at in one
// go. False: a block without rows.
template <int ROWS>
__device__ __forceinline__ bool block_by_number(const PromptParams &p, int blk, PromptBlock &b) {
  const int G = p.num_q_heads / p.num_kv_heads, lane = threadIdx.x & 63;
  int seq = -1, q1 = 0, k1 = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += 63) {
    const int i = min(s0 + lane, p.num_seqs);
    const int cq = p.cu_q[i], ck = p.cu_k[i];
    const uint64_t before =
        __ballot(s0 + lane < p.num_seqs && lane < 63 && (int)(((int64_t)cq * G) / ROWS) + s0 + lane <= blk);
    if (!before) break;
    const int at = 63 - __builtin_clzll(before);
    seq = s0 + at;
    b.q0 = __builtin_amdgcn_readlane(cq, at);
    q1 = __builtin_amdgcn_readlane(cq, at + 1);
    b.k0 = __builtin_amdgcn_readlane(ck, at);
    k1 = __builtin_amdgcn_readlane(ck, at + 1);
    if (at < 62) break;
  }
  if (seq < 0) return false;
  b.q0 = max(0, b.q0);
  b.k0 = max(0, b.k0);
  b.qlen = min(q1, p.num_tokens) - b.q0;
  b.n = max(0, min(k1, p.num_keys) - b.k0);
  b.r0 = (blk - (int)(((int64_t)b.q0 * G) / ROWS) - seq) * ROWS;
  return true;
}

template <int ROWS>
__device__ __forceinline__ bool prompt_block(const PromptParams &p, PromptBlock &b) {
  // Workgroups go to the 8 XCDs in turn: 2^share of them take the row blocks of the same (KV head, split) pairs, so that
  // the blocks that share keys share as few L2s as balance allows. Later blocks, which see more keys, come first.
  const uint32_t lin = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
  const uint32_t pairs = gridDim.y * gridDim.z, share = prompt_share(pairs), per = gridDim.x >> share;
  const uint32_t xcd = lin & 7, turn = (lin >> 3) / per;
  const uint32_t pair = (xcd >> share) * ((pairs << share) >> 3) + turn;
  const int blk = (int)(gridDim.x - 1 - ((((lin >> 3) - turn * per) << share) + (xcd & ((1u << share) - 1))));
  b.kvh = (int)(pair % gridDim.y);
  b.split = (int)(pair / gridDim.y);
  const int G = p.num_q_heads / p.num_kv_heads;
  if (!(p.step ? block_by_length<ROWS>(p, (int)gridDim.x - 1 - blk, b) : block_by_number<ROWS>(p, blk, b))) return false;
  b.nrows = b.qlen * G;
  if (b.r0 < 0 || b.r0 >= b.nrows) return false;
  const int last = p.causal ? b.n - b.qlen + (min(b.nrows, b.r0 + ROWS) - 1) / G : b.n - 1;
  const int seg = segment_keys(b.n, p.num_splits, p.min_keys);
  const int64_t kb = (int64_t)b.split * seg;
  if (p.num_splits > 1 && kb >= b.n) return false;  // an empty segment: the merge does not read it
  b.kb = (int)kb;
  b.ke = uniform((int)min((int64_t)max(0, min(b.n, last + 1)), kb + seg));
  return true;
}

// The V^T operand's lane offset in a tile of rows of HS channels: A row 8 q + 4 hh + j of channel tile ct is channel
// 32 ct + 16 hh + 4 q + j, so that a lane's accumulators are 16 consecutive channels. A 16-lane group reads four keys' rows,
// lanes 4 k .. 4 k + 3 the four 4-channel chunks 16 (c & 1) + 4 (c >> 1) of key k (8 channels further in the upper group),
// and gets them transposed: a lane four keys of its channel.
__device__ __forceinline__ int v_row(int lane) { return 4 * (lane >> 5) + ((lane >> 2) & 3); }
__device__ __forceinline__ int v_channel(int lane) {
  return 16 * (lane & 1) + 4 * ((lane >> 1) & 1) + 8 * ((lane >> 4) & 1);
}

// The operand's 8 keys of a channel: keys 4 h .. and 8 + 4 h .. of 16 (h the wave half), as the packed probabilities lie.
template <int HS>
__device__ __forceinline__ u32x4_t v_operand(const uint8_t *at) {
  u32x4_t r;
#pragma unroll
  for (int eight = 0; eight < 2; ++eight) {
    const i16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4_t *)(const __attribute__((address_space(3))) uint8_t *)(at + eight * 16 * HS));
    const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
    r[2 * eight] = y[0];
    r[2 * eight + 1] = y[1];
  }
  return r;
}

// Infinities and NaN in the values of keys that some row of a wave does not see: such a row's probability is 0, and the
// MFMA would make NaN of the product. A wave that meets them takes zeros in their place, and adds the value itself to the
// rows that see the key afterwards (any probability is above 0).
template <bool F16>
struct Odd {
  static constexpr uint32_t kInf = F16 ? 0x7C00u : 0x7F80u;
  static __device__ __forceinline__ u32x4_t without(u32x4_t x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((x[j] & kInf) == kInf) x[j] &= 0xFFFF0000u;
      if ((x[j] & (kInf << 16)) == kInf << 16) x[j] &= 0xFFFFu;
    }
    return x;
  }
  // values of keys [key, end) up to row_pos, a lane's channels 32 ct + 0..15 from `row` on, of rows `stride` bytes apart
  template <int CT>
  static __device__ __forceinline__ void restore(f32x16_t (&acc)[CT], const uint8_t *row, uint32_t stride, int key, int end,
                                                 int row_pos) {
    for (; key < end; ++key, row += stride) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const u32x4_t y[2] = {*reinterpret_cast<const u32x4_t *>(row + 64 * ct),
                              *reinterpret_cast<const u32x4_t *>(row + 64 * ct + 16)};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint16_t x = (uint16_t)(y[i >> 3][(i >> 1) & 3] >> (16 * (i & 1)));
          if ((x & kInf) == kInf && key <= row_pos) acc[ct][i] += from_bits<F16>(x);
        }
      }
    }
  }
};

// Whether 32 rows of a V tile hold any, for the whole wave.
template <int HS, bool F16>
__device__ __forceinline__ bool odd_values(const uint8_t *vt, int lane) {
  u16x2_t most = {0, 0};
#pragma unroll 2
  for (int d = lane; d < 32 * HS / 8; d += 64) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t *>(vt + 16 * d);
#pragma unroll
    for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, x[j] & 0x7FFF7FFFu));
  }
  return __any(most[0] >= Odd<F16>::kInf || most[1] >= Odd<F16>::kInf);
}

// The largest of a lane's 16 scores.
__device__ __forceinline__ float largest(const f32x16_t &x) {
  float a = fmaxf(fmaxf(x[0], x[1]), x[2]), b = fmaxf(fmaxf(x[3], x[4]), x[5]);
  a = fmaxf(fmaxf(a, x[6]), x[7]);
  b = fmaxf(fmaxf(b, x[8]), x[9]);
  a = fmaxf(fmaxf(a, x[10]), x[11]);
  b = fmaxf(fmaxf(b, x[12]), x[13]);
  a = fmaxf(fmaxf(a, x[14]), x[15]);
  return fmaxf(a, b);
}

// Scores of keys past the row's position or the split's end are -inf; key0: the key of the lane's first score.
__device__ __forceinline__ void mask_scores(f32x16_t &x, int key0, int row_pos, int ke) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int key = key0 + 8 * (i >> 2) + (i & 3);
    if (key > row_pos || key >= ke) x[i] = -INFINITY;
  }
}

// A row's reference m is raised for `top` (the largest score of the lane's keys, unscaled) where that exceeds it by more than the
// headroom, and what was summed up relative to the old one is scaled. A row's bits do not go by its neighbours': each is raised
// for itself. In fp16 the difference is the one that the exponentials take, so that none exceeds the type's range, however large
// the scores; bf16 has room for the scaled score's rounding (with fp16's form a token over 65536 keys takes 63.6 us, not 61.5).
template <bool F16, int CT>
__device__ __forceinline__ void raise(float top, float scale_log2, float &m, float &l, f32x16_t (&acc)[CT]) {
  constexpr float kMost = prompt_below<F16> + kPromptHeadroom;
  if (!F16) top *= scale_log2;
  auto exceeds = [&](float x) { return F16 ? fmaf(x, scale_log2, -m) > kMost : x > m + kMost; };
  if (__any(exceeds(top))) {
    const float most = other_half_max(top);
    const float to = exceeds(most) ? (F16 ? fmaf(most, scale_log2, -prompt_below<F16>) : most) : m;
    const float alpha = __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= alpha;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[ct][i] *= alpha;
  }
}

// A row's result: channels 32 ct + 16 h + 0..15 of `channel` on, to out or to the split's partial.
template <int HS, bool F16, int CT>
__device__ __forceinline__ void store_row(const PromptParams &p, const PromptBlock &b, int tok, int jh, int channel, bool stats,
                                          float m, float sum, const f32x16_t (&acc)[CT]) {
  if (tok < 0) return;
  const int64_t t = b.q0 + tok, head = b.kvh * (p.num_q_heads / p.num_kv_heads) + jh;
  if (p.num_splits == 1) {
    const float inv = sum != 0.f ? 1.f / sum : 0.f;  // (a sum that is no number stays none)
    uint16_t *orow = p.out + t * p.os0 + head * p.os1 + channel;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4_t y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = pack_prompt<F16>(acc[ct][8 * i + 2 * j] * inv, acc[ct][8 * i + 2 * j + 1] * inv);
        *reinterpret_cast<u32x4_t *>(orow + 32 * ct + 8 * i) = y;
      }
    if (p.lse && stats)
      p.lse[t * p.ls0 + head * p.ls1] = sum != 0.f ? (m + log2f(sum)) * (1.f / kLog2e) : -INFINITY;
  } else {
    const int64_t at = (t * p.num_q_heads + head) * p.num_splits + b.split;
    float *orow = p.so + at * HS + channel;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4 *>(orow + 32 * ct + i) = make_float4(acc[ct][i], acc[ct][i + 1], acc[ct][i + 2], acc[ct][i + 3]);
    if (stats) {
      p.smax[at] = m;
      p.ssum[at] = sum;
    }
  }
}

// ------------------------------------------------------------------------------------- heads of 64, 128 and 256

template <int HS_, bool F16_, int WAVES, int GROUPS = 1>
struct PromptShape {
  static constexpr int HS = HS_;
  static constexpr bool F16 = F16_;
  // Two waves per SIMD up to head 128, in one workgroup or two: prompt_rows says which. At 256 a wave takes 512 registers.
  static constexpr int kWaves = WAVES;
  static constexpr int kWavesPerSimd = HS <= 128 ? 2 : 1;
  // Two groups of waves share the rows, each with half of the keys, tiles of its own and a share of the sums, which are
  // joined through LDS at the end: twice the waves where there are few blocks.
  static constexpr int kGroups = GROUPS;
  static constexpr int kThreads = kGroups * kWaves * 64;
  static constexpr int kRows = kWaves * 32;
  static constexpr int kKeys = 64;                   // keys per tile, two sub-tiles of 32
  static constexpr int kU = HS / 8;                  // 16-byte units of a row
  static constexpr int kTile = kKeys * HS * 2;       // bytes of a tile's K (and of its V)
  static constexpr int kKRing = 2, kVRing = 3;       // tiles of K and V in LDS
  static constexpr int kOffV = kKRing * kTile;
  static constexpr int kLds = kOffV + kVRing * kTile;
  static constexpr int kCopies = kTile / 1024 / kWaves;  // 1 KiB copies of a wave, K and V each
  static constexpr int kCopyRows = kWaves * 64 / kU;     // rows of copy i of all waves
  static constexpr int kOffsets = kCopyRows >= 16 ? 1 : kCopies;
  static_assert(kTile % (1024 * kWaves) == 0 && kGroups * kLds <= 160 * 1024, "LDS");
  // Position of unit c in row r of a K tile: 16 rows' reads of one unit hit every bank of the LDS once.
  static __host__ __device__ constexpr int k_swz(int r, int c) { return HS == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); }
  // The same in a V tile, in blocks of four units (32 channels, what a transposing read takes of a row): the four rows of
  // a 16-lane group hit different banks. At head 64 a row has two blocks, and two rows every bank.
  static __host__ __device__ constexpr int v_swz(int r, int c) {
    return HS == 64 ? c ^ (((r >> 1) & 1) << 2) : c ^ ((r & 3) << 2);
  }
};

template <class Sh>
__global__ __launch_bounds__(Sh::kThreads, Sh::kWavesPerSimd) void prompt_kernel(const PromptParams p) {
  constexpr int HS = Sh::HS, KT = Sh::kKeys, U = Sh::kU;
  constexpr bool F16 = Sh::F16;
  constexpr int kCs = HS / 16, kCt = HS / 32;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Sh::kGroups * Sh::kLds];
  PromptBlock b;
  if (!prompt_block<Sh::kRows>(p, b)) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), w = wave % Sh::kWaves, group = wave / Sh::kWaves;
  const int place = group * Sh::kLds;  // of the group's tiles
  const int col = lane & 31, h = lane >> 5;
  const int G = p.num_q_heads / p.num_kv_heads;
  // the group's keys [kb, ke), of which there may be none in the last one; every wave walks ntiles tiles
  const int tiles = b.ke > b.kb ? (b.ke - b.kb + KT - 1) / KT : 0, ntiles = (tiles + Sh::kGroups - 1) / Sh::kGroups;
  const int kb = b.kb + group * ntiles * KT, ke = group == Sh::kGroups - 1 ? b.ke : min(b.ke, kb + ntiles * KT);
  auto last_pos = [&](int row) { return p.causal ? b.n - b.qlen + row / G : b.n - 1; };  // the last key that a row sees

  // ---- the wave's rows: lane row col -> (token rr / G, query head rr % G)
  const int wrow = b.r0 + 32 * w, rr = wrow + col;
  const bool active = wrow < b.nrows, valid = rr < b.nrows;
  const int tok = valid ? rr / G : -1, jh = valid ? rr - tok * G : 0;
  const int row_pos = valid ? last_pos(rr) : -1;
  u32x4_t qop[kCs];
  {
    const uint16_t *src = p.q + (int64_t)(b.q0 + max(0, tok)) * p.qs0 + (int64_t)(b.kvh * G + jh) * p.qs1 + 8 * h;
#pragma unroll
    for (int cs = 0; cs < kCs; ++cs)
      qop[cs] = valid ? *reinterpret_cast<const u32x4_t *>(src + 16 * cs) : u32x4_t{0u, 0u, 0u, 0u};
  }
  f32x16_t acc[kCt];
  float m = kPromptNone, l = 0.f;
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) acc[ct] = f32x16_t{};

  if (ntiles > 0) {
    auto seen = [&](int row) { return max(0, min(last_pos(row) + 1, ke) - kb); };  // keys of the split that a row sees
    const int wplain = uniform(active ? seen(wrow) : 0) / 32;  // sub-tiles that every row of the wave sees whole,
    const int wend = uniform(active ? seen(min(b.nrows, wrow + 32) - 1) + 31 : 0) / 32;  // and that some row sees at all

    // ---- HBM -> LDS: copy i of a wave fills 16-byte units 64 (w + kWaves i) .. of the tile, lane by lane; the unit's row
    // and column are those that the swizzle puts there
    const uint32_t lds0 = lds_addr(smem) + place;
    const uint8_t *kbase = reinterpret_cast<const uint8_t *>(p.k + (int64_t)(b.k0 + kb) * p.ks0 + (int64_t)b.kvh * p.ks1);
    const uint8_t *vbase = reinterpret_cast<const uint8_t *>(p.v + (int64_t)(b.k0 + kb) * p.vs0 + (int64_t)b.kvh * p.vs1);
    const uint32_t ksb = (uint32_t)(p.ks0 * 2), vsb = (uint32_t)(p.vs0 * 2);
    // the lane's byte offsets in a whole tile; copies a multiple of 16 rows apart differ by those rows only
    uint32_t kvo[Sh::kOffsets], vvo[Sh::kOffsets];
#pragma unroll
    for (int i = 0; i < Sh::kOffsets; ++i) {
      const int d = 64 * (w + Sh::kWaves * i) + lane, r = d / U, c = d % U;
      kvo[i] = (uint32_t)r * ksb + 16u * (uint32_t)Sh::k_swz(r, c);
      vvo[i] = (uint32_t)r * vsb + 16u * (uint32_t)Sh::v_swz(r, c);
    }
    auto copy = [&](int t, int kslot, int vslot) {
      const int left = ke - kb - t * KT - 1;  // the tile's last key (rows past it repeat it: always mapped memory)
      if (Sh::kGroups > 1 && left < 0) return;
      const uint8_t *kt = kbase + (int64_t)t * KT * ksb, *vt = vbase + (int64_t)t * KT * vsb;
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i) {
        const int at = 64 * (w + Sh::kWaves * i);
        const int base = i / Sh::kOffsets * Sh::kOffsets * Sh::kCopyRows;
        const uint8_t *kc = kt + (int64_t)base * ksb, *vc = vt + (int64_t)base * vsb;
        uint32_t ko = kvo[i % Sh::kOffsets], vo = vvo[i % Sh::kOffsets];
        if (left < KT - 1) {
          const int over = max(0, (64 * (w + Sh::kWaves * (i % Sh::kOffsets)) + lane) / U + base - left);
          kc = kt;
          vc = vt;
          ko += (uint32_t)(base - over) * ksb;
          vo += (uint32_t)(base - over) * vsb;
        }
        dma16_saddr<false>(kc, ko, lds0 + (uint32_t)(kslot * Sh::kTile + 16 * at));
        dma16_saddr<false>(vc, vo, lds0 + (uint32_t)(Sh::kOffV + vslot * Sh::kTile + 16 * at));
      }
    };
    // ---- operands. A swizzle changes the low bits of a unit's place only: a few lane offsets serve all steps, with the rest
    // immediate.
    constexpr int kKo = kCs < 8 ? kCs : 8, kVo = kCt < 4 ? kCt : 4;
    uint32_t koff[kKo], voff[kVo];
#pragma unroll
    for (int i = 0; i < kKo; ++i) koff[i] = place + col * (2 * HS) + 16 * Sh::k_swz(col, 2 * i + h);
#pragma unroll
    for (int i = 0; i < kVo; ++i)
      voff[i] = place + v_row(lane) * (2 * HS) + 16 * Sh::v_swz(v_row(lane), 4 * i) + 2 * v_channel(lane);
    auto k_op = [&](const uint8_t *kt, int cs) {
      return *reinterpret_cast<const u32x4_t *>(kt + koff[cs % kKo] + 256 * (cs / kKo));
    };
    auto v_op = [&](const uint8_t *vt, int ks, int ct) {
      return v_operand<HS>(vt + voff[ct % kVo] + 32 * ks * HS + 256 * (ct / kVo));
    };

    f32x16_t s;  // the running sub-tile's scores
    // Sub-tile g's softmax and second product beside the scores of g + 1. MASK: some row may not see all of g + 1 (or none
    // of it: whatever lies in its place is then masked). ODD: sub-tile g's values hold infinities or NaN.
    auto body = [&](const uint8_t *kn, const uint8_t *vt, int g, auto mask_tag, auto odd_tag) {
      constexpr bool MASK = decltype(mask_tag)::value, ODD = decltype(odd_tag)::value;
      constexpr int kP = 2 * kCt, kPre = 2;
      f32x16_t sn = {}, sn2 = {};
      u32x4_t kbuf[kPre], vbuf[kPre], pop[2];
#pragma unroll
      for (int c = 0; c < kPre; ++c) {
        kbuf[c] = k_op(kn, c);
        vbuf[c] = v_op(vt, c / kCt, c % kCt);
      }
      auto pair = [&](int i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * i], p.scale_log2, -m));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], p.scale_log2, -m));
        l += p0 + p1;  // (unrounded: the log-sum-exp is kept to fp32)
        pop[i >> 2][i & 3] = pack_prompt<F16>(p0, p1);
      };
      constexpr int kFirst = 6;    // pairs beside the first product, the others beside the second
      constexpr bool kTwo = HS == 256;  // two chains of MFMAs for the scores where one wave has a SIMD for itself
#pragma unroll
      for (int c = 0; c < kCs; ++c) {
        const u32x4_t kop = kbuf[c % kPre];
        if (c + kPre < kCs) kbuf[c % kPre] = k_op(kn, c + kPre);
        if (kTwo && (c & 1)) sn2 = mfma_prompt<F16>(kop, qop[c], sn2);
        else sn = mfma_prompt<F16>(kop, qop[c], sn);
#pragma unroll
        for (int i = 0; i < kFirst; ++i)
          if (i * kCs / kFirst == c) pair(i);
      }
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kP; ++c) {
        u32x4_t vop = vbuf[c % kPre];
        if constexpr (ODD) vop = Odd<F16>::without(vop);
        if (c + kPre < kP) vbuf[c % kPre] = v_op(vt, (c + kPre) / kCt, (c + kPre) % kCt);
        acc[c % kCt] = mfma_prompt<F16>(vop, pop[c / kCt], acc[c % kCt]);
        if (c < kCt) {
#pragma unroll
          for (int i = kFirst; i < 8; ++i)
            if ((i - kFirst) * kCt / (8 - kFirst) == c) pair(i);
        }
        if (c == kP / 2) {
          if constexpr (kTwo) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sn[i] += sn2[i];
          }
          if constexpr (MASK) mask_scores(sn, kb + 32 * (g + 1) + 4 * h, row_pos, ke);
          top = largest(sn);
        }
      }
      s = sn;
      raise<F16>(top, p.scale_log2, m, l, acc);
    };

    // ---- the walk. Tile t's last sub-tile is worked through beside the first scores of tile t + 1: before it the waves
    // meet, tile t + 1 having landed. Then every wave is past tile t's scores and tile t - 1's values, and tile t + 2 is
    // copied in their place.
    using No = std::false_type;
    using Yes = std::true_type;
    copy(0, 0, 0);
    if (ke - kb > KT) {
      copy(1, 1, 1);
      wait_vmcnt<2 * Sh::kCopies>();
    } else {
      wait_vmcnt<0>();
    }
    __syncthreads();
    if (wend > 0) {
      s = f32x16_t{};
#pragma unroll
      for (int c = 0; c < kCs; ++c) s = mfma_prompt<F16>(k_op(smem, c), qop[c], s);
      if (wplain == 0) mask_scores(s, kb + 4 * h, row_pos, ke);
      raise<F16>(largest(s), p.scale_log2, m, l, acc);
    }
    int t = 0, vslot = 0;
    auto k_at = [&](int t) { return smem + (t & 1) * Sh::kTile; };
    auto meet = [&] {
      wait_vmcnt<0>();
      __syncthreads();
      if (t + 2 < ntiles) copy(t + 2, t & 1, vslot == 0 ? 2 : vslot - 1);
    };
    for (; 2 * t + 2 < wplain; ++t) {  // both sub-tiles, and the one after, are seen whole by every row
      const uint8_t *vt = smem + Sh::kOffV + vslot * Sh::kTile;
      body(k_at(t) + 64 * HS, vt, 2 * t, No{}, No{});
      meet();
      body(k_at(t + 1), vt + 64 * HS, 2 * t + 1, No{}, No{});
      vslot = vslot == 2 ? 0 : vslot + 1;
    }
    for (; t < ntiles; ++t) {
      const uint8_t *tile = smem + Sh::kOffV + vslot * Sh::kTile;
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        if (u == 1) meet();
        const int g = 2 * t + u;
        if (g >= wend) continue;
        const uint8_t *kn = u == 0 ? k_at(t) + 64 * HS : k_at(t + 1), *vt = tile + u * 64 * HS;
        if (g >= wplain && odd_values<HS, F16>(vt + place, lane)) {
          body(kn, vt, g, Yes{}, Yes{});
          Odd<F16>::restore(acc, vbase + (int64_t)(32 * g) * vsb + 32 * h, vsb, kb + 32 * g, min(ke, kb + 32 * g + 32), row_pos);
        } else {
          body(kn, vt, g, Yes{}, No{});
        }
      }
      vslot = vslot == 2 ? 0 : vslot + 1;
    }
  }
  if constexpr (Sh::kGroups > 1) {
    if (ntiles > 0) {
      constexpr int kWave = kCt * 4096 + 512;  // a wave's sums, then its statistics
      f32x4_t *sums = reinterpret_cast<f32x4_t *>(smem + w * kWave) + lane;
      float2 *stats = reinterpret_cast<float2 *>(smem + w * kWave + kCt * 4096) + lane;
      __syncthreads();
      if (group == 1) {
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sums[64 * (4 * ct + i)] = f32x4_t{acc[ct][4 * i], acc[ct][4 * i + 1], acc[ct][4 * i + 2], acc[ct][4 * i + 3]};
        *stats = make_float2(m, l);
      }
      __syncthreads();
      if (group == 1) return;
      const float2 st = *stats;
      const float to = fmaxf(m, st.x), own = __builtin_amdgcn_exp2f(m - to), other = __builtin_amdgcn_exp2f(st.x - to);
      m = to;
      l = l * own + st.y * other;
#pragma unroll
      for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4_t x = sums[64 * (4 * ct + i)];
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[ct][4 * i + j] = acc[ct][4 * i + j] * own + x[j] * other;
        }
    } else if (group == 1) {
      return;
    }
  }
  // (at 256 there are registers to keep the arguments in, which is 1 % faster)
  store_row<HS, F16>(HS == 256 ? p : late_params(), b, tok, jh, 16 * h, h == 0, m, l + shfl_xor_f(l, 32), acc);
}

// -------------------------------------------------------------------------------------------- heads of 512
//
// A row tile's accumulators and query operands would take 384 registers: two waves share it, each with half of the channels
// of q, K, V and out. Each makes the scores of its channels, and the two parts are added through LDS; both then have the same
// bits and make the same probabilities.

template <bool F16>
__global__ __launch_bounds__(256) void prompt_wide_kernel(const PromptParams p) {
  constexpr int HS = 512, KT = 32, U = HS / 8, kHc = HS / 2, kWaves = 4;
  constexpr int kCs = kHc / 16, kCt = kHc / 32;
  constexpr int kTile = KT * HS * 2, kStage = 2 * kTile, kScores = 2 * kStage, kCopies = kTile / 1024 / kWaves;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kScores + kWaves * 4096];
  auto k_swz = [](int r, int c) { return c ^ (r & 15); };
  auto v_swz = [](int r, int c) { return c ^ ((r & 3) << 2); };
  PromptBlock b;
  if (!prompt_block<kPromptWideRows>(p, b)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5, part = w & 1;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int kb = b.kb, ke = b.ke;
  auto last_pos = [&](int row) { return p.causal ? b.n - b.qlen + row / G : b.n - 1; };
  const int rr = b.r0 + 32 * (w >> 1) + col;
  const bool valid = rr < b.nrows;
  const int tok = valid ? rr / G : -1, jh = valid ? rr - tok * G : 0;
  const int row_pos = valid ? last_pos(rr) : -1;
  u32x4_t qop[kCs];
  const uint16_t *src = p.q + (int64_t)(b.q0 + max(0, tok)) * p.qs0 + (int64_t)(b.kvh * G + jh) * p.qs1 + kHc * part + 8 * h;
#pragma unroll
  for (int cs = 0; cs < kCs; ++cs)
    qop[cs] = valid ? *reinterpret_cast<const u32x4_t *>(src + 16 * cs) : u32x4_t{0u, 0u, 0u, 0u};
  f32x16_t acc[kCt];
  float m = kPromptNone, l = 0.f;
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) acc[ct] = f32x16_t{};

  const int ntiles = ke > kb ? (ke - kb + KT - 1) / KT : 0;
  if (ntiles > 0) {
    const int plain = uniform(max(0, min(last_pos(b.r0) + 1, ke) - kb) / KT);  // tiles that every row of the block sees whole
    const uint32_t lds0 = lds_addr(smem);
    const uint8_t *kbase = reinterpret_cast<const uint8_t *>(p.k + (int64_t)(b.k0 + kb) * p.ks0 + (int64_t)b.kvh * p.ks1);
    const uint8_t *vbase = reinterpret_cast<const uint8_t *>(p.v + (int64_t)(b.k0 + kb) * p.vs0 + (int64_t)b.kvh * p.vs1);
    const uint32_t ksb = (uint32_t)(p.ks0 * 2), vsb = (uint32_t)(p.vs0 * 2);
    auto copy = [&](int t) {  // a copy is one row: 64 units
      const int left = ke - kb - t * KT - 1;
      const uint8_t *kt = kbase + (int64_t)t * KT * ksb, *vt = vbase + (int64_t)t * KT * vsb;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int r = w + kWaves * i, rs = min(r, left);
        const uint32_t dst = lds0 + (uint32_t)((t & 1) * kStage + 1024 * r);
        dma16_saddr<false>(kt + (int64_t)rs * ksb, 16u * (uint32_t)k_swz(r, lane), dst);
        dma16_saddr<false>(vt + (int64_t)rs * vsb, 16u * (uint32_t)v_swz(r, lane), dst + kTile);
      }
    };
    uint32_t koff[8], voff[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) koff[i] = col * (2 * HS) + 16 * (k_swz(col, 2 * i + h) + (kHc / 8) * part);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      voff[i] = v_row(lane) * (2 * HS) + 16 * (v_swz(v_row(lane), 4 * i) + (kHc / 8) * part) + 2 * v_channel(lane);
    auto tile = [&](const uint8_t *kt, int t, auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      const uint8_t *vt = kt + kTile;
      auto v_op = [&](int c) { return v_operand<HS>(vt + voff[c % kCt % 4] + 32 * (c / kCt) * HS + 256 * (c % kCt / 4)); };
      f32x16_t s = {}, s2 = {};
#pragma unroll
      for (int cs = 0; cs < kCs; ++cs) {
        const u32x4_t kop = *reinterpret_cast<const u32x4_t *>(kt + koff[cs % 8] + 256 * (cs / 8));
        if (cs & 1) s2 = mfma_prompt<F16>(kop, qop[cs], s2);
        else s = mfma_prompt<F16>(kop, qop[cs], s);
      }
      f32x4_t *own = reinterpret_cast<f32x4_t *>(smem + kScores + 4096 * w) + lane;
      const f32x4_t *other = reinterpret_cast<const f32x4_t *>(smem + kScores + 4096 * (w ^ 1)) + lane;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] += s2[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) own[64 * i] = f32x4_t{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4_t x = other[64 * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * i + j] += x[j];
      }
      if constexpr (MASK) mask_scores(s, kb + t * KT + 4 * h, row_pos, ke);
      raise<F16>(largest(s), p.scale_log2, m, l, acc);
      u32x4_t pop[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * i], p.scale_log2, -m));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], p.scale_log2, -m));
        l += p0 + p1;
        pop[i >> 2][i & 3] = pack_prompt<F16>(p0, p1);
      }
#pragma unroll
      for (int c = 0; c < 2 * kCt; ++c) acc[c % kCt] = mfma_prompt<F16>(v_op(c), pop[c / kCt], acc[c % kCt]);
    };
    // zeros in the place of a tile's infinities and NaN; whether there were any
    auto settle = [&](uint8_t *vt) {
      const bool odd = odd_values<HS, F16>(vt, lane);  // (every wave looks at all of it)
      __syncthreads();
      if (!odd) return false;
      for (int d = tid; d < KT * U; d += 256)
        *reinterpret_cast<u32x4_t *>(vt + 16 * d) = Odd<F16>::without(*reinterpret_cast<u32x4_t *>(vt + 16 * d));
      __syncthreads();
      return true;
    };
    // one tile in flight; the barrier says that it has landed, and that every wave has left the other stage
    copy(0);
    for (int t = 0; t < ntiles; ++t) {
      wait_vmcnt<0>();
      __syncthreads();
      if (t + 1 < ntiles) copy(t + 1);
      uint8_t *kt = smem + (t & 1) * kStage;
      if (t < plain) {
        tile(kt, t, std::false_type{});
        continue;
      }
      const bool odd = settle(kt + kTile);
      tile(kt, t, std::true_type{});
      if (odd)
        Odd<F16>::restore(acc, vbase + (int64_t)t * KT * vsb + 2 * (kHc * part + 16 * h), vsb, kb + t * KT,
                          min(ke, kb + (t + 1) * KT), row_pos);
    }
  }
  store_row<HS, F16>(p, b, tok, jh, kHc * part + 16 * h, h == 0 && part == 0, m, l + shfl_xor_f(l, 32), acc);
}

// The log-sum-exp merge of split partials, kPer waves per (token, query head) row: the row's splits weighed by
// 2^(m - max m). A wave has its splits' statistics in its lanes and takes 8 splits' channels at a time, all loads issued
// before any is used.
template <int HS, bool F16, int kPer>
__global__ __launch_bounds__(256) void prompt_merge_kernel(const PromptParams p) {
  constexpr int E = HS / 64, kBatch = 8;
  __shared__ float part[kPer > 1 ? (kPer - 1) * HS : 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wr = w % kPer;
  const int64_t row = (int64_t)blockIdx.x * (4 / kPer) + w / kPer;
  const int t = (int)(row / p.num_q_heads), head = (int)(row - (int64_t)t * p.num_q_heads);
  if (t >= p.num_tokens) return;  // (with kPer 4 a workgroup has one row: all of it returns)
  int seq = -1, k0 = 0, k1 = 0;   // the last sequence that starts at or before the token
  for (int s0 = 0; s0 < p.num_seqs; s0 += 63) {
    const int i = min(s0 + lane, p.num_seqs);
    const int cq = p.cu_q[i], ck = p.cu_k[i];
    const uint64_t before = __ballot(s0 + lane < p.num_seqs && lane < 63 && cq <= t);
    if (!before) break;
    const int at = 63 - __builtin_clzll(before);
    seq = t < __builtin_amdgcn_readlane(cq, at + 1) ? s0 + at : -1;
    k0 = __builtin_amdgcn_readlane(ck, at);
    k1 = __builtin_amdgcn_readlane(ck, at + 1);
    if (at < 62) break;
  }
  if (seq < 0) return;  // a row of no sequence: left as it is
  k0 = max(0, k0);
  const int n = max(0, min(k1, p.num_keys) - k0);
  const int seg = segment_keys(n, p.num_splits, p.min_keys);
  const int used = segments_used(n, p.num_splits, seg);
  const float *smax = p.smax + row * p.num_splits, *ssum = p.ssum + row * p.num_splits;
  const float m0 = lane < used ? smax[lane] : kPromptNone, m1 = lane + 64 < used ? smax[lane + 64] : kPromptNone;
  const float l0 = lane < used ? ssum[lane] : 0.f, l1 = lane + 64 < used ? ssum[lane + 64] : 0.f;
  float top = fmaxf(m0, m1);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, shfl_xor_f(top, o));
  const float f0 = __builtin_amdgcn_exp2f(m0 - top), f1 = __builtin_amdgcn_exp2f(m1 - top);
  float sum = fmaf(l0, f0, l1 * f1);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += shfl_xor_f(sum, o);
  const float *so = p.so + row * p.num_splits * HS + E * lane;
  float x[E] = {};
  for (int s0 = wr * kBatch; s0 < used; s0 += kPer * kBatch) {
    float v[kBatch][E];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = min(s0 + i, used - 1);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] = so[(int64_t)s * HS + e];
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = s0 + i;
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s < 64 ? f0 : f1), s & 63));
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (s < used) x[e] = fmaf(v[i][e], f, x[e]);
    }
  }
  if constexpr (kPer > 1) {
    if (wr > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) part[(wr - 1) * HS + E * lane + e] = x[e];
    }
    __syncthreads();
    if (wr > 0) return;
#pragma unroll
    for (int i = 0; i < kPer - 1; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += part[i * HS + E * lane + e];
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  uint16_t *orow = p.out + t * p.os0 + head * p.os1 + E * lane;
  if constexpr (E == 1) {
    *orow = (uint16_t)pack_prompt<F16>(x[0] * inv, 0.f);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(orow + e) = pack_prompt<F16>(x[e] * inv, x[e + 1] * inv);
  }
  if (p.lse && lane == 0)
    p.lse[t * p.ls0 + head * p.ls1] = sum != 0.f ? (top + log2f(sum)) * (1.f / kLog2e) : -INFINITY;
}

// Rows of a workgroup's block.
int prompt_rows(const qp_prompt_args *a) {
  if (a->head_size == 512) return kPromptWideRows;
  if (a->head_size != 128) return 128;
  // Head 128: blocks of 256 rows, which share a tile's copies, where there are two for each CU, or where one wave has all rows
  // and the copies are the work; else two workgroups of 128 rows per CU. 128 against 256 rows, us, 32 / 8 heads: one prompt of
  // 1024 tokens 28 / 34, 2048 53 / 60, 4096 152 / 140, 16384 2030 / 1950; 64 prompts of up to 100, 16 / 16 heads, 28 / 35; one
  // token over 65536 keys, 64 / 8 heads, 75 / 61. (Head 64: 60 in blocks of 128 on four turns of up to 509 tokens over up to
  // 4605 keys, 63 in blocks of 256.)
  const int64_t rows = (int64_t)a->num_tokens * (a->num_q_heads / a->num_kv_heads), seqs = a->num_seqs;
  if (rows <= 32 * seqs) return 256;
  if (rows <= 128 * seqs) return 128;
  return std::max((rows + 255) / 256, seqs) * a->num_kv_heads >= 2 * device_cus() ? 256 : 128;
}

// Workgroups of one key split at most: sequence s owns row blocks [cu_q[s] G / R + s, cu_q[s + 1] G / R + s + 1) of R rows.
int64_t prompt_blocks(const qp_prompt_args *a) {
  return (int64_t)a->num_tokens * (a->num_q_heads / a->num_kv_heads) / prompt_rows(a) + a->num_seqs;
}

// Key splits of a call, of 256 keys at least: 1 where the row blocks alone fill the GPU, else the count with the least
// estimate, in tiles: rounds of workgroups by a split's tiles and the 6 that a workgroup's start and end cost, and the merge
// with its launch and traffic. Measured, us, with one split and the count chosen: a token over 65536 keys, 64 / 8 heads of
// 128, 895 and 52; twice 300 tokens over 9300, 32 / 8 heads, 166 and 119 (3 splits); 2048 tokens alone 53, but 107 with 2
// splits: partials are fp32 and pass through memory.
constexpr int kPromptSplitKeys = 256;

int prompt_splits(const qp_prompt_args *a) {
  if (a->num_splits > 0) return a->num_splits;
  const int64_t cus = device_cus(), G = a->num_q_heads / a->num_kv_heads, rows = prompt_rows(a);
  const int64_t filled = ((int64_t)a->num_tokens * G + rows - 1) / rows;  // (every sequence has a block of its own, too)
  const int64_t wgs = (filled > a->num_seqs ? filled : a->num_seqs) * a->num_kv_heads;
  if (wgs >= cus) return 1;
  const double tiles = a->max_seqlen_k / 64.0, out = (double)a->num_tokens * a->num_q_heads * a->head_size;
  auto cost = [&](int64_t s) {
    return (double)((wgs * s + cus - 1) / cus) * (tiles / s + 6) + (s > 1 ? 6 + out * s * 2e-6 : 0);
  };
  int64_t most = a->max_seqlen_k / kPromptSplitKeys, best = 1;
  if (most > 128) most = 128;
  for (int64_t s = 2; s <= most; ++s)
    if (cost(s) < cost(best)) best = s;
  return (int)best;
}

int64_t prompt_partial_bytes(const qp_prompt_args *a, int splits) {
  if (splits <= 1) return 0;
  return (int64_t)a->num_tokens * a->num_q_heads * splits * (a->head_size + 2) * 4;
}

// Groups of waves that share a block's keys: two where there are up to three blocks for two CUs and 1024 keys or more, us
// with two and with one, 32 / 8 heads of 128 and of 64: 1000 tokens after 8000 155 / 169, 96 / 112, after 2048 58 / 63, 37 /
// 43; four turns of up to 509 tokens over up to 4605 keys 65 / 73, 46 / 50; 600 tokens 20 / 19; 2048 tokens, two blocks per
// CU, 54 / 54, 36 / 33.
int prompt_groups(const PromptParams &p, dim3 grid) {
  return p.group_keys >= 1024 && 2 * (int64_t)grid.x * grid.y <= 3 * (int64_t)device_cus() ? 2 : 1;
}

template <int HS, bool F16>
void launch_prompt(const PromptParams &p, int rows, dim3 grid, hipStream_t s) {
  const uint32_t share = prompt_share(grid.y * grid.z);
  grid.x = ((grid.x + (1u << share) - 1) >> share) << share;
  if constexpr (HS == 512) {
    prompt_wide_kernel<F16><<<grid, 256, 0, s>>>(p);
  } else if constexpr (HS == 256) {
    prompt_kernel<PromptShape<HS, F16, 4>><<<grid, 256, 0, s>>>(p);
  } else if (HS == 128 && rows == 256) {
    if constexpr (HS == 128) prompt_kernel<PromptShape<HS, F16, 8>><<<grid, 512, 0, s>>>(p);
  } else if (prompt_groups(p, grid) == 2) {
    prompt_kernel<PromptShape<HS, F16, 4, 2>><<<grid, 512, 0, s>>>(p);
  } else {
    prompt_kernel<PromptShape<HS, F16, 4>><<<grid, 256, 0, s>>>(p);
  }
  if (p.num_splits > 1) {
    const int64_t out_rows = (int64_t)p.num_tokens * p.num_q_heads;
    if (p.num_splits > 8) prompt_merge_kernel<HS, F16, 4><<<(unsigned)out_rows, 256, 0, s>>>(p);
    else prompt_merge_kernel<HS, F16, 1><<<(unsigned)((out_rows + 3) / 4), 256, 0, s>>>(p);
  }
}

template <int HS>
void launch_prompt_type(const PromptParams &p, int dtype, int rows, dim3 grid, hipStream_t s) {
  if (dtype == QP_DTYPE_F16) launch_prompt<HS, true>(p, rows, grid, s);
  else launch_prompt<HS, false>(p, rows, grid, s);
}

// What a call refuses.
int check_prompt(const qp_prompt_args *a) {
  QP_REQUIRE(a, "qp_prompt: null argument");
  QP_REQUIRE(a->num_seqs >= 0 && a->num_tokens >= 0 && a->num_keys >= 0 && a->max_seqlen_k >= 0, "qp_prompt: bad sizes");
  QP_SUPPORTED(a->head_size == 64 || a->head_size == 128 || a->head_size == 256 || a->head_size == 512,
               "qp_prompt: head size must be 64, 128, 256 or 512");
  QP_SUPPORTED(a->dtype == QP_DTYPE_BF16 || a->dtype == QP_DTYPE_F16, "qp_prompt: bf16 or fp16 tensors");
  QP_REQUIRE(a->num_kv_heads > 0 && a->num_q_heads > 0 && a->num_q_heads % a->num_kv_heads == 0,
             "qp_prompt: query heads must be a multiple of KV heads");
  QP_REQUIRE(a->num_splits >= 0 && a->num_splits <= 128, "qp_prompt: 0..128 splits");
  QP_REQUIRE(a->softmax_scale > 0.f && a->softmax_scale < INFINITY, "qp_prompt: the softmax scale must be positive");
  const int64_t rows = (int64_t)a->num_tokens * a->num_q_heads;  // (the merge has up to 256 threads for each)
  QP_SUPPORTED(rows < (int64_t(1) << 31) && a->num_kv_heads < 65536, "qp_prompt: too many rows");
  QP_SUPPORTED(a->num_splits <= 1 || rows < (int64_t(1) << 24), "qp_prompt: too many rows for splits");
  return QP_OK;
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_prompt_workspace_size(const qp_prompt_args *a) {
  if (check_prompt(a) != QP_OK || a->num_seqs == 0 || a->num_tokens == 0) return 0;
  return prompt_partial_bytes(a, prompt_splits(a));
}

extern "C" int qp_prompt(const qp_prompt_args *a, qp_stream_t stream) {
  const int st = check_prompt(a);
  if (st != QP_OK) return st;
  if (a->num_seqs == 0 || a->num_tokens == 0) return QP_OK;
  QP_REQUIRE(a->query && a->out && a->cu_seqlens_q && a->cu_seqlens_k, "qp_prompt: null tensor");
  QP_REQUIRE(a->num_keys == 0 || (a->key && a->value), "qp_prompt: null tensor");
  const int64_t *strides[] = {a->query_stride, a->key_stride, a->value_stride, a->out_stride};
  const void *tensors[] = {a->query, a->key, a->value, a->out};
  for (int i = 0; i < 4; ++i) {
    QP_REQUIRE(aligned(tensors[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0,
               "qp_prompt: rows must be 16-byte aligned");
    QP_REQUIRE(strides[i][0] >= 0 && strides[i][1] >= 0, "qp_prompt: strides must not be negative");
  }
  // (the lanes of a tile's copies reach its rows by 32-bit offsets)
  QP_SUPPORTED(a->key_stride[0] < (1 << 23) && a->value_stride[0] < (1 << 23), "qp_prompt: key rows more than 16 MiB apart");
  const int64_t rows = (int64_t)a->num_tokens * a->num_q_heads, group = a->num_q_heads / a->num_kv_heads;
  const int64_t blocks = prompt_blocks(a);
  int splits = prompt_splits(a);
  if (splits > 1 && (!a->workspace || a->workspace_bytes < prompt_partial_bytes(a, splits))) {
    QP_REQUIRE(a->num_splits == 0, "qp_prompt: workspace too small for the requested splits");
    splits = 1;  // without a workspace the keys of a row block are walked by one workgroup
  }
  QP_REQUIRE(splits == 1 || aligned(a->workspace, 16), "qp_prompt: workspace must be 16-byte aligned");
  PromptParams p;
  p.q = static_cast<const uint16_t *>(a->query);
  p.qs0 = a->query_stride[0];
  p.qs1 = a->query_stride[1];
  p.k = static_cast<const uint16_t *>(a->key);
  p.ks0 = a->key_stride[0];
  p.ks1 = a->key_stride[1];
  p.v = static_cast<const uint16_t *>(a->value);
  p.vs0 = a->value_stride[0];
  p.vs1 = a->value_stride[1];
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.out = static_cast<uint16_t *>(a->out);
  p.os0 = a->out_stride[0];
  p.os1 = a->out_stride[1];
  p.lse = a->lse;
  p.ls0 = a->lse_stride[0];
  p.ls1 = a->lse_stride[1];
  p.so = splits > 1 ? static_cast<float *>(a->workspace) : nullptr;
  p.smax = splits > 1 ? p.so + rows * splits * a->head_size : nullptr;
  p.ssum = splits > 1 ? p.smax + rows * splits : nullptr;
  p.num_seqs = a->num_seqs;
  p.num_tokens = a->num_tokens;
  p.num_keys = a->num_keys;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.num_splits = splits;
  p.min_keys = a->num_splits == 0 ? kPromptSplitKeys : 0;
  p.causal = a->causal != 0;
  p.group_keys = a->num_splits == 0 && splits == 1 ? a->max_seqlen_k : 0;
  // A few sequences whose blocks take turns: longest first, which costs a workgroup 0.1 us and as much for every two sequences.
  // In order of length against order of place, us: four turns of up to 509 tokens over up to 4605 keys, 32 / 8 heads of 64,
  // 48 / 61, of 128 72 / 88; prompts of up to 2048 tokens, heads of 128, 3 of them 67 / 71, 8 152 / 154 and 85 / 86; 12 of up
  // to 1500 105 / 104; 64 of up to 100 32 / 27.
  // (Its products of keys and group, of 64 steps or of any sequence, stay below 2^31; max_seqlen_k may say less than there is.)
  const int64_t longest = std::max({a->max_seqlen_k, a->num_keys, a->num_tokens, 64 * 64});
  const bool by_length = p.causal && splits == 1 && a->num_seqs > 1 && a->num_seqs <= 8 &&
                         blocks * a->num_kv_heads > device_cus() && longest * group < (1 << 29);
  p.step = by_length ? std::max(64, a->max_seqlen_k / 63) : 0;
  p.scale_log2 = a->softmax_scale * kLog2e;
  const int block_rows = prompt_rows(a);
  const dim3 grid((unsigned)blocks, a->num_kv_heads, splits);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->head_size == 64) launch_prompt_type<64>(p, a->dtype, block_rows, grid, s);
  else if (a->head_size == 128) launch_prompt_type<128>(p, a->dtype, block_rows, grid, s);
  else if (a->head_size == 256) launch_prompt_type<256>(p, a->dtype, block_rows, grid, s);
  else launch_prompt_type<512>(p, a->dtype, block_rows, grid, s);
  return launch_status();
}
