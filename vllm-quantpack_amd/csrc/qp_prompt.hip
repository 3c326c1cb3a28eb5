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
// lie in memory, two tiles ahead of their use; the V^T operand comes from the LDS's transposing reads (ds_read_b64_tr_b16).
#include "qp_common.h"
#include "quantpack_ops.h"

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
  float scale_log2;
};

constexpr float kPromptNone = -1e30f;  // a row's maximum before it has seen a key
// A row's maximum m is raised when a score exceeds it by more than this (log2 units): probabilities stay below 2^8, well
// within fp16, whose smallest normal number is then 2^-22 of the largest probability.
constexpr float kPromptHeadroom = 8.f;

template <int HS_, bool F16_>
struct PromptShape {
  static constexpr int HS = HS_;
  static constexpr bool F16 = F16_;
  static constexpr int kWaves = HS <= 128 ? 8 : 4;   // two waves per SIMD, or one where a row tile takes over 256 registers
  // Waves that share a row tile, each with its part of the channels of q, K, V and the accumulators. At head 512 (where
  // they would take 384 registers) two: each makes the scores of its channels, and the two parts are added through LDS.
  static constexpr int kParts = HS == 512 ? 2 : 1;
  static constexpr int kChannels = HS / kParts;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int kRt = 1;                      // 32-row tiles per wave
  static constexpr int kRows = kWaves / kParts * kRt * 32;
  static constexpr int kKeys = HS == 512 ? 32 : 64;  // keys per tile
  static constexpr int kStages = HS <= 128 ? 3 : 2;
  static constexpr int kU = HS / 8;                  // 16-byte units of a row
  static constexpr int kHalf = kKeys * HS * 2;       // bytes of a tile's K (and of its V)
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kScores = kStages * kStage;   // parts of the scores, 4 KiB per wave; or the word of a vote
  static constexpr int kLds = kScores + (kParts > 1 ? kWaves * 4096 : 16);
  static constexpr int kCopies = kHalf / 1024 / kWaves;  // 1 KiB copies of a wave, K and V each
  static_assert(kHalf % (1024 * kWaves) == 0 && kLds <= 160 * 1024, "LDS");
  // Position of unit c in row r of a K tile: 16 rows' reads of one unit hit every bank of the LDS once.
  static __host__ __device__ constexpr int k_swz(int r, int c) { return HS == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); }
  // The same in a V tile, in blocks of four units (32 channels, what a transposing read takes of a row): the four rows of
  // a 16-lane group hit different banks. At head 64 a row has two blocks, and two rows every bank.
  static __host__ __device__ constexpr int v_swz(int r, int c) {
    return HS == 64 ? c ^ (((r >> 1) & 1) << 2) : c ^ ((r & 3) << 2);
  }
};

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

template <class Sh>
__global__ __launch_bounds__(Sh::kThreads) void prompt_kernel(const PromptParams p) {
  constexpr int HS = Sh::HS, KT = Sh::kKeys, RT = Sh::kRt, U = Sh::kU;
  constexpr bool F16 = Sh::F16;
  constexpr int kParts = Sh::kParts, kHc = Sh::kChannels;
  constexpr int kCs = kHc / 16, kCt = kHc / 32, kSubs = KT / 32;
  static_assert(kParts == 1 || (RT == 1 && kSubs == 1 && kParts == 2), "parts of the scores");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Sh::kLds];

  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int part = w % kParts;
  const int blk = (int)gridDim.x - 1 - (int)blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads;
  // row block -> sequence: sequence s's rows own blocks [cu_q[s] G / kRows + s, ...)
  int lo = 0, hi = p.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int)(((int64_t)p.cu_q[mid] * G) / Sh::kRows) + mid <= blk) lo = mid;
    else hi = mid - 1;
  }
  const int seq = lo;
  const int q0 = max(0, p.cu_q[seq]), qlen = min(p.cu_q[seq + 1], p.num_tokens) - q0;
  const int k0 = max(0, p.cu_k[seq]), n = max(0, min(p.cu_k[seq + 1], p.num_keys) - k0);
  const int nrows = qlen * G;
  const int r0 = (blk - (int)(((int64_t)q0 * G) / Sh::kRows) - seq) * Sh::kRows;
  if (r0 < 0 || r0 >= nrows) return;
  // the last position that a token sees, first and last token of the block
  auto last_pos = [&](int tok) { return p.causal ? n - qlen + tok : n - 1; };
  const int kend = max(0, min(n, last_pos((min(nrows, r0 + Sh::kRows) - 1) / G) + 1));
  const int S = p.num_splits;
  const int seg = segment_keys(n, S, p.min_keys);
  const int64_t kb64 = (int64_t)split * seg;
  if (S > 1 && kb64 >= n) return;  // an empty segment: the merge does not read it
  const int kb = (int)kb64;
  const int ke = uniform(min((int64_t)kend, kb64 + seg));

  // ---- the wave's rows: lane row col of tile rt -> (token rr / G, query head rr % G)
  const int wrow = r0 + 32 * RT * (w / kParts);
  const bool active = wrow < nrows;
  int row_pos[RT], tok[RT], jh[RT];
  u32x4_t qop[RT][kCs];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int rr = wrow + 32 * rt + col;
    const bool valid = rr < nrows;
    tok[rt] = valid ? rr / G : -1;
    jh[rt] = valid ? rr - tok[rt] * G : 0;
    row_pos[rt] = valid ? last_pos(tok[rt]) : -1;
    const uint16_t *src = p.q + (int64_t)(q0 + max(0, tok[rt])) * p.qs0 + (int64_t)(kvh * G + jh[rt]) * p.qs1 + kHc * part + 8 * h;
#pragma unroll
    for (int cs = 0; cs < kCs; ++cs)
      qop[rt][cs] = valid ? *reinterpret_cast<const u32x4_t *>(src + 16 * cs) : u32x4_t{0u, 0u, 0u, 0u};
  }
  f32x16_t acc[RT][kCt];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = kPromptNone;
    l[rt] = 0.f;
#pragma unroll
    for (int ct = 0; ct < kCt; ++ct) acc[rt][ct] = f32x16_t{};
  }

  const int ntiles = ke > kb ? (ke - kb + KT - 1) / KT : 0;
  if (ntiles > 0) {
    // tiles whose keys every row of the block (of the wave) sees, and tiles that some row of the wave sees
    auto plain_tiles = [&](int row) { return max(0, min(last_pos(row / G) + 1, ke) - kb) / KT; };
    // (waves that share scores meet at barriers in a tile, so there the block goes by its own bounds)
    const int bplain = uniform(plain_tiles(r0));
    const int wlast = last_pos((min(nrows, wrow + 32 * RT) - 1) / G);
    const int wplain = kParts > 1 ? bplain : uniform(active ? plain_tiles(wrow) : 0);
    const int wend = kParts > 1 ? ntiles : uniform(active ? (max(0, min(ke, wlast + 1) - kb) + KT - 1) / KT : 0);

    // ---- HBM -> LDS: copy i of a wave fills 16-byte units 64 (w + kWaves i) .. of the tile, lane by lane; the unit's row
    // and column are those that the swizzle puts there
    const uint32_t lds0 = lds_addr(smem);
    const uint8_t *kbase = reinterpret_cast<const uint8_t *>(p.k + (int64_t)(k0 + kb) * p.ks0 + (int64_t)kvh * p.ks1);
    const uint8_t *vbase = reinterpret_cast<const uint8_t *>(p.v + (int64_t)(k0 + kb) * p.vs0 + (int64_t)kvh * p.vs1);
    const uint32_t ksb = (uint32_t)(p.ks0 * 2), vsb = (uint32_t)(p.vs0 * 2);
    auto copy = [&](int t, int stage) {
      const int left = ke - kb - t * KT - 1;  // the tile's last key (rows past it repeat it: always mapped memory)
      const uint8_t *kt = kbase + (int64_t)t * KT * ksb, *vt = vbase + (int64_t)t * KT * vsb;
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i) {
        const int at = 64 * (w + Sh::kWaves * i), d = at + lane;
        const int r = d / U, c = d % U, rs = min(r, left);
        const uint32_t dst = lds0 + (uint32_t)(stage * Sh::kStage + 16 * at);
        dma16_saddr<false>(kt, (uint32_t)rs * ksb + 16u * (uint32_t)Sh::k_swz(r, c), dst);
        dma16_saddr<false>(vt, (uint32_t)rs * vsb + 16u * (uint32_t)Sh::v_swz(r, c), dst + Sh::kHalf);
      }
    };
    // ---- operands. K: row 32 u + col, unit 2 cs + h. V^T: A row 8 q + 4 hh + j of channel tile ct is channel
    // 32 ct + 16 hh + 4 q + j, so that a lane's accumulators are 16 consecutive channels; the four 4-channel chunks that a
    // 16-lane group's rows take are then 16 (c & 1) + 4 (c >> 1), and 8 more for the upper group.
    // A swizzle changes the low bits of a unit's place only: a few lane offsets serve all steps, with the rest immediate.
    constexpr int kKo = kCs < 8 ? kCs : 8, kVo = kCt < 4 ? kCt : 4;
    uint32_t koff[kKo], voff[kVo];
#pragma unroll
    for (int i = 0; i < kKo; ++i) koff[i] = col * (2 * HS) + 16 * (Sh::k_swz(col, 2 * i + h) + (kHc / 8) * part);
    const int vrow = 4 * h + ((lane >> 2) & 3);
    const int vch = 16 * (lane & 1) + 4 * ((lane >> 1) & 1) + 8 * ((lane >> 4) & 1);
#pragma unroll
    for (int i = 0; i < kVo; ++i)
      voff[i] = vrow * (2 * HS) + 16 * (Sh::v_swz(vrow, 4 * i) + (kHc / 8) * part + (vch >> 3)) + 2 * (vch & 7);
    auto k_op = [&](const uint8_t *kt, int u, int cs) {
      return *reinterpret_cast<const u32x4_t *>(kt + koff[cs % kKo] + 32 * u * (2 * HS) + 256 * (cs / kKo));
    };
    auto v_op = [&](const uint8_t *vt, int ks, int ct) {
      u32x4_t r;
#pragma unroll
      for (int eight = 0; eight < 2; ++eight) {
        const uint8_t *at = vt + voff[ct % kVo] + (16 * ks + 8 * eight) * (2 * HS) + 256 * (ct / kVo);
        const i16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4_t *)(const __attribute__((address_space(3))) uint8_t *)at);
        const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
        r[2 * eight] = y[0];
        r[2 * eight + 1] = y[1];
      }
      return r;
    };

    auto tile = [&](const uint8_t *kt, int t, auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      const uint8_t *vt = kt + Sh::kHalf;
      f32x16_t s[RT][kSubs];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < kSubs; ++u) s[rt][u] = f32x16_t{};
#pragma unroll
      for (int cs = 0; cs < kCs; ++cs)
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
          const u32x4_t kop = k_op(kt, u, cs);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][u] = mfma_prompt<F16>(kop, qop[rt][cs], s[rt][u]);
        }
      if constexpr (kParts > 1) {
        f32x4_t *own = reinterpret_cast<f32x4_t *>(smem + Sh::kScores + 4096 * w) + lane;
        const f32x4_t *other = reinterpret_cast<const f32x4_t *>(smem + Sh::kScores + 4096 * (w ^ 1)) + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          own[64 * i] = f32x4_t{s[0][0][4 * i], s[0][0][4 * i + 1], s[0][0][4 * i + 2], s[0][0][4 * i + 3]};
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4_t x = other[64 * i];
#pragma unroll
          for (int j = 0; j < 4; ++j) s[0][0][4 * i + j] += x[j];  // (the same sum in both waves)
        }
      }
      u32x4_t pop[RT][2 * kSubs];
      float top[RT];
      bool raise = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if constexpr (MASK) {
              const int key = kb + t * KT + 32 * u + 8 * (i >> 2) + 4 * h + (i & 3);
              if (key > row_pos[rt] || key >= ke) s[rt][u][i] = -INFINITY;
            }
            x = fmaxf(x, s[rt][u][i]);
          }
        top[rt] = x * p.scale_log2;
        raise |= top[rt] > m[rt] + kPromptHeadroom;
      }
      if (__any(raise)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float most = other_half_max(top[rt]);
          const float to = most > m[rt] + kPromptHeadroom ? most : m[rt];  // (a row's bits do not go by its neighbours)
          const float alpha = __builtin_amdgcn_exp2f(m[rt] - to);
          m[rt] = to;
          l[rt] *= alpha;
#pragma unroll
          for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[rt][ct][i] *= alpha;
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[rt][u][2 * i], p.scale_log2, -m[rt]));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[rt][u][2 * i + 1], p.scale_log2, -m[rt]));
            l[rt] += p0 + p1;  // (unrounded: the log-sum-exp is kept to fp32)
            pop[rt][2 * u + (i >> 2)][i & 3] = pack_prompt<F16>(p0, p1);
          }
#pragma unroll
      for (int ks = 0; ks < 2 * kSubs; ++ks)
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
          const u32x4_t vop = v_op(vt, ks, ct);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][ct] = mfma_prompt<F16>(vop, pop[rt][ks], acc[rt][ct]);
        }
    };

    // ---- infinities and NaN in V of a tile that some row does not see whole. Such a row's probability is 0, and the MFMA
    // would make NaN of it: the tile gets zeros in their place (settle), and the rows that see the key the value itself
    // afterwards, read from memory again (restore): any probability is above 0.
    constexpr uint32_t kInf = F16 ? 0x7C00u : 0x7F80u;
    auto odd = [&](uint32_t x) { return ((x & kInf) == kInf) || ((x & (kInf << 16)) == kInf << 16); };
    auto settle = [&](uint8_t *vt) {
      uint32_t *vote = reinterpret_cast<uint32_t *>(smem + Sh::kScores);
      bool any = false;
      for (int d = tid; d < KT * U; d += Sh::kThreads) {
        const u32x4_t x = *reinterpret_cast<const u32x4_t *>(vt + 16 * d);
        any |= odd(x[0]) || odd(x[1]) || odd(x[2]) || odd(x[3]);
      }
      if (tid == 0) *vote = 0;
      __syncthreads();
      if (any) *vote = 1;
      __syncthreads();
      any = *vote != 0;
      if constexpr (kParts > 1) __syncthreads();  // (the word lies where the next scores go)
      if (!any) return false;
      for (int d = tid; d < KT * U; d += Sh::kThreads) {
        u32x4_t x = *reinterpret_cast<const u32x4_t *>(vt + 16 * d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((x[j] & kInf) == kInf) x[j] &= 0xFFFF0000u;
          if ((x[j] & (kInf << 16)) == kInf << 16) x[j] &= 0xFFFFu;
        }
        *reinterpret_cast<u32x4_t *>(vt + 16 * d) = x;
      }
      __syncthreads();
      return true;
    };
    auto restore = [&](int t) {
      for (int key = kb + t * KT; key < min(ke, kb + (t + 1) * KT); ++key) {
        const uint8_t *row = vbase + (int64_t)(key - kb) * vsb + 2 * (kHc * part + 16 * h);
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
          const u32x4_t y[2] = {*reinterpret_cast<const u32x4_t *>(row + 64 * ct),
                                *reinterpret_cast<const u32x4_t *>(row + 64 * ct + 16)};
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint16_t x = (uint16_t)(y[i >> 3][(i >> 1) & 3] >> (16 * (i & 1)));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              if ((x & kInf) == kInf && key <= row_pos[rt]) acc[rt][ct][i] += from_bits<F16>(x);
          }
        }
      }
    };

    // ---- the walk: kStages - 1 tiles in flight; each iteration waits for its own, and the barrier after that also says
    // that every wave has left the stage which the next copy fills
    constexpr int kAhead = Sh::kStages - 1;
#pragma unroll
    for (int t = 0; t < kAhead; ++t)
      if (t < ntiles) copy(t, t);
    int stage = 0;
    for (int t = 0; t < ntiles; ++t) {
      if (kAhead == 1 || t + 1 >= ntiles) wait_vmcnt<0>();
      else wait_vmcnt<2 * Sh::kCopies>();
      __syncthreads();
      const int into = stage == 0 ? Sh::kStages - 1 : stage - 1;
      if (t + kAhead < ntiles) copy(t + kAhead, into);
      uint8_t *kt = smem + stage * Sh::kStage;
      const bool odd_values = t >= bplain && settle(kt + Sh::kHalf);
      if (t < wplain) tile(kt, t, std::false_type{});
      else if (t < wend) tile(kt, t, std::true_type{});
      if (odd_values && active) restore(t);
      stage = stage + 1 == Sh::kStages ? 0 : stage + 1;
    }
  }

  // ---- epilogue: a lane's 16 consecutive channels of each channel tile
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = l[rt] + shfl_xor_f(l[rt], 32);
    if (tok[rt] < 0) continue;
    const int64_t t = q0 + tok[rt], head = kvh * G + jh[rt];
    if (S == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;  // (a sum that is no number stays none)
      uint16_t *orow = p.out + t * p.os0 + head * p.os1 + kHc * part + 16 * h;
#pragma unroll
      for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u32x4_t y;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[j] = pack_prompt<F16>(acc[rt][ct][8 * i + 2 * j] * inv, acc[rt][ct][8 * i + 2 * j + 1] * inv);
          *reinterpret_cast<u32x4_t *>(orow + 32 * ct + 8 * i) = y;
        }
      if (p.lse && h == 0 && part == 0)
        p.lse[t * p.ls0 + head * p.ls1] = sum != 0.f ? (m[rt] + log2f(sum)) * (1.f / kLog2e) : -INFINITY;
    } else {
      const int64_t at = (t * p.num_q_heads + head) * S + split;
      float *orow = p.so + at * HS + kHc * part + 16 * h;
#pragma unroll
      for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4 *>(orow + 32 * ct + i) =
              make_float4(acc[rt][ct][i], acc[rt][ct][i + 1], acc[rt][ct][i + 2], acc[rt][ct][i + 3]);
      if (h == 0 && part == 0) {
        p.smax[at] = m[rt];
        p.ssum[at] = sum;
      }
    }
  }
}

// The log-sum-exp merge of split partials, a wave per (token, query head) row: the row's splits weighed by 2^(m - max m).
template <int HS, bool F16>
__global__ __launch_bounds__(256) void prompt_merge_kernel(const PromptParams p) {
  constexpr int E = HS / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t t = row / p.num_q_heads, head = row - t * p.num_q_heads;
  if (t >= p.num_tokens) return;
  int lo = 0, hi = p.num_seqs - 1;  // the last sequence that starts at or before the token
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_q[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  if (t < p.cu_q[lo] || t >= p.cu_q[lo + 1]) return;  // a row of no sequence: left as it is
  const int k0 = max(0, p.cu_k[lo]), n = max(0, min(p.cu_k[lo + 1], p.num_keys) - k0);
  const int seg = segment_keys(n, p.num_splits, p.min_keys);
  const int used = min(p.num_splits, (int)(((int64_t)n + seg - 1) / seg));
  const float *smax = p.smax + row * p.num_splits, *ssum = p.ssum + row * p.num_splits;
  const float *so = p.so + row * p.num_splits * HS + E * lane;
  float top = kPromptNone;
  for (int s = 0; s < used; ++s) top = fmaxf(top, smax[s]);
  float sum = 0.f, x[E] = {};
  for (int s = 0; s < used; ++s) {
    const float f = __builtin_amdgcn_exp2f(smax[s] - top);
    sum = fmaf(ssum[s], f, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaf(so[(int64_t)s * HS + e], f, x[e]);
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

template <int HS>
constexpr int prompt_rows() { return PromptShape<HS, false>::kRows; }

int prompt_block_rows(int hs) {
  return hs == 64 ? prompt_rows<64>() : hs == 128 ? prompt_rows<128>() : hs == 256 ? prompt_rows<256>() : prompt_rows<512>();
}

// Workgroups of one key split at most: sequence s owns row blocks [cu_q[s] G / R + s, cu_q[s + 1] G / R + s + 1) of R rows.
int64_t prompt_blocks(const qp_prompt_args *a) {
  return (int64_t)a->num_tokens * (a->num_q_heads / a->num_kv_heads) / prompt_block_rows(a->head_size) + a->num_seqs;
}

// Key splits of a call: 1 where the row blocks alone fill the GPU, else about two workgroups per CU, of 256 keys at least.
constexpr int kPromptSplitKeys = 256;

int prompt_splits(const qp_prompt_args *a) {
  if (a->num_splits > 0) return a->num_splits;
  const int64_t wgs = prompt_blocks(a) * a->num_kv_heads, cus = device_cus();
  if (wgs >= cus) return 1;
  int64_t s = (2 * cus + wgs - 1) / wgs;
  const int64_t most = a->max_seqlen_k / kPromptSplitKeys;
  if (s > most) s = most;
  return s < 1 ? 1 : s > 128 ? 128 : (int)s;
}

int64_t prompt_partial_bytes(const qp_prompt_args *a, int splits) {
  if (splits <= 1) return 0;
  return (int64_t)a->num_tokens * a->num_q_heads * splits * (a->head_size + 2) * 4;
}

template <int HS, bool F16>
void launch_prompt(const PromptParams &p, dim3 grid, hipStream_t s) {
  using Sh = PromptShape<HS, F16>;
  prompt_kernel<Sh><<<grid, Sh::kThreads, 0, s>>>(p);
  if (p.num_splits > 1) {
    const int64_t rows = (int64_t)p.num_tokens * p.num_q_heads;
    prompt_merge_kernel<HS, F16><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(p);
  }
}

template <int HS>
void launch_prompt_type(const PromptParams &p, int dtype, dim3 grid, hipStream_t s) {
  if (dtype == QP_DTYPE_F16) launch_prompt<HS, true>(p, grid, s);
  else launch_prompt<HS, false>(p, grid, s);
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
  const int64_t rows = (int64_t)a->num_tokens * a->num_q_heads;
  const int64_t blocks = prompt_blocks(a);
  QP_SUPPORTED(rows < (int64_t(1) << 31) && a->num_kv_heads < 65536, "qp_prompt: too many rows");
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
  p.scale_log2 = a->softmax_scale * kLog2e;
  const dim3 grid((unsigned)blocks, a->num_kv_heads, splits);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->head_size == 64) launch_prompt_type<64>(p, a->dtype, grid, s);
  else if (a->head_size == 128) launch_prompt_type<128>(p, a->dtype, grid, s);
  else if (a->head_size == 256) launch_prompt_type<256>(p, a->dtype, grid, s);
  else launch_prompt_type<512>(p, a->dtype, grid, s);
  return launch_status();
}
