// Attention of a few queries over a key / value cache held in 4 bits (layout: kv4.hip), gfx950.
//
//   S = (q . k + edge) / temperature,  O = sum_j softmax(S)_j v_j,  k = s_k n + m_k, v = s_v n + m_v
//
// with codes n = 0 .. 15 and a scale s and minimum m per token and 64 channels.  Scale and minimum
// leave the products:
//   q . k = s_k (q . n) + m_k sum(q)
//   sum_j p_j v_j = sum_j (p_j s_v) n + sum_j p_j m_v
// so both products run on the bf16 matrix cores with the codes as exact operands: a code becomes
// the bf16 number 16 + n by a shift and an and-or for two (its bits are the top mantissa bits of
// 16 .. 32); the 16 comes off in the epilogue, q . n = q . (16 + n) - 16 sum(q).
//
// Roundings: bf16 queries are exact operands, float32 ones are split into three bf16 parts; p s_v
// is split into two (bf16 tensors: 16 bits; 23.5 times the same parts comes off the sum, so that what
// they lose is weighted by n - 7.5 and not by 16 + n: 6e-6 of a result of many tokens, where a bf16
// rounding 2e-3) or three parts (float32: all 24 bits).  For float32 23.5 = 16 + 7.5 is taken off
// inside the matrix products, every 32 channels or tokens: their accumulators start with the largest
// part's product with a constant operand, so that the sums that are rounded are of q (n - 7.5), not
// of q (16 + n), which are 5 times as large and in a long average over tokens many times.  What that
// start was rounded by is the same product once more, minus the start; it joins the lower parts,
// which have sums of their own.  (Root of the mean square against 64 bits 4e-7 of the result for 777
// tokens; with the start rounded 1.2e-6; a float32 attention over the dequantised cache 6e-7.)
//
// Work: a wave takes tiles of TT = 128 (head dim 64) or 64 tokens, 8 KB of codes, on its own, with
// its own running maximum; four waves of a workgroup and, for few heads, several workgroups
// (`splits`, joined by kv4_join_kernel) share a sequence.
//   S^T = K Q^T: operand A = 16 cached tokens as they lie in memory, operand B = 16 query rows.
//   O^T = V^T P^T: operand A = 16 channels x 32 tokens, again as they lie in memory.
// The rows of K are taken in an order in which a lane's part of S^T is its part of operand B of the
// second product, so that with 5 to 16 query rows (R = 16) the softmax runs where the scores are.
// With fewer rows (one, in plain decoding) most columns of S^T are idle; the scores then go through
// LDS, where the wave spreads the R = 1, 2 or 4 rows over its 64 lanes: the softmax costs 2 R
// evaluations a lane and 128 tokens instead of 32.
// The running maximum moves only when a score exceeds it by 8 (exp(8) is harmless in float32):
// noticing that is one vote, the reduction over lanes is the exception.
// The next tile's K codes are requested when this one's scores are done, its V codes when this
// one's products are: a code is dequantised out of the register that it was loaded into.
//
// Bound by memory: 72 bytes a token and cached head at head dim 64 (256 in bf16).  bf16, 64 x 16
// heads x 1024 tokens, one query: 18 us (75 MB, 4.1 TB/s; a large copy reaches 4.95); 8 x 8 heads of
// 4 queries x 32768 tokens at head dim 128: 59 us and 5 for the join (265 MB, 4.5 TB/s).  Short calls
// are bound by the chain of loads: 40 tokens of one sentence's 8 heads 6.5 us, an empty kernel 2.5.
#include "common.h"
#include "kernels.h"

namespace gnlp {
namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

__device__ __forceinline__ void wave_lds_sync() {   // order a wave's LDS writes before its reads
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// 8 codes -> 8 bf16 numbers 16 + n (nibble i and i + 4 are elements 2 i and 2 i + 1)
__device__ __forceinline__ bf16x8 codes16(uint32_t w) {
  u32x4 r;
  r[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
  r[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
  r[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
  r[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
  return __builtin_bit_cast(bf16x8, r);
}

__device__ __forceinline__ float scale_of(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float min_of(uint32_t w) {
  return __builtin_bit_cast(float, w & 0xffff0000u);
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 all4(float x) { return (f32x4){x, x, x, x}; }

// base: the same in all lanes
template <typename V>
__device__ __forceinline__ V load_at(const void *base, uint32_t off) {
  return *reinterpret_cast<const V *>((const char *)base + off);
}

// x = the sum of its bf16 parts, the last one rounded
template <int N>
__device__ __forceinline__ void split(float x, bf16 (&part)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    part[k] = (bf16)x;
    x -= (float)part[k];
  }
}

// Waves a SIMD that the registers are cut for, nothing spilled (bf16 / 64 / R = 1, float32 / 64 / R = 1
// and float32 / 128 / R = 4, all with a bias, come out with room for one more).
constexpr int waves_of(bool f32, int DP, int R, bool bias) {
  if (R <= 4 && f32) return DP == 64 ? (R == 1 && !bias ? 3 : 2) : (R == 4 && bias ? 1 : 2);
  if (R <= 4) return DP == 64 && !bias ? 4 : 3;
  return f32 ? (bias ? 1 : 2) : (bias ? 2 : 3);
}

// BIAS: edge_scores, edge_table or mask given
template <typename T, int DP, int R, bool BIAS>
__global__ void __launch_bounds__(256, waves_of(sizeof(T) == 4, DP, R, BIAS))
kv4_attn_kernel(Kv4Attn a) {
  constexpr int G = DP / 64;             // groups of a token
  constexpr int TT = 128 / G;            // tokens of a tile
  constexpr int NSUB = TT / 32;
  constexpr bool DIRECT = R == 16;       // softmax in the layout of the scores
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int QS = F32 ? 3 : 1;        // bf16 parts of a query value
  constexpr int PS = F32 ? 3 : 2;        // bf16 parts of p s_v
  constexpr int LPR = DIRECT ? 4 : 64 / R;        // lanes of a row in the softmax
  constexpr int TPL = TT / LPR;          // tokens of a lane there
  constexpr int VW = TPL < 4 ? TPL : 4;  // ... in vectors of
  constexpr int NV = TPL / VW;
  constexpr int NP = TT / 64;            // tokens whose parameters a lane fetches
  constexpr bool OWN_PAR = R == 1;       // ... which are the ones that it evaluates
  constexpr int SROW = TT + 4, PROW = TT + 8;
  constexpr float NEG = -__builtin_inff();
  constexpr float LOG2E = 1.4426950408889634f;
  // scores in units of log2 where no bias of the type's lowest number can overflow them
  constexpr float STEP = BIAS ? 8.0f : 8.0f * LOG2E, UNIT = BIAS ? LOG2E : 1.f;
  constexpr int KROW = DP / 2, VROW = DP * 4;     // bytes of a token's K, of 8 tokens' V

  // per wave: scores (G, R, SROW) float, P (G, PS, R, PROW) bf16, parameters (2, G, TT), alpha (R)
  constexpr int S_BYTES = DIRECT ? 0 : G * R * SROW * 4;
  constexpr int P_BYTES = DIRECT ? 0 : G * PS * R * PROW * 2;
  constexpr int PAR_BYTES = OWN_PAR ? 0 : 2 * G * TT * 4;
  constexpr int WAVE_BYTES = (S_BYTES + P_BYTES + PAR_BYTES + 2 * 16 * 4 + 15) / 16 * 16;
  constexpr int OROW = DP + 4;
  constexpr int OUT_BYTES = 4 * R * (OROW + 2 + G) * 4;
  __shared__ __attribute__((aligned(16)))
      unsigned char smem[4 * WAVE_BYTES > OUT_BYTES ? 4 * WAVE_BYTES : OUT_BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  unsigned char *mine = smem + wave * WAVE_BYTES;
  float *sc = (float *)mine;
  bf16 *pr = (bf16 *)(mine + S_BYTES);
  uint32_t *parl = (uint32_t *)(mine + S_BYTES + P_BYTES);
  float *al = (float *)(mine + S_BYTES + P_BYTES + PAR_BYTES);

  // ---- which rows, which tokens ----
  uint32_t lin = blockIdx.x;
  const uint32_t rt = a.row_tiles == 1 ? 0 : lin % (uint32_t)a.row_tiles;
  if (a.row_tiles > 1) lin /= (uint32_t)a.row_tiles;
  const uint32_t split_no = a.splits == 1 ? 0 : lin % (uint32_t)a.splits;
  if (a.splits > 1) lin /= (uint32_t)a.splits;
  const int b = (int)(lin / (uint32_t)a.H), h = (int)(lin - (uint32_t)b * (uint32_t)a.H);
  const int Lq = (int)a.Lq, S = (int)a.S, row0 = (int)rt * 16;
  const int rows = Lq * a.share - row0;                    // of this tile: row = query * share + r
  const int tile_rows = rows < 16 ? rows : 16;
  const int64_t head = (int64_t)b * a.H + h;
  const char *kc = (const char *)a.k_codes + head * a.S * KROW;
  const char *vc = (const char *)a.v_codes + head * a.S * KROW;
  const uint32_t *kp = (const uint32_t *)a.k_par + head * G * a.S;
  const uint32_t *vp = (const uint32_t *)a.v_par + head * G * a.S;

  u32x2 kw[NSUB][2][G];
  u32x4 vw[NSUB][G];
  uint32_t kpw[G][NP], vpw[G][NP];
  const uint32_t k_off = (8 * (col >> 2) + (col & 3)) * KROW + 8 * g;
  const uint32_t v_off = g * VROW + 16 * col;
  // tile t, 32 tokens at a time, none beyond the `most`th
  auto fetch_k = [&](int t, int most) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      int sub = t * NSUB + s;
      sub = sub < most ? sub : most;
      const char *base = kc + (int64_t)sub * 32 * KROW;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
          kw[s][blk][grp] = load_at<u32x2>(base + blk * 4 * KROW + grp * 32, k_off);
    }
    const uint32_t tok = (uint32_t)t * TT + NP * lane, end = S - NP;
    const uint32_t off = (tok < end ? tok : end) * 4;
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        kpw[grp][e] = load_at<uint32_t>(kp + grp * a.S + e, off);
        vpw[grp][e] = load_at<uint32_t>(vp + grp * a.S + e, off);
      }
  };
  auto fetch_v = [&](int t, int most) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      int sub = t * NSUB + s;
      sub = sub < most ? sub : most;
      const char *base = vc + (int64_t)sub * 4 * VROW;
#pragma unroll
      for (int grp = 0; grp < G; ++grp) vw[s][grp] = load_at<u32x4>(base + grp * 256, v_off);
    }
  };
  // the first tile does not depend on the length where no split does; where sequences are expected
  // to reach it, it is requested before the length is known (64 x 16 heads x 1000 tokens: 18.7 us,
  // 19.5 without)
  if (a.ahead) {
    fetch_k(wave, S / 32 - 1);
    fetch_v(wave, S / 32 - 1);
  }

  int64_t len64 = load_len(a.length, a.length_dtype, b);
  const int len = len64 < 0 ? 0 : (len64 > S ? S : (int)len64);
  int64_t ql64 = a.q_length ? load_len(a.q_length, a.q_length_dtype, b) : Lq;
  const int ql = ql64 < 0 ? 0 : (ql64 > Lq ? Lq : (int)ql64);
  const int reach = a.Lm < S ? (int)a.Lm : S;
  auto seen = [&](int i) -> int {                          // keys that query i sees
    int n = a.causal ? len - ql + i + 1 : len;
    n = n > reach ? reach : n;
    return i < ql && n > 0 ? n : 0;
  };
  int last = (int)((uint32_t)(row0 + tile_rows - 1) / (uint32_t)a.share);   // sees most
  last = last >= ql ? ql - 1 : last;
  const int top = last >= 0 && (last + 1) * a.share > row0 ? seen(last) : 0;
  const int ntiles = (top + TT - 1) / TT;
  int t_begin = 0, t_end = ntiles;
  if (a.splits > 1) {
    const int per = (int)((uint32_t)(ntiles + a.splits - 1) / (uint32_t)a.splits);
    t_begin = (int)split_no * per;
    t_end = t_begin + per < ntiles ? t_begin + per : ntiles;
  }
  // last 32 tokens that this workgroup reads (requests past its end go there again)
  int sub_last = top > 0 ? (top - 1) / 32 : 0;
  if (t_end * NSUB - 1 < sub_last) sub_last = t_end > 0 ? t_end * NSUB - 1 : 0;

  int t = t_begin + wave;
  if (!a.ahead && t < t_end) {
    fetch_k(t, sub_last);
    fetch_v(t, sub_last);
  }

  // ---- queries: operand B of K Q^T, channel 64 grp + 16 g + 8 s + j of row col ----
  bf16x8 qf[G][2][QS];
  // what the accumulators start with, the same for all tokens: -16 sum(q); F32: -23.5 sum(q) over the
  // 32 channels of each product, and what its rounding lost, with the lower parts of q
  float start[G][F32 ? 2 : 1], rest[G];
  float qsum[G];
  {
    const int qr = row0 + col, i = (int)((uint32_t)qr / (uint32_t)a.share);
    const int64_t hq = (int64_t)h * a.share + (qr - i * a.share);
    const T *qp = (const T *)a.q + b * a.q_stride[0] + hq * a.q_stride[1] + i * a.q_stride[2];
    const bool live = col < tile_rows;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
      qsum[grp] = 0.f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int c0 = 64 * grp + 16 * g + 8 * s;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.q_vec) {
          if (live && c0 < a.d) {
            if (F32) {
              const f32x4 lo = *reinterpret_cast<const f32x4 *>(qp + c0);
              const f32x4 hi = *reinterpret_cast<const f32x4 *>(qp + c0 + 4);
#pragma unroll
              for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
            } else {
              const bf16x8 w = *reinterpret_cast<const bf16x8 *>(qp + c0);
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = (float)w[j];
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (live && c0 + j < a.d) x[j] = to_f32(qp[c0 + j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          qsum[grp] += x[j];
          bf16 part[QS];
          split(x[j], part);
#pragma unroll
          for (int k = 0; k < QS; ++k) qf[grp][s][k][j] = part[k];
        }
      }
      qsum[grp] += __shfl_xor(qsum[grp], 16, 64);
      qsum[grp] += __shfl_xor(qsum[grp], 32, 64);
      if (!DIRECT && lane < R) sc[grp * 16 + lane] = qsum[grp];
    }
  }
  const bf16 cen = (bf16)(-23.5f);
  const bf16x8 center = {cen, cen, cen, cen, cen, cen, cen, cen};
#pragma unroll
  for (int grp = 0; grp < G; ++grp) {
    if (F32) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f32x4 sum = mfma16(center, qf[grp][s][0], all4(0.f));
        f32x4 lost = mfma16(center, qf[grp][s][0], -sum);
#pragma unroll
        for (int k = 1; k < QS; ++k) lost = mfma16(center, qf[grp][s][k], lost);
        start[grp][s] = sum[0];
        rest[grp] = s == 0 ? lost[0] : rest[grp] + lost[0];
      }
    } else {
      start[grp][0] = -16.f * qsum[grp];
    }
  }
  int row = col;                                           // the lane's row in the softmax
  const int sl = DIRECT ? g : lane % LPR;
  if (!DIRECT) {
    wave_lds_sync();
    row = lane / LPR;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) qsum[grp] = sc[grp * 16 + row];
    wave_lds_sync();
  }
  // (lanes without a row see nothing, but what they load has to exist: the last row's)
  const int at_row = row0 + (row < tile_rows ? row : tile_rows - 1);
  const int qi = (int)((uint32_t)at_row / (uint32_t)a.share);
  const int64_t hq = (int64_t)h * a.share + (at_row - qi * a.share);
  const int vis = row < tile_rows ? seen(qi) : 0;
  const int pos = len - ql + qi;
  const T *edge = nullptr;
  const int table_last = (int)a.table_len - 1;
  if (BIAS && a.edge)
    edge = (const T *)a.edge + b * a.edge_stride[0] + hq * a.edge_stride[1] +
           qi * a.edge_stride[2];
  const T *table = BIAS && a.table ? (const T *)a.table + hq * a.table_len : nullptr;
  const uint8_t *mask =
      BIAS && a.mask ? a.mask + b * a.mask_stride[0] + qi * a.mask_stride[1] : nullptr;

  // a score from the product, for the token of parameters w
  auto scaled = [&](float dot, uint32_t w, int grp) -> float {
    const float s = scale_of(w);
    const float c = F32 ? fmaf(7.5f, s, min_of(w)) : min_of(w);
    return fmaf(s, dot, c * qsum[grp]);
  };
  const float scale = BIAS ? a.inv_temperature : a.inv_temperature * LOG2E;
  const int seen_last = vis > 0 ? vis - 1 : 0;             // (loads stay on keys that exist)
  // the bias of key j, -inf where the mask is off; key j's score with it
  auto bias_of = [&](int j) -> float {
    float z = 0.f;
    const int jj = j < seen_last ? j : seen_last;
    if (edge) z = to_f32(edge[(int64_t)jj * a.edge_stride[3]]);
    if (table) {
      int at = table_last - pos + jj;
      at = at < 0 ? 0 : (at > table_last ? table_last : at);
      z = to_f32(table[at]);
    }
    if (mask) z = mask[(int64_t)jj * a.mask_stride[2]] != 0 ? z : NEG;
    return z;
  };
  auto finish = [&](float z, float bias, int j) -> float {
    if (BIAS) z = bias == NEG ? NEG : z + bias;
    return j < vis ? z * scale : NEG;
  };

  // ---- running state ----
  float ref = NEG, l = 0.f, csum[G];
  f32x4 acc[G][4];
#pragma unroll
  for (int grp = 0; grp < G; ++grp) {
    csum[grp] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[grp][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  auto rebase = [&](float most) {                          // a larger maximum for the lane's row
#pragma unroll
    for (int o = DIRECT ? 32 : LPR / 2; o > (DIRECT ? 8 : 0); o >>= 1)
      most = fmaxf(most, __shfl_xor(most, o, 64));
    const float to = fmaxf(ref, most);
    const float alpha = ref == to ? 1.f : __builtin_amdgcn_exp2f((ref - to) * UNIT);
    ref = to;
    l *= alpha;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) csum[grp] *= alpha;
    float ac = alpha;
    if (!DIRECT) {
      if (sl == 0) al[row] = alpha;
      wave_lds_sync();
      ac = al[col < R ? col : R - 1];
    }
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[grp][i][e] *= ac;
  };
  // weight p of a token with V parameters w: parts of p s_v, its share of the per-row sum
  auto weigh = [&](float p, bool off, uint32_t w, int grp, bf16 (&part)[PS]) {
    split(off ? 0.f : p * scale_of(w), part);
    csum[grp] = fmaf(p, off ? 0.f : fmaf(7.5f, scale_of(w), min_of(w)), csum[grp]);
    // (the products take 16 + n, of the parts as they are; F32: n - 7.5)
    if (!F32) {
#pragma unroll
      for (int k = 0; k < PS; ++k) csum[grp] = fmaf(-23.5f, (float)part[k], csum[grp]);
    }
  };
  // O^T += V^T P^T of 32 tokens: channel 64 grp + 4 row + i of operand A's row
  auto products = [&](int s, int grp, const bf16x8 (&pb)[PS]) {
    if (F32) {
      const f32x4 from = mfma16(center, pb[0], all4(0.f));
      f32x4 lost = mfma16(center, pb[0], -from);
#pragma unroll
      for (int k = 1; k < PS; ++k) lost = mfma16(center, pb[k], lost);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 v8 = codes16(vw[s][grp][i]);
        const f32x4 o = mfma16(v8, pb[0], from);
        f32x4 low = lost;
#pragma unroll
        for (int k = 1; k < PS; ++k) low = mfma16(v8, pb[k], low);
        acc[grp][i] += o + low;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 v8 = codes16(vw[s][grp][i]);
#pragma unroll
        for (int k = 0; k < PS; ++k) acc[grp][i] = mfma16(v8, pb[k], acc[grp][i]);
      }
    }
  };

  for (; t < t_end; t += 4) {
    float x[TPL];
    uint32_t vpr[G][OWN_PAR ? TPL : 1], kpr[G][OWN_PAR ? TPL : 1];
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        if (OWN_PAR) {
          kpr[grp][e] = kpw[grp][e];
          vpr[grp][e] = vpw[grp][e];
        } else {
          parl[grp * TT + NP * lane + e] = kpw[grp][e];
          parl[(G + grp) * TT + NP * lane + e] = vpw[grp][e];
        }
      }
    float bias[TPL];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VW; ++e)
        bias[v * VW + e] =
            BIAS && !DIRECT ? bias_of(t * TT + v * LPR * VW + sl * VW + e) : 0.f;
    if (DIRECT) wave_lds_sync();
    // ---- scores: S^T = K Q^T, rows of 32 tokens as V wants them ----
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        if (DIRECT)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[(s * 2 + blk) * 4 + e] = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          f32x4 d = all4(start[grp][0]);
          if (F32) {
            f32x4 d2 = all4(start[grp][F32 ? 1 : 0]), low = all4(0.f);
            const bf16x8 k0 = codes16(kw[s][blk][grp][0]), k1 = codes16(kw[s][blk][grp][1]);
            d = mfma16(k0, qf[grp][0][0], d);
            d2 = mfma16(k1, qf[grp][1][0], d2);
#pragma unroll
            for (int k = 1; k < QS; ++k) {
              low = mfma16(k0, qf[grp][0][k], low);
              low = mfma16(k1, qf[grp][1][k], low);
            }
            d = (d + d2) + (low + rest[grp]);
          } else {
            d = mfma16(codes16(kw[s][blk][grp][0]), qf[grp][0][0], d);
            d = mfma16(codes16(kw[s][blk][grp][1]), qf[grp][1][0], d);
          }
          if (DIRECT) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(parl + grp * TT + s * 32 + 8 * g +
                                                             4 * blk);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[(s * 2 + blk) * 4 + e] += scaled(d[e], w[e], grp);
          } else if (col < R) {
            *reinterpret_cast<f32x4 *>(sc + (grp * R + col) * SROW + s * 32 + 8 * g + 4 * blk) = d;
          }
        }
      }
    fetch_k(t + 4, sub_last);
    float most = NEG;
    if (DIRECT) {
#pragma unroll
      for (int n = 0; n < TPL; ++n) {
        const int j = t * TT + (n >> 3) * 32 + 8 * g + (n & 7);
        x[n] = finish(x[n], BIAS ? bias_of(j) : 0.f, j);
        most = fmaxf(most, x[n]);
      }
    } else {
      wave_lds_sync();
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const int n = v * VW + e, tok = v * LPR * VW + sl * VW + e;
          float z = 0.f;
#pragma unroll
          for (int grp = 0; grp < G; ++grp)
            z += scaled(sc[(grp * R + row) * SROW + tok],
                        OWN_PAR ? kpr[grp][n] : parl[grp * TT + tok], grp);
          x[n] = finish(z, bias[n], t * TT + tok);
          most = fmaxf(most, x[n]);
        }
    }
    if (__any(most > ref + STEP || (ref == NEG && most > NEG))) rebase(most);
    // ---- weights and the second product ----
    if (DIRECT) {
#pragma unroll
      for (int s = 0; s < NSUB; ++s) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = x[s * 8 + e];
          p[e] = z == NEG ? 0.f : __builtin_amdgcn_exp2f((z - ref) * UNIT);
          l += p[e];
        }
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          bf16x8 pb[PS];
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(parl + (G + grp) * TT + s * 32 +
                                                             8 * g + 4 * blk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              bf16 part[PS];
              weigh(p[blk * 4 + e], x[s * 8 + blk * 4 + e] == NEG, w[e], grp, part);
#pragma unroll
              for (int k = 0; k < PS; ++k) pb[k][blk * 4 + e] = part[k];
            }
          }
          products(s, grp, pb);
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float p[VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const float z = x[v * VW + e];
          p[e] = z == NEG ? 0.f : __builtin_amdgcn_exp2f((z - ref) * UNIT);
          l += p[e];
        }
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          const int tok = v * LPR * VW + sl * VW;
          bf16 part[VW][PS];
#pragma unroll
          for (int e = 0; e < VW; ++e)
            weigh(p[e], x[v * VW + e] == NEG,
                  OWN_PAR ? vpr[grp][v * VW + e] : parl[(G + grp) * TT + tok + e], grp, part[e]);
#pragma unroll
          for (int k = 0; k < PS; ++k) {
            bf16 *to = pr + ((grp * PS + k) * R + row) * PROW + tok;
#pragma unroll
            for (int e = 0; e < VW; ++e) to[e] = part[e][k];
          }
        }
      }
      wave_lds_sync();
#pragma unroll
      for (int s = 0; s < NSUB; ++s)
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          bf16x8 pb[PS];
#pragma unroll
          for (int k = 0; k < PS; ++k)
            pb[k] = *reinterpret_cast<const bf16x8 *>(
                pr + ((grp * PS + k) * R + (col < R ? col : R - 1)) * PROW + s * 32 + 8 * g);
          products(s, grp, pb);
        }
    }
    fetch_v(t + 4, sub_last);
    wave_lds_sync();
  }

  // ---- join the four waves: each row's sum over its lanes, then the waves through LDS ----
#pragma unroll
  for (int o = DIRECT ? 32 : LPR / 2; o > (DIRECT ? 8 : 0); o >>= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int grp = 0; grp < G; ++grp) csum[grp] += __shfl_xor(csum[grp], o, 64);
  }
  __syncthreads();
  float *jo = (float *)smem;                       // (4, R, OROW)
  float *jm = jo + 4 * R * OROW;                    // (4, R, 2 + G): ref, l, csum
  if (col < R) {
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4 *>(jo + (wave * R + col) * OROW + 64 * grp + 16 * g + 4 * e) =
            (f32x4){acc[grp][0][e], acc[grp][1][e], acc[grp][2][e], acc[grp][3][e]};
  }
  if (sl == 0) {
    float *m = jm + (wave * R + row) * (2 + G);
    m[0] = ref;
    m[1] = l;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) m[2 + grp] = csum[grp];
  }
  __syncthreads();
  const int64_t first_row = ((int64_t)b * a.H + h) * ((int64_t)Lq * a.share) + row0;
  for (int idx = threadIdx.x; idx < R * DP; idx += 256) {
    const int orow = idx / DP, c = idx % DP;
    if (orow >= tile_rows) continue;
    float mx = NEG;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, jm[(w * R + orow) * (2 + G)]);
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float *m = jm + (w * R + orow) * (2 + G);
      const float f = m[0] == mx ? 1.f : __builtin_amdgcn_exp2f((m[0] - mx) * UNIT);
      sum += f * m[1];
      o += f * (jo[(w * R + orow) * OROW + c] + m[2 + c / 64]);
    }
    if (a.splits == 1) {
      const int i = (int)((uint32_t)(row0 + orow) / (uint32_t)a.share);
      const int64_t oh = (int64_t)h * a.share + (row0 + orow - i * a.share);
      if (c < a.d)
        ((T *)a.out)[b * a.o_stride[0] + oh * a.o_stride[1] + i * a.o_stride[2] + c] =
            from_f32<T>(sum == 0.f ? 0.f : o / sum);
    } else {
      const int64_t at = (first_row + orow) * a.splits + split_no;
      a.part_o[at * DP + c] = o;
      if (c == 0) {
        a.part_ml[at * 2] = mx * UNIT;             // in units of log2
        a.part_ml[at * 2 + 1] = sum;
      }
    }
  }
}

// The splits of a row: O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  A workgroup takes one
// row: 256 threads = DP / 4 channel quads x groups of splits, added up in a fixed order.
template <typename T, int DP>
__global__ void __launch_bounds__(256) kv4_join_kernel(Kv4Attn a) {
  constexpr int Q = DP / 4, GROUPS = 256 / Q;
  __shared__ float f[KV4_MAX_SPLITS];
  __shared__ f32x4 part[GROUPS][Q];
  __shared__ float total;
  const int64_t row = blockIdx.x;
  const float *ml = a.part_ml + row * a.splits * 2;
  const f32x4 *po = (const f32x4 *)(a.part_o + row * a.splits * DP);
  const int q = threadIdx.x % Q, grp = threadIdx.x / Q;
  f32x4 v[KV4_MAX_SPLITS / GROUPS];
#pragma unroll
  for (int k = 0; k < KV4_MAX_SPLITS / GROUPS; ++k) {
    const int s = grp + k * GROUPS;
    v[k] = s < a.splits ? po[(int64_t)s * Q + q] : (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  if (threadIdx.x < 64) {
    const int s = threadIdx.x;
    const float m = s < a.splits ? ml[2 * s] : -__builtin_inff();
    const float l = s < a.splits ? ml[2 * s + 1] : 0.f;
    const float mx = wave_max(m);
    const float w = m == mx ? 1.f : __builtin_amdgcn_exp2f(m - mx);
    f[s] = w;
    const float sum = wave_sum(w * l);
    if (s == 0) total = sum;
  }
  __syncthreads();
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < KV4_MAX_SPLITS / GROUPS; ++k) {
    const int s = grp + k * GROUPS;
    if (s < a.splits) {
      const float w = f[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(w, v[k][e], o[e]);
    }
  }
  part[grp][q] = o;
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= a.d) return;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) sum += part[k][c / 4][c % 4];
  const uint32_t per = (uint32_t)(a.Lq * a.share);
  const uint32_t bh = (uint32_t)row / per, rr = (uint32_t)row - bh * per;
  const uint32_t b = bh / (uint32_t)a.H, h = bh - b * (uint32_t)a.H, i = rr / (uint32_t)a.share;
  const int64_t hq = (int64_t)h * a.share + (rr - i * (uint32_t)a.share);
  ((T *)a.out)[b * a.o_stride[0] + hq * a.o_stride[1] + i * a.o_stride[2] + c] =
      from_f32<T>(total == 0.f ? 0.f : sum / total);
}

// Rows of a workgroup.  One query: 64 x 16 heads x 1000 tokens 18.7 us with R = 1, 21.0 with 4, 27.1
// with 16; 8 heads x 40 tokens 6.6, 7.6 and 11.0; four queries x 32768 tokens 60 us with R = 4, 75
// with 16.
template <typename T, int DP, bool BIAS>
void launch_rows(const Kv4Attn &a, hipStream_t s) {
  const int64_t rows = a.Lq * a.share;
  const dim3 grid((unsigned)(a.B * a.H * a.row_tiles * a.splits)), block(256);
#define GO(R) hipLaunchKernelGGL((kv4_attn_kernel<T, DP, R, BIAS>), grid, block, 0, s, a)
  if (rows > 4) GO(16);
  else if (rows > 2) GO(4);
  else if (rows > 1) GO(2);
  else GO(1);
#undef GO
}

template <typename T, int DP>
void launch(const Kv4Attn &a, hipStream_t s) {
  if (a.edge || a.table || a.mask) launch_rows<T, DP, true>(a, s);
  else launch_rows<T, DP, false>(a, s);
  if (a.splits > 1) {
    const int64_t all = a.B * a.H * a.Lq * a.share;
    hipLaunchKernelGGL((kv4_join_kernel<T, DP>), dim3((unsigned)all), dim3(256), 0, s, a);
  }
}

}  // namespace

// Splits of a sequence: up to 1024 workgroups at head dim 64 and 512 at 128, and no more than give each
// the same number of rounds of four tiles.  bf16 kernels up to 4 rows without a bias keep them all
// resident (4 a CU, 3 at head dim 128); of the others' (bf16 3, with a bias 4 to 2, float32 3 to 1 a
// CU) some may wait for the first to end.  Measured where all are resident, one query a head, us:
//   32 x 8 heads of 128, 2048 tokens: 512 workgroups 18.8, 256 19.8, 1024 21.5
//   64 x 16 heads of 64, 1000 tokens: 1024 workgroups 18.7, 2048 24.0 and a join
//   4 x 12 heads of 64, 16384 tokens: 16 splits (768 workgroups, 2 rounds each) 16.0, 22 (1056; 1.5
//   rounds, and 32 workgroups that wait for the others to end) 19.6; float32 20.8 and 27.2
//   5 x 8 heads of 128 with 4 queries, 20000 tokens: 12 splits (480) 27.8, 13 (520) 32.4
// 300 to 800 workgroups that hold a sequence each gain as much from 2 splits as the join costs.
int kv4_attn_plan(int64_t B, int64_t H, int64_t rows, int64_t keys, int64_t d) {
  const int64_t tile = d > 64 ? 64 : 128, aim = d > 64 ? 512 : 1024;
  const int64_t wgs = B * H * ((rows + 15) / 16);
  const int64_t rounds = keys > 0 ? (keys + 4 * tile - 1) / (4 * tile) : 1;   // of four tiles
  int64_t n = aim / wgs;
  n = n < 1 ? 1 : (n > KV4_MAX_SPLITS ? KV4_MAX_SPLITS : n);
  const int64_t each = (rounds + n - 1) / n;
  return (int)((rounds + each - 1) / each);
}

void launch_kv4_attn(const Kv4Attn &a, int dtype, hipStream_t s) {
  if (dtype == GNLP_BF16) {
    if (a.d > 64) launch<bf16, 128>(a, s);
    else launch<bf16, 64>(a, s);
  } else {
    if (a.d > 64) launch<float, 128>(a, s);
    else launch<float, 64>(a, s);
  }
}

}  // namespace gnlp
