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
// is split into two (bf16 tensors: 16 bits) or three parts (float32: all 24 bits).  What the parts
// lose multiplies n - 7.5, not n: the rest of p s_v goes into the per-row sum with 7.5.  For float32
// the 23.5 = 16 + 7.5 is also taken off inside the matrix product, 32 tokens at a time (a product
// with a constant operand starts the accumulators): sums over a long context would otherwise grow
// to 23.5 sum(p s_v) and lose the digits of a result that averages out.
//
// Work: a wave takes tiles of TT = 128 (head dim 64) or 64 tokens, 8 KB of codes, on its own, with
// its own running maximum; four waves of a workgroup and, for few heads, several workgroups
// (`splits`, joined by kv4_join_kernel) share a sequence.
//   S^T = K Q^T: operand A = 16 cached tokens as they lie in memory, operand B = 16 query rows.
//   O^T = V^T P^T: operand A = 16 channels x 32 tokens, again as they lie in memory.
// With fewer than 16 query rows (one, in plain decoding) most columns of S^T are idle; the scores
// therefore go through LDS, where the wave spreads the R rows that exist over its 64 lanes: the
// softmax costs R tokens x 128 / 64 instead of 32 evaluations a lane.  R = 1, 2, 4, 8, 16.
// The running maximum moves only when a score exceeds it by 8 (exp(8) is harmless in float32):
// noticing that is one vote, the reduction over lanes is the exception.
//
// Bound by memory: 72 bytes a token and cached head at head dim 64 (256 in bf16).
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

template <typename T, int DP, int R>
__global__ void __launch_bounds__(256) kv4_attn_kernel(Kv4Attn a) {
  constexpr int G = DP / 64;             // groups of a token
  constexpr int TT = 128 / G;            // tokens of a tile
  constexpr int NSUB = TT / 32;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int QS = F32 ? 3 : 1;        // bf16 parts of a query value
  constexpr int PS = F32 ? 3 : 2;        // bf16 parts of p s_v
  constexpr int LPR = 64 / R;            // lanes of a row in the softmax
  constexpr int TPL = TT / LPR;          // tokens of a lane there (R == 1, TT == 64: one)
  constexpr int VW = TPL < 4 ? TPL : 4;  // ... in vectors of
  constexpr int NV = TPL / VW;
  constexpr int SROW = TT + 4, PROW = TT + 8;
  constexpr float NEG = -__builtin_inff();
  constexpr float STEP = 8.0f, LOG2E = 1.4426950408889634f;

  // per wave: scores (G, R, SROW) float, P (G, PS, R, PROW) bf16, parameters (2, G, TT), alpha (R)
  constexpr int S_BYTES = G * R * SROW * 4, P_BYTES = G * PS * R * PROW * 2;
  constexpr int PAR_BYTES = R > 1 ? 2 * G * TT * 4 : 0;
  constexpr int WAVE_BYTES = (S_BYTES + P_BYTES + PAR_BYTES + 16 * 4 + 15) / 16 * 16;
  constexpr int OUT_BYTES = 4 * R * (DP + 2 + G) * 4;
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
  const uint32_t rt = lin % a.row_tiles;
  lin /= a.row_tiles;
  const uint32_t split = lin % a.splits;
  lin /= a.splits;
  const uint32_t h = lin % (uint32_t)a.H;
  const int64_t b = lin / (uint32_t)a.H;
  const int rows = (int)(a.Lq * a.share) - (int)rt * 16;   // of this tile: row = query * share + r
  int64_t len = load_len(a.length, a.length_dtype, b);
  len = len < 0 ? 0 : (len > a.S ? a.S : len);
  int64_t ql = a.q_length ? load_len(a.q_length, a.q_length_dtype, b) : a.Lq;
  ql = ql < 0 ? 0 : (ql > a.Lq ? a.Lq : ql);
  auto seen = [&](int64_t i) -> int {                      // keys that query i sees
    int64_t n = a.causal ? len - ql + i + 1 : len;
    n = n > a.Lm ? a.Lm : n;
    return i < ql && n > 0 ? (int)n : 0;
  };
  const int tile_rows = rows < 16 ? rows : 16;
  int64_t last = ((int64_t)rt * 16 + tile_rows - 1) / a.share;   // the row that sees most
  last = last >= ql ? ql - 1 : last;
  const int top = last * a.share + a.share > (int64_t)rt * 16 && last >= 0 ? seen(last) : 0;
  const int ntiles = (top + TT - 1) / TT, per = (ntiles + a.splits - 1) / a.splits;
  const int t_begin = split * per, t_end = t_begin + per < ntiles ? t_begin + per : ntiles;
  const int sub_last = top > 0 ? (top - 1) / 32 : 0;       // last 32 tokens that are read

  const int64_t head = b * a.H + h;
  const uint32_t *kc = (const uint32_t *)a.k_codes + head * a.S * (DP / 8);
  const uint32_t *vc = (const uint32_t *)a.v_codes + head * a.S * (DP / 8);
  const uint32_t *kp = (const uint32_t *)a.k_par + head * G * a.S;
  const uint32_t *vp = (const uint32_t *)a.v_par + head * G * a.S;

  // ---- queries: operand B of K Q^T, channel 64 grp + 16 g + 8 s + j of row col ----
  bf16x8 qf[G][2][QS];
  {
    float qsum[G];
    const int rr = (int)rt * 16 + col;
    const int64_t i = rr / a.share, hq = (int64_t)h * a.share + rr % a.share;
    const T *qp = (const T *)a.q + b * a.q_stride[0] + hq * a.q_stride[1] + i * a.q_stride[2];
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
      qsum[grp] = 0.f;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = 64 * grp + 16 * g + 8 * s + j;
          float x = 0.f;
          if (col < tile_rows && c < a.d) x = to_f32(qp[c]);
          qsum[grp] += x;
#pragma unroll
          for (int k = 0; k < QS; ++k) {
            const bf16 part = (bf16)x;
            qf[grp][s][k][j] = part;
            x -= (float)part;
          }
        }
      qsum[grp] += __shfl_xor(qsum[grp], 16, 64);
      qsum[grp] += __shfl_xor(qsum[grp], 32, 64);
      if (lane < R) sc[grp * 16 + lane] = qsum[grp];
    }
  }
  wave_lds_sync();
  const int row = lane / LPR, sl = lane % LPR;             // the lane's row in the softmax
  float qs[G];
#pragma unroll
  for (int grp = 0; grp < G; ++grp) qs[grp] = sc[grp * 16 + row];
  wave_lds_sync();
  const int rr = (int)rt * 16 + row;
  const int64_t qi = rr / a.share, hq = (int64_t)h * a.share + rr % a.share;
  const int vis = row < tile_rows ? seen(qi) : 0;
  const int pos = (int)(len - ql + qi);
  const T *edge = nullptr;
  if (a.edge)
    edge = (const T *)a.edge + b * a.edge_stride[0] + hq * a.edge_stride[1] +
           qi * a.edge_stride[2];
  const T *table = a.table ? (const T *)a.table + hq * a.table_len : nullptr;
  const uint8_t *mask = a.mask ? a.mask + b * a.mask_stride[0] + qi * a.mask_stride[1] : nullptr;

  // ---- running state ----
  float ref = NEG, l = 0.f, csum[G];
  f32x4 acc[G][4];
#pragma unroll
  for (int grp = 0; grp < G; ++grp) {
    csum[grp] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[grp][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const bf16 cen = (bf16)(-23.5f);
  const bf16x8 center = {cen, cen, cen, cen, cen, cen, cen, cen};

  u32x2 kw[NSUB][2][G];
  u32x4 vw[NSUB][G];
  constexpr int NP = TT / 64;                              // tokens whose parameters a lane fetches
  uint32_t kpw[G][NP], vpw[G][NP];
  auto fetch = [&](int t) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      int sub = t * NSUB + s;
      sub = sub < sub_last ? sub : sub_last;               // (past the end: the last ones again)
      const int64_t tok = (int64_t)sub * 32;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
          kw[s][blk][grp] = *reinterpret_cast<const u32x2 *>(
              kc + (tok + 8 * (col >> 2) + 4 * blk + (col & 3)) * (DP / 8) + grp * 8 + 2 * g);
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
        vw[s][grp] = *reinterpret_cast<const u32x4 *>(vc + (tok / 8 + g) * DP + grp * 64 + 4 * col);
    }
    int64_t tok = (int64_t)t * TT + NP * lane;
    const int64_t most = (int64_t)sub_last * 32 + 32 - NP;
    tok = tok < most ? tok : most;
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        kpw[grp][e] = kp[grp * a.S + tok + e];
        vpw[grp][e] = vp[grp * a.S + tok + e];
      }
  };

  int t = t_begin + wave;
  if (t < t_end) fetch(t);
  for (; t < t_end; t += 4) {
    // ---- scores of the tile: S^T = K Q^T, rows of 32 tokens as V wants them ----
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const bf16x8 k8 = codes16(kw[s][blk][grp][st]);
#pragma unroll
            for (int k = 0; k < QS; ++k) x = mfma16(k8, qf[grp][st][k], x);
          }
          if (col < R)
            *reinterpret_cast<f32x4 *>(sc + (grp * R + col) * SROW + s * 32 + 8 * g + 4 * blk) = x;
        }
    uint32_t kpr[G][TPL], vpr[G][TPL];
    if (R > 1) {
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          parl[grp * TT + NP * lane + e] = kpw[grp][e];
          parl[(G + grp) * TT + NP * lane + e] = vpw[grp][e];
        }
    }
    u32x4 vnow[NSUB][G];
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int grp = 0; grp < G; ++grp) vnow[s][grp] = vw[s][grp];
    if (R == 1) {
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int e = 0; e < TPL; ++e) {
          kpr[grp][e] = kpw[grp][e < NP ? e : 0];
          vpr[grp][e] = vpw[grp][e < NP ? e : 0];
        }
    }
    if (t + 4 < t_end) fetch(t + 4);
    wave_lds_sync();

    // ---- softmax: lane (row, sl), tokens v LPR VW + sl VW + e of the tile ----
    float x[TPL];
    float most = NEG;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const int n = v * VW + e, tok = v * LPR * VW + sl * VW + e, j = t * TT + tok;
        float z = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          if (R > 1) {
            kpr[grp][n] = parl[grp * TT + tok];
            vpr[grp][n] = parl[(G + grp) * TT + tok];
          }
          const float dot = fmaf(-16.f, qs[grp], sc[(grp * R + row) * SROW + tok]);
          z += fmaf(scale_of(kpr[grp][n]), dot, min_of(kpr[grp][n]) * qs[grp]);
        }
        bool on = j < vis;
        if (on) {
          if (edge) z += to_f32(edge[(int64_t)j * a.edge_stride[3]]);
          if (table) {
            int64_t at = a.table_len - 1 - (pos - j);
            at = at < 0 ? 0 : (at >= a.table_len ? a.table_len - 1 : at);
            z += to_f32(table[at]);
          }
          if (mask) on = mask[(int64_t)j * a.mask_stride[2]] != 0;
        }
        x[n] = on ? z * a.inv_temperature : NEG;
        most = fmaxf(most, x[n]);
      }
    if (__any(most > ref + STEP || (ref == NEG && most > NEG))) {
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
      const float to = fmaxf(ref, most);
      const float alpha = ref == to ? 1.f : __builtin_amdgcn_exp2f((ref - to) * LOG2E);
      ref = to;
      l *= alpha;
#pragma unroll
      for (int grp = 0; grp < G; ++grp) csum[grp] *= alpha;
      if (sl == 0) al[row] = alpha;
      wave_lds_sync();
      const float ac = al[col < R ? col : R - 1];
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[grp][i][e] *= ac;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float p[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const float z = x[v * VW + e];
        p[e] = z == NEG ? 0.f : __builtin_amdgcn_exp2f((z - ref) * LOG2E);
        l += p[e];
      }
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        bf16 part[PS][VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const uint32_t w = vpr[grp][v * VW + e];
          const bool off = x[v * VW + e] == NEG;
          const float pv = off ? 0.f : p[e] * scale_of(w);
          float rest = pv, sum = 0.f;
#pragma unroll
          for (int k = 0; k < PS; ++k) {
            part[k][e] = (bf16)rest;
            sum += (float)part[k][e];
            rest -= (float)part[k][e];
          }
          // F32: the 23.5 comes off inside the product
          csum[grp] += (off ? 0.f : p[e] * min_of(w)) + fmaf(7.5f, pv, F32 ? 0.f : -23.5f * sum);
        }
#pragma unroll
        for (int k = 0; k < PS; ++k) {
          bf16 *to = pr + ((grp * PS + k) * R + row) * PROW + v * LPR * VW + sl * VW;
#pragma unroll
          for (int e = 0; e < VW; ++e) to[e] = part[k][e];
        }
      }
    }
    wave_lds_sync();

    // ---- O^T += V^T P^T: channel 64 grp + 4 row + i of operand A's row ----
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        bf16x8 pb[PS];
#pragma unroll
        for (int k = 0; k < PS; ++k)
          pb[k] = *reinterpret_cast<const bf16x8 *>(
              pr + ((grp * PS + k) * R + (col < R ? col : R - 1)) * PROW + s * 32 + 8 * g);
        if (F32) {
          f32x4 start = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < PS; ++k) start = mfma16(center, pb[k], start);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bf16x8 v8 = codes16(vnow[s][grp][i]);
            f32x4 o = start;
#pragma unroll
            for (int k = 0; k < PS; ++k) o = mfma16(v8, pb[k], o);
            acc[grp][i] += o;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bf16x8 v8 = codes16(vnow[s][grp][i]);
#pragma unroll
            for (int k = 0; k < PS; ++k) acc[grp][i] = mfma16(v8, pb[k], acc[grp][i]);
          }
        }
      }
    wave_lds_sync();
  }

  // ---- join the four waves: each row's sum over its lanes, then the waves through LDS ----
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int grp = 0; grp < G; ++grp) csum[grp] += __shfl_xor(csum[grp], o, 64);
  }
  __syncthreads();
  float *jo = (float *)smem;                       // (4, R, DP)
  float *jm = jo + 4 * R * DP;                     // (4, R, 2 + G): ref, l, csum
  if (col < R) {
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          jo[(wave * R + col) * DP + 64 * grp + 16 * g + 4 * e + i] = acc[grp][i][e];
  }
  if (sl == 0) {
    float *m = jm + (wave * R + row) * (2 + G);
    m[0] = ref;
    m[1] = l;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) m[2 + grp] = csum[grp];
  }
  __syncthreads();
  const int64_t first_row = (b * a.H + h) * (a.Lq * a.share) + (int64_t)rt * 16;
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
      const float f = m[0] == mx ? 1.f : __builtin_amdgcn_exp2f((m[0] - mx) * LOG2E);
      sum += f * m[1];
      o += f * (jo[(w * R + orow) * DP + c] + m[2 + c / 64]);
    }
    if (a.splits == 1) {
      const int orr = (int)rt * 16 + orow;
      const int64_t i = orr / a.share, oh = (int64_t)h * a.share + orr % a.share;
      if (c < a.d)
        ((T *)a.out)[b * a.o_stride[0] + oh * a.o_stride[1] + i * a.o_stride[2] + c] =
            from_f32<T>(sum == 0.f ? 0.f : o / sum);
    } else {
      const int64_t at = (first_row + orow) * a.splits + split;
      a.part_o[at * DP + c] = o;
      if (c == 0) {
        a.part_ml[at * 2] = mx;
        a.part_ml[at * 2 + 1] = sum;
      }
    }
  }
}

// The splits of a row, in order: O = sum_s exp(m_s - M) O_s / sum_s exp(m_s - M) l_s.
template <typename T, int DP>
__global__ void __launch_bounds__(256) kv4_join_kernel(Kv4Attn a) {
  constexpr float LOG2E = 1.4426950408889634f;
  const int64_t rows = a.B * a.H * a.Lq * a.share;
  const int64_t row = (int64_t)blockIdx.x * (256 / DP) + threadIdx.x / DP;
  const int c = threadIdx.x % DP;
  if (row >= rows || c >= a.d) return;
  const float *ml = a.part_ml + row * a.splits * 2;
  const float *po = a.part_o + row * a.splits * DP + c;
  float mx = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, ml[2 * s]);
  float sum = 0.f, o = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float f = ml[2 * s] == mx ? 1.f : __builtin_amdgcn_exp2f((ml[2 * s] - mx) * LOG2E);
    sum += f * ml[2 * s + 1];
    o += f * po[(int64_t)s * DP];
  }
  const int64_t per = a.Lq * a.share, bh = row / per, rr = row - bh * per;
  const int64_t b = bh / a.H, h = bh - b * a.H, i = rr / a.share;
  const int64_t hq = h * a.share + rr - i * a.share;
  ((T *)a.out)[b * a.o_stride[0] + hq * a.o_stride[1] + i * a.o_stride[2] + c] =
      from_f32<T>(sum == 0.f ? 0.f : o / sum);
}

template <typename T, int DP>
void launch(const Kv4Attn &a, hipStream_t s) {
  const int64_t rows = a.Lq * a.share;
  const dim3 grid((unsigned)(a.B * a.H * a.row_tiles * a.splits)), block(256);
#define GO(R) hipLaunchKernelGGL((kv4_attn_kernel<T, DP, R>), grid, block, 0, s, a)
  if (rows > 8) GO(16);
  else if (rows > 4) GO(8);
  else if (rows > 2) GO(4);
  else if (rows > 1) GO(2);
  else GO(1);
#undef GO
  if (a.splits > 1) {
    const int64_t all = a.B * a.H * rows, per = 256 / DP;
    hipLaunchKernelGGL((kv4_join_kernel<T, DP>), dim3((unsigned)((all + per - 1) / per)), block, 0,
                       s, a);
  }
}

}  // namespace

int kv4_attn_plan(int64_t B, int64_t H, int64_t rows, int64_t keys, int64_t d) {
  const int64_t tile = d > 64 ? 64 : 128;
  const int64_t wgs = B * H * ((rows + 15) / 16), most = (keys + 4 * tile - 1) / (4 * tile);
  int64_t n = (1024 + wgs - 1) / wgs;
  n = n > most ? most : n;
  return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
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
