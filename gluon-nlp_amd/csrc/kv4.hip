// A key / value cache held in 4 bits: storing tokens (quantisation) and reading them back, gfx950.
// The attention over it is kv4_attn.hip.
//
// Format.  A group = 64 consecutive channels of one token and head (the last one may be shorter):
//   scale = bf16((max - min) * fl32(1 / 15)),  minimum = bf16(min)      (one 32-bit word a group)
//   code  = clamp(rint((x - minimum) / scale), 0, 15),  value = code * scale + minimum
// in 32-bit arithmetic; value's product is exact (8 + 4 bits), so fma and mul + add agree.  A scale
// below 2^-126 counts as 0 (codes 0).  A group whose range or minimum is not finite, or that holds
// a NaN, gets scale = minimum = NaN: all of it reads back as NaN.
//
// Layout (per layer; S = slots, a multiple of 32; DP = head channels padded to 64 or 128):
//   k_codes [B][H][S][DP / 2]      a token's channels together: one 32-bit word = 8 channels
//   v_codes [B][H][S / 8][DP]      one 32-bit word = 8 consecutive tokens of one channel
//   k_par, v_par [B][H][DP / 64][S]   scale in the low 16 bits, minimum in the high
// Element e (channel or token) of a word sits at nibble (e >> 1) + 4 (e & 1): shifting by 4 i and
// masking two nibbles gives elements 2 i and 2 i + 1 in the halves of a register.  The two code
// arrays are what the two matrix products of the attention want as operands: K rows along the
// channels, V columns along the tokens, both without a transpose there.  The price is paid here: a
// V word is shared by 8 tokens, so storing one token rewrites the words (a wave owns all 8 tokens
// of a word: no two waves of a call touch the same one).
//
// Both kernels: a wave = one (batch, head, group, block of 8 slots) of K or V; lane 8 r + c holds
// channels 8 c .. 8 c + 7 of token tok(r).  V goes through an 8 x 8 nibble transpose over the r
// lanes in three exchange steps.  Bound by memory: 2 or 4 bytes a value in (out), 0.5625 out (in);
// writes come near their limit of instructions too, about 18 a value, 4 of them the quotient.
// bfloat16, 32 x 512 tokens (lengths 256 .. 512) of 16 heads of 64: written in 18.7 us (64 MB,
// 3.4 TB/s), read back in 19.0 us (81 MB, 4.3 TB/s; a large copy reaches 4.95); one token of 16 x 12
// heads: 3.5 us each, an empty kernel's time.
#include "common.h"
#include "kernels.h"

namespace gnlp {
namespace {

// row r of lanes <-> token of the 8-slot block: nibble position r holds token tok(r)
__device__ __forceinline__ int tok_of(int r) { return r < 4 ? 2 * r : 2 * r - 7; }

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf,
                                                            0xf, true));
}
// a NaN makes these NaN
__device__ __forceinline__ float lesser(float x, float y) {
  return __builtin_elementwise_minimum(x, y);
}
__device__ __forceinline__ float greater(float x, float y) {
  return __builtin_elementwise_maximum(x, y);
}
// over the 8 lanes that hold one group: quad exchanges, then the mirror of the half row
__device__ __forceinline__ float min8(float x) {
  x = lesser(x, dpp<0xB1>(x));
  x = lesser(x, dpp<0x4E>(x));
  return lesser(x, dpp<0x141>(x));
}
__device__ __forceinline__ float max8(float x) {
  x = greater(x, dpp<0xB1>(x));
  x = greater(x, dpp<0x4E>(x));
  return greater(x, dpp<0x141>(x));
}

// word of lane row r (nibble k = element (r, k)) -> nibble t = element (t, r), over lanes 8 apart
__device__ __forceinline__ uint32_t transpose8(uint32_t w, int r) {
  uint32_t p = __shfl_xor(w, 32, 64);
  w = (r & 4) ? (p >> 16) | (w & 0xffff0000u) : (w & 0xffffu) | (p << 16);
  p = __shfl_xor(w, 16, 64);
  w = (r & 2) ? ((p >> 8) & 0x00ff00ffu) | (w & 0xff00ff00u)
              : (w & 0x00ff00ffu) | ((p & 0x00ff00ffu) << 8);
  p = __shfl_xor(w, 8, 64);
  return (r & 1) ? ((p >> 4) & 0x0f0f0f0fu) | (w & 0xf0f0f0f0u)
                 : (w & 0x0f0f0f0fu) | ((p & 0x0f0f0f0fu) << 4);
}

struct Unit {      // what a wave works on: the blocks of 8 slots from slot0 on
  int b, h, grp, which;              // which: 0 = K, 1 = V
  int slot0, first, end;             // slot0: the block's first slot; [first, end): the call's slots
  bool on;
};

// a length within what 32-bit arithmetic on slots (below 2^30, as L is) takes
__device__ __forceinline__ int bounded(int64_t n) {
  return n > (1 << 30) ? 1 << 30 : (n < -(1 << 30) ? -(1 << 30) : (int)n);
}

// grid: x = (block of slots, head, group), four waves a workgroup; y = sequence; z = K or V.  Heads
// run fastest: neighbouring waves read neighbouring rows of an (N, T, H, d) tensor.
template <int UN>
__device__ __forceinline__ Unit unit_of(const Kv4Io &a) {
  Unit u;
  const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t per = (uint32_t)a.H << a.g_shift, blk = w / per, hg = w - blk * per;
  const int L = (int)a.L;
  u.b = blockIdx.y;
  u.which = blockIdx.z;
  u.h = (int)(hg >> a.g_shift);
  u.grp = (int)(hg & ((1u << a.g_shift) - 1));
  if (a.write) {                     // the last new_length slots of the sequence
    u.end = a.length ? bounded(load_len(a.length, a.length_dtype, u.b)) : L;
    int n = a.count ? bounded(load_len(a.count, a.count_dtype, u.b)) : L;
    n = n < 0 ? 0 : (n > L ? L : n);
    u.first = u.end - n;
  } else {
    u.first = a.count ? bounded(load_len(a.count, a.count_dtype, u.b)) : 0;
    u.end = u.first > 0x7fffffff - L ? 0x7fffffff : u.first + L;
  }
  // blocks of 8 slots, counted from the first slot's (also below slot 0, where nothing is held)
  u.on = blk * UN < a.nblk;
  const int64_t slot0 = (int64_t)(u.first & ~7) + 8 * UN * (int64_t)blk;
  u.on = u.on && slot0 < u.end;
  u.slot0 = u.on ? (int)slot0 : 0;
  return u;
}

// 8 channels of a token, as they were loaded (0 where nothing was)
template <typename T, bool VEC> struct Values {
  typedef typename VecOf<T>::type V;
  static constexpr int N = VecOf<T>::N;
  V v[8 / N];
  __device__ __forceinline__ void load(bool live, const T *p, int c0, int d) {
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[i][e] = (T)0.f;
      if (VEC) {
        if (live && c0 < d) v[i] = *reinterpret_cast<const V *>(p + c0 + i * N);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (live && c0 + i * N + e < d) v[i][e] = p[c0 + i * N + e];
      }
    }
  }
  __device__ __forceinline__ float get(int e) const { return to_f32((T)v[e / N][e % N]); }
};

// WHOLE: all slots of the unit are stored
template <typename T, bool VEC, int UN, bool WHOLE>
__device__ __forceinline__ void store(const Kv4Io &a, const Unit &u) {
  const int lane = threadIdx.x & 63;
  const int r = lane >> 3, c = lane & 7, S = (int)a.S, d = (int)a.d, tok = tok_of(r);
  const int c0 = u.grp * 64 + 8 * c;
  const int64_t head = (int64_t)u.b * a.H + u.h;
  uint32_t *codes = (uint32_t *)(u.which ? a.v_codes : a.k_codes);
  uint32_t *par = (uint32_t *)(u.which ? a.v_par : a.k_par) + ((head << a.g_shift) + u.grp) * S;
  const int64_t step = u.which ? a.v_stride[2] : a.k_stride[2];
  const T *src = (const T *)(u.which ? a.v : a.k) +
                 (u.which ? u.b * a.v_stride[0] + u.h * a.v_stride[1]
                          : u.b * a.k_stride[0] + u.h * a.k_stride[1]) +
                 (u.slot0 - u.first) * step;
  const int64_t mine = tok * step;         // (what differs between lanes)
  const uint32_t word = u.which ? c0 + r : (uint32_t)(tok * (int)a.DP + c0) >> 3;
  auto stored = [&](int slot) {
    return WHOLE || (slot >= u.first && slot < u.end && slot >= 0 && slot < S);
  };
  Values<T, VEC> in[UN];
#pragma unroll
  for (int k = 0; k < UN; ++k)
    in[k].load(stored(u.slot0 + 8 * k + tok), src + 8 * k * step + mine, c0, d);
#pragma unroll
  for (int k = 0; k < UN; ++k) {
    const int block = u.slot0 + 8 * k;
    const bool live = stored(block + tok);
    const uint64_t on = WHOLE ? ~0ull : __ballot(live);
    if (!WHOLE && on == 0) continue;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = in[k].get(e);
    uint32_t *word_at = codes + (u.which ? (head * (S >> 3) + (block >> 3)) * a.DP
                                         : ((head * S + block) * a.DP) >> 3) + word;
    // a block that this call stores in part: nibbles of the other tokens are kept
    uint32_t keep = 0xffffffffu, old = 0;
    if (u.which && on != ~0ull) {
      keep = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if ((on >> (8 * t)) & 1) keep |= 0xfu << (4 * t);
      old = *word_at;
    }

    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      if (VEC || c0 + e < d) {
        lo = lesser(lo, x[e]);
        hi = greater(hi, x[e]);
      }
    }
    if (c0 >= d) { lo = __builtin_inff(); hi = -__builtin_inff(); }   // (no channel of the head)
    lo = min8(lo);
    hi = max8(hi);
    const bf16 sb = (bf16)((hi - lo) * (float)(1.0 / 15.0)), mb = (bf16)lo;
    float s = (float)sb;
    const float m = (float)mb, largest = 3.4028234663852886e38f;
    const bool bad = !(s <= largest) || !(fabsf(m) <= largest);   // (NaN and infinities end here)
    s = s < 1.1754943508222875e-38f ? 0.f : s;
    uint32_t group = (uint32_t)__builtin_bit_cast(uint16_t, (bf16)s) |
                     ((uint32_t)__builtin_bit_cast(uint16_t, mb) << 16);
    if (bad) { group = 0x7fc07fc0u; s = 0.f; }
    // The quotient (x - m) / s, rounded as a division rounds it: the residual of an approximate
    // quotient is exact in one fma, another corrects it (exact halves, which a few in a hundred
    // bf16 values are, stay exact).  Outside the range where reciprocal and residual are normal
    // numbers: the division.  Adding 1.5 2^23 rounds to a whole number in the low bits; what the
    // high bits add up to in the packed word comes off at the end.
    constexpr float ROUND = 12582912.f;
    constexpr uint32_t HIGH = 0x4b400000u;
    float inv = __builtin_amdgcn_rcpf(s);
    inv = fmaf(fmaf(-s, inv, 1.f), inv, inv);
    const bool flat = s == 0.f, plain = s > 1e-30f && s < 1e30f;
    if (flat) { inv = 0.f; }
    const bool exact = __any(!flat && !plain);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = x[e] - m;
      y[e] = t * inv;
      y[e] = fmaf(fmaf(-y[e], s, t), inv, y[e]);
    }
    if (exact) {
      asm volatile("");                       // (a branch: not to be computed ahead)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!flat && !plain) y[e] = (x[e] - m) / s;
    }
    uint32_t w = 0, high = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = __builtin_amdgcn_fmed3f(y[e], 0.f, 15.f) + ROUND;
      const int at = u.which ? 4 * e : 4 * ((e >> 1) + 4 * (e & 1));
      w += __builtin_bit_cast(uint32_t, n) << at;
      high += HIGH << at;
    }
    w -= high;
    if (u.which) {
      w = transpose8(w, r);
      *word_at = WHOLE ? w : (old & ~keep) | (w & keep);
    } else if (live) {
      *word_at = w;
    }
    if (live && c == 0) par[block + tok] = group;
  }
}

template <typename T, bool VEC, int UN>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4Io a) {
  const Unit u = unit_of<UN>(a);
  if (!u.on) return;
  const int last = u.end < (int)a.S ? u.end : (int)a.S;
  if (u.slot0 >= u.first && u.slot0 >= 0 && u.slot0 + 8 * UN <= last) store<T, VEC, UN, true>(a, u);
  else store<T, VEC, UN, false>(a, u);
}

template <typename T, bool VEC, int UN>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Io a) {
  const int lane = threadIdx.x & 63;
  const Unit u = unit_of<UN>(a);
  if (!u.on) return;
  const int r = lane >> 3, c = lane & 7, S = (int)a.S, d = (int)a.d;
  int len = a.length ? bounded(load_len(a.length, a.length_dtype, u.b)) : S;
  len = len > S ? S : len;
  const int c0 = u.grp * 64 + 8 * c;
  const int64_t head = (int64_t)u.b * a.H + u.h;
  const uint32_t *codes = (const uint32_t *)(u.which ? a.v_codes : a.k_codes);
  const uint32_t *par =
      (const uint32_t *)(u.which ? a.v_par : a.k_par) + ((head << a.g_shift) + u.grp) * S;
  uint32_t w[UN], word[UN];
#pragma unroll
  for (int k = 0; k < UN; ++k) {
    const int block = u.slot0 + 8 * k, slot = block + tok_of(r);
    w[k] = word[k] = 0;
    if (slot >= 0 && slot < len) word[k] = par[slot];
    if (block >= 0 && block < len)
      w[k] = codes[u.which ? (head * (S >> 3) + (block >> 3)) * a.DP + c0 + r
                           : ((head * S + slot) * a.DP + c0) >> 3];
  }
  T *out0 = (T *)(u.which ? a.v : a.k) +
            (u.which ? u.b * a.v_stride[0] + u.h * a.v_stride[1]
                     : u.b * a.k_stride[0] + u.h * a.k_stride[1]);
  const int64_t step = u.which ? a.v_stride[2] : a.k_stride[2];
#pragma unroll
  for (int k = 0; k < UN; ++k) {
    const int slot = u.slot0 + 8 * k + tok_of(r);
    if (u.which) w[k] = transpose8(w[k], r);
    if (slot < u.first || slot >= u.end) continue;
    const bool held = slot >= 0 && slot < len;
    const float s = __builtin_bit_cast(float, word[k] << 16);
    const float m = __builtin_bit_cast(float, word[k] & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = u.which ? 4 * e : 4 * ((e >> 1) + 4 * (e & 1));
      x[e] = held ? fmaf((float)((w[k] >> at) & 15), s, m) : 0.f;
    }
    T *out = out0 + (slot - u.first) * step;
    if (VEC) {
      if (c0 < d) {
        typedef typename VecOf<T>::type V;
#pragma unroll
        for (int i = 0; i < 8 / VecOf<T>::N; ++i) {
          V v;
#pragma unroll
          for (int e = 0; e < VecOf<T>::N; ++e) v[e] = from_f32<T>(x[i * VecOf<T>::N + e]);
          *reinterpret_cast<V *>(out + c0 + i * VecOf<T>::N) = v;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < d) out[c0 + e] = from_f32<T>(x[e]);
    }
  }
}

}  // namespace

void launch_kv4_io(const Kv4Io &a, int dtype, hipStream_t s) {
  // Blocks of 8 tokens a wave: with four it requests 4 KB of bf16 before it waits.  512 tokens, write
  // and read: 21 and 19 us with four, 22 and 20 with two, 26 and 25 with one.  Short calls want the
  // waves: one token 3.5 and 3.4 us with one, 3.8 and 4.0 with four.
  const int un = a.nblk >= 8 ? 4 : 1;
  const int64_t waves = ((int64_t)((a.nblk + un - 1) / un) * a.H) << a.g_shift;
  const dim3 grid((unsigned)((waves + 3) / 4), (unsigned)a.B, 2), block(256);
  // 16-byte accesses need whole 8-channel pieces at 16-byte aligned places
  auto aligned = [&](const void *p, const int64_t *st) {
    const int64_t per = dtype == GNLP_BF16 ? 8 : 4;
    return ((uintptr_t)p & 15) == 0 && st[0] % per == 0 && st[1] % per == 0 && st[2] % per == 0;
  };
  const bool vec = a.d % 8 == 0 && aligned(a.k, a.k_stride) && aligned(a.v, a.v_stride);
#define GO3(KERNEL, T, VEC) \
  do { \
    if (un == 4) hipLaunchKernelGGL((KERNEL<T, VEC, 4>), grid, block, 0, s, a); \
    else hipLaunchKernelGGL((KERNEL<T, VEC, 1>), grid, block, 0, s, a); \
  } while (0)
#define GO(KERNEL) \
  do { \
    if (dtype == GNLP_BF16) { \
      if (vec) GO3(KERNEL, bf16, true); \
      else GO3(KERNEL, bf16, false); \
    } else { \
      if (vec) GO3(KERNEL, float, true); \
      else GO3(KERNEL, float, false); \
    } \
  } while (0)
  if (a.write) GO(kv4_write_kernel);
  else GO(kv4_read_kernel);
#undef GO
#undef GO3
}

}  // namespace gnlp
