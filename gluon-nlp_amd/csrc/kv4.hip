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
// lanes in three exchange steps.  Bound by memory: 2 or 4 bytes a value in (out), 0.5625 out (in).
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
// over the 8 lanes that hold one group: quad exchanges, then the mirror of the half row
__device__ __forceinline__ float min8(float x) {
  x = fminf(x, dpp<0xB1>(x));
  x = fminf(x, dpp<0x4E>(x));
  return fminf(x, dpp<0x141>(x));
}
__device__ __forceinline__ float max8(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  return fmaxf(x, dpp<0x141>(x));
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

struct Unit {      // what a wave works on
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
  u.on = blk < a.nblk && blk <= (uint32_t)((0x7ffffff0 - u.first) >> 3);
  u.slot0 = (int)((u.first & ~7) + (u.on ? 8 * blk : 0));
  u.on = u.on && u.slot0 < u.end;
  return u;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(float (&x)[8], const T *p, int c0, int d) {
  if (VEC) {
    if (c0 < d) {
      if (sizeof(T) == 2) {
        const bf16x8 v = *reinterpret_cast<const bf16x8 *>(p + c0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
      } else {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(p + c0);
        const f32x4 w = *reinterpret_cast<const f32x4 *>(p + c0 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = v[e]; x[4 + e] = w[e]; }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < d) x[e] = to_f32(p[c0 + e]);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4Io a) {
  const int lane = threadIdx.x & 63;
  const Unit u = unit_of(a);
  if (!u.on) return;
  const int r = lane >> 3, c = lane & 7, S = (int)a.S, d = (int)a.d;
  const int slot = u.slot0 + tok_of(r);
  const bool live = slot >= u.first && slot < u.end && slot >= 0 && slot < S;
  const uint64_t on = __ballot(live);
  if (on == 0) return;
  const int c0 = u.grp * 64 + 8 * c;
  const int64_t head = (int64_t)u.b * a.H + u.h;
  uint32_t *codes = (uint32_t *)(u.which ? a.v_codes : a.k_codes);
  uint32_t *par = (uint32_t *)(u.which ? a.v_par : a.k_par);
  const T *src = (const T *)(u.which ? a.v : a.k) +
                 (u.which ? u.b * a.v_stride[0] + u.h * a.v_stride[1]
                          : u.b * a.k_stride[0] + u.h * a.k_stride[1]);
  const int64_t step = u.which ? a.v_stride[2] : a.k_stride[2];

  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8<T, VEC>(x, src + (slot - u.first) * step, c0, d);
  // a block that this call stores in part: nibbles of the other tokens are kept
  uint32_t *word_at = u.which ? codes + (head * (S >> 3) + (u.slot0 >> 3)) * a.DP + c0 + r
                              : codes + (((head * S + slot) * a.DP + c0) >> 3);
  uint32_t keep = 0xffffffffu, old = 0;
  if (u.which && on != ~0ull) {
    keep = 0;
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if ((on >> (8 * t)) & 1) keep |= 0xfu << (4 * t);
    old = *word_at;
  }

  float lo = __builtin_inff(), hi = -__builtin_inff(), odd = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (VEC ? c0 < d : c0 + e < d) {
      lo = fminf(lo, x[e]);
      hi = fmaxf(hi, x[e]);
      odd = fmaf(x[e], 0.f, odd);             // NaN where a value is not finite
    }
  lo = min8(lo);
  hi = max8(hi);
  const uint64_t odds = __ballot(!(odd == 0.f));
  const bf16 sb = (bf16)((hi - lo) * (float)(1.0 / 15.0)), mb = (bf16)lo;
  float s = (float)sb;
  const float m = (float)mb, largest = 3.4028234663852886e38f;
  const bool bad = ((odds >> (lane & 56)) & 0xff) != 0 || !(s <= largest) || !(fabsf(m) <= largest);
  s = s < 1.1754943508222875e-38f ? 0.f : s;
  uint32_t word = (uint32_t)__builtin_bit_cast(uint16_t, (bf16)s) |
                  ((uint32_t)__builtin_bit_cast(uint16_t, mb) << 16);
  if (bad) { word = 0x7fc07fc0u; s = 0.f; }
  // Codes: (x - m) times the hardware's reciprocal of s, off by less than 1e-5 of a code, and the
  // true quotient where that is near a half (one value in a thousand of bf16 tensors, where exact
  // halves occur) or the reciprocal is not a normal number.  Adding 1.5 2^23 rounds to a whole
  // number in the low bits; what the high bits add up to in the packed word comes off at the end.
  constexpr float ROUND = 12582912.f;
  constexpr uint32_t HIGH = 0x4b400000u;
  const bool plain = s > 1e-36f && s < 1e36f;
  const float inv = plain ? __builtin_amdgcn_rcpf(s) : 0.f;
  uint32_t w = 0, high = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = x[e] - m;
    float y = __builtin_amdgcn_fmed3f(t * inv, 0.f, 15.f);
    float n = y + ROUND;
    if (fabsf(y - (n - ROUND)) > 0.4999f || (!plain && s > 0.f))
      n = fminf(fmaxf(t / s, 0.f), 15.f) + ROUND;
    const int at = u.which ? 4 * e : 4 * ((e >> 1) + 4 * (e & 1));
    w += __builtin_bit_cast(uint32_t, n) << at;
    high += HIGH << at;
  }
  w -= high;
  if (u.which) {
    w = transpose8(w, r);
    *word_at = (old & ~keep) | (w & keep);
  } else if (live) {
    *word_at = w;
  }
  if (live && c == 0) par[((head << a.g_shift) + u.grp) * S + slot] = word;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Io a) {
  const int lane = threadIdx.x & 63;
  const Unit u = unit_of(a);
  if (!u.on) return;
  const int r = lane >> 3, c = lane & 7, S = (int)a.S, d = (int)a.d;
  const int slot = u.slot0 + tok_of(r);
  const bool wanted = slot >= u.first && slot < u.end;
  int len = a.length ? bounded(load_len(a.length, a.length_dtype, u.b)) : S;
  len = len > S ? S : len;
  const bool held = slot >= 0 && slot < len;
  const int c0 = u.grp * 64 + 8 * c;
  const int64_t head = (int64_t)u.b * a.H + u.h;
  const uint32_t *codes = (const uint32_t *)(u.which ? a.v_codes : a.k_codes);
  const uint32_t *par = (const uint32_t *)(u.which ? a.v_par : a.k_par);
  uint32_t w = 0, word = 0;
  if (held) word = par[((head << a.g_shift) + u.grp) * S + slot];
  if (u.which == 0) {
    if (held) w = codes[((head * S + slot) * a.DP + c0) >> 3];
  } else {
    if (u.slot0 >= 0 && u.slot0 < S)
      w = codes[(head * (S >> 3) + (u.slot0 >> 3)) * a.DP + c0 + r];
    w = transpose8(w, r);
  }
  if (!wanted) return;
  const float s = __builtin_bit_cast(float, word << 16);
  const float m = __builtin_bit_cast(float, word & 0xffff0000u);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = u.which ? e : (e >> 1) + 4 * (e & 1);
    x[e] = held ? fmaf((float)((w >> (4 * at)) & 15), s, m) : 0.f;
  }
  T *out = (T *)(u.which ? a.v : a.k) +
           (u.which ? u.b * a.v_stride[0] + u.h * a.v_stride[1]
                    : u.b * a.k_stride[0] + u.h * a.k_stride[1]) +
           (slot - u.first) * (u.which ? a.v_stride[2] : a.k_stride[2]);
  if (VEC) {
    if (c0 < d) {
      if (sizeof(T) == 2) {
        bf16x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (bf16)x[e];
        *reinterpret_cast<bf16x8 *>(out + c0) = v;
      } else {
        *reinterpret_cast<f32x4 *>(out + c0) = (f32x4){x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4 *>(out + c0 + 4) = (f32x4){x[4], x[5], x[6], x[7]};
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < d) out[c0 + e] = from_f32<T>(x[e]);
  }
}

}  // namespace

void launch_kv4_io(const Kv4Io &a, int dtype, hipStream_t s) {
  const int64_t waves = ((int64_t)a.nblk * a.H) << a.g_shift;
  const dim3 grid((unsigned)((waves + 3) / 4), (unsigned)a.B, 2), block(256);
  // 16-byte accesses need whole 8-channel pieces at 16-byte aligned places
  auto aligned = [&](const void *p, const int64_t *st) {
    const int64_t per = dtype == GNLP_BF16 ? 8 : 4;
    return ((uintptr_t)p & 15) == 0 && st[0] % per == 0 && st[1] % per == 0 && st[2] % per == 0;
  };
  const bool vec = a.d % 8 == 0 && aligned(a.k, a.k_stride) && aligned(a.v, a.v_stride);
#define GO(KERNEL) \
  do { \
    if (dtype == GNLP_BF16) { \
      if (vec) hipLaunchKernelGGL((KERNEL<bf16, true>), grid, block, 0, s, a); \
      else hipLaunchKernelGGL((KERNEL<bf16, false>), grid, block, 0, s, a); \
    } else { \
      if (vec) hipLaunchKernelGGL((KERNEL<float, true>), grid, block, 0, s, a); \
      else hipLaunchKernelGGL((KERNEL<float, false>), grid, block, 0, s, a); \
    } \
  } while (0)
  if (a.write) GO(kv4_write_kernel);
  else GO(kv4_read_kernel);
#undef GO
}

}  // namespace gnlp
