// One step of a beam search on the device: the choice of the K best continuations of each item's K
// beams over the vocabulary, and the reordering of the decoding states that follows it, gfx950.
//
// Selection.  With z = outputs / temperature (sanitised: NaN counts as -inf, +inf as the largest
// finite number) a candidate of an unfinished beam k and token v scores
//   (prev[k] * lp_prev + z[k, v] - logsumexp(z[k])) / lp_new
// (logsumexp 0 when the outputs are log-probabilities already), a finished beam has one candidate,
// itself with its old score.  The K best of an item are returned in order, ties to the lowest index
// k V + v (finished beams: K V + k).  A beam whose previous score is not above -1e15 is dead: all
// its candidates count as -inf.
//
// Candidates of one beam are ordered by their logits alone, so the K best of every chunk of 4096 or
// 8192 logits are found first (beam_chunk_kernel, one pass over the logits, which also leaves the
// maximum and the sum of exponentials), and the few that are left are scored in 64 bits
// (beam_merge_kernel: beams that come near each other are told apart by the logsumexp's last
// digits).
//   The K best of a chunk: a wave's 64 lane maxima are bisected, by ballots over the high bits of an
//   order-preserving integer, for a bound that K / 4 lanes reach; the least of the four waves' bounds
//   leaves little more than K values, which a list in LDS ranks by counting.  Where ties overfill
//   the list (a masked or a constant row), the exact bound and the first K of its ties do it.
//   The merge does the same with the chunks' best candidates and reads on only in the lists that
//   reach its bound, all of them at once.
// Bound by memory (the logits once) and by the instructions of the pass: a logit's maximum, fma,
// exponential and sum, and 200 or so a wave on top.  128 rows of 250112 bfloat16 logits: 20 us
// (58 MB of beams that go on, 2.9 TB/s); 512 rows of 32128 float32: 18 us (53 MB); 4 rows 5.2 us.
// The merge is a chain of dependent loads, 5 us for one item, 10 for 8 items of 496 lists; more threads,
// deeper prefetches and a tighter bound made it no faster.
//
// Reordering.  out[row] = in[parent's row] for a list of tensors of any size, in one launch.  In
// place, a thread holds its 16 bytes of all K beams before it writes any, and rows that keep their
// place are not written.  Bound by memory: the chosen rows once, the changed rows once (24 tensors
// of 80 rows, 630 MB moved, in 116 us); in place with 5 beams, whose pieces take 174 registers, by the
// two waves a SIMD that this leaves (the same tensors, 538 MB moved, in 264 us).
#include "common.h"
#include "kernels.h"

namespace gnlp {
namespace {

constexpr int CAP = 512;                        // list of survivors
constexpr float NEG = -__builtin_inff();

// larger float <-> larger unsigned
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
// a number whose ordered() is at most `bits` (low bits of the integer cleared by the bisection)
__device__ __forceinline__ float unordered(uint32_t bits) {
  if (bits <= 0x007fffffu) return NEG;                  // (below every number: -inf)
  return __builtin_bit_cast(float, (bits & 0x80000000u) ? bits & 0x7fffffffu : ~bits);
}

// NaN counts as -inf, +inf as the largest number (by comparisons: a median of three with -inf is
// folded to a minimum, which is the largest number for a NaN)
__device__ __forceinline__ float sane(float x) {
  const float largest = 3.4028234663852886e38f;
  return x <= largest ? x : (x > largest ? largest : NEG);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_else(float other, float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
      __builtin_bit_cast(int, other), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float lane63(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float all_max(float x) {      // row shifts, then the rows' last lanes
  x = fmaxf(x, dpp_else<0x111, 0xf>(NEG, x));
  x = fmaxf(x, dpp_else<0x112, 0xf>(NEG, x));
  x = fmaxf(x, dpp_else<0x114, 0xf>(NEG, x));
  x = fmaxf(x, dpp_else<0x118, 0xf>(NEG, x));
  x = fmaxf(x, dpp_else<0x142, 0xa>(NEG, x));
  x = fmaxf(x, dpp_else<0x143, 0xc>(NEG, x));
  return lane63(x);
}
__device__ __forceinline__ float all_sum(float x) {
  x += dpp_else<0x111, 0xf>(0.f, x);
  x += dpp_else<0x112, 0xf>(0.f, x);
  x += dpp_else<0x114, 0xf>(0.f, x);
  x += dpp_else<0x118, 0xf>(0.f, x);
  x += dpp_else<0x142, 0xa>(0.f, x);
  x += dpp_else<0x143, 0xc>(0.f, x);
  return lane63(x);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double all_sum(double x) {
  x += dpp_or_zero<0x111, 0xf>(x);
  x += dpp_or_zero<0x112, 0xf>(x);
  x += dpp_or_zero<0x114, 0xf>(x);
  x += dpp_or_zero<0x118, 0xf>(x);
  x += dpp_or_zero<0x142, 0xa>(x);
  x += dpp_or_zero<0x143, 0xc>(x);
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// a bound, of the high bits of the keys down to LOW, that at least K of the wave's 64 keys reach (0
// if fewer than K are above 0)
template <int LOW>
__device__ __forceinline__ uint32_t wave_bound(uint32_t key, int K) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t next = bound | (1u << bit);
    if ((int)__popcll(__ballot(key >= next)) >= K) bound = next;
  }
  return bound;
}

__device__ __forceinline__ bool better(float x, uint32_t i, float y, uint32_t j) {
  return x > y || (x == y && i < j);
}

// p[i] by way of its aligned word: a scalar load, the same in all lanes
__device__ __forceinline__ bool flag_at(const uint8_t *p, int64_t i) {
  const uintptr_t at = (uintptr_t)(p + i);
  return (*reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3) >> (8 * (at & 3))) & 0xff;
}

__device__ __forceinline__ float max3(float a, float b, float c) {   // (fmaxf would quieten NaNs)
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(a) : "v"(b), "v"(c));
  return a;
}

// E: values of a thread
template <typename T, bool VEC, int E>
__global__ void __launch_bounds__(256, E == 32 && !VEC ? 4 : 8) beam_chunk_kernel(BeamSelect a) {
  __shared__ uint64_t list[CAP];           // ordered value above, complement of the index below
  __shared__ uint32_t sh_n, sh_bound[4], sh_same[4];
  __shared__ float sh_m[4], sh_s[4];
  constexpr int GROUP = 4;                 // values that are compared with the bound together
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.y;
  const uint32_t chunk = blockIdx.x, base = chunk * (256 * E), V = (uint32_t)a.V;
  if (a.finished && flag_at(a.finished, row)) return;
  const bool dead = !(a.scores[row] > -1e15f);
  const T *src = (const T *)a.outputs + row * a.row_stride;
  const int64_t slot = row * a.chunks + chunk;
  float *ox = a.cand_x + slot * a.K;
  int32_t *oi = a.cand_i + slot * a.K;
  if (dead) {                              // all of its candidates tie at -inf
    for (int r = tid; r < a.K; r += 256) {
      ox[r] = NEG;
      oi[r] = base + r < V ? (int32_t)(base + r) : -1;
    }
    if (tid < 2) a.stats[slot * 2 + tid] = tid ? 0.f : NEG;
    return;
  }
  if (tid == 0) sh_n = 0;

  // value e of a thread is element base + at(e)
  constexpr int PER = VEC ? 16 / (int)sizeof(T) : 1;
  auto at = [&](int e) -> uint32_t { return base + (e / PER) * (256 * PER) + tid * PER + e % PER; };
  float x[E], top[E / GROUP];
  const bool whole = base + 256 * E <= V;
  if (VEC && whole) {
    typename VecOf<T>::type w[E / PER];
#pragma unroll
    for (int v = 0; v < E / PER; ++v)
      w[v] = *reinterpret_cast<const typename VecOf<T>::type *>(src + at(v * PER));
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32((T)w[e / PER][e % PER]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = at(e) < V ? to_f32(src[at(e)]) : NEG;
  }
  auto tops = [&]() -> float {
    float most = NEG;
#pragma unroll
    for (int q = 0; q < E / GROUP; ++q) {
      top[q] = x[q * GROUP];
      top[q] = max3(top[q], x[q * GROUP + 1], x[q * GROUP + 2]);
      most = max3(most, top[q], x[q * GROUP + 3]);
      top[q] = fmaxf(top[q], x[q * GROUP + 3]);
    }
    return most;
  };
  float most = tops(), wm = all_max(most), s = 0.f;
  bool plain = fabsf(wm) * a.exp_scale < 4096.f;
  if (plain) {
    // exp2(x scale - c), c = wm scale rounded: one fma; what the rounding of c adds to every term
    // comes off the sum, r = wm scale - c exactly (at most 2^-13 here: 2^-r = 1 - r ln 2 to 4e-9)
    const float c = wm * a.exp_scale, r = fmaf(wm, a.exp_scale, -c);
#pragma unroll
    for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(fmaf(x[e], a.exp_scale, -c));
    s = all_sum(s) * (1.f - 0.6931471806f * r);
    plain = s == s;
  }
  if (!plain) {      // NaN, +inf, nothing but -inf, masks of -1e9 or of the type's lowest number
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = sane(x[e]);
    most = tops();
    wm = all_max(most);
    s = 0.f;
    if (wm > NEG) {
#pragma unroll
      for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((x[e] - wm) * a.exp_scale);
      s = all_sum(s);
    }
  }
  // A bound that K values reach: K / 4 lanes of each wave and so its least over the waves, or,
  // where the vocabulary ends before every lane has a value, K lanes of one.
  const bool full = V - base >= 256 * PER;
  const int of_wave = full ? (a.K + 3) / 4 : a.K;
  const uint32_t key = at(0) < V ? ordered(most) : 0u, bound = wave_bound<16>(key, of_wave);
  auto shared_bound = [&]() -> float {
    const uint32_t b0 = sh_bound[0], b1 = sh_bound[1], b2 = sh_bound[2], b3 = sh_bound[3];
    return unordered(full ? min(min(b0, b1), min(b2, b3)) : max(max(b0, b1), max(b2, b3)));
  };
  const bool alike = __all(most == wm);
  if (lane == 0) {
    sh_bound[wave] = bound;
    sh_same[wave] = alike;
    sh_m[wave] = wm;
    sh_s[wave] = s;
  }
  __syncthreads();
  if (tid == 0) {
    const float m = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
    float t = 0.f;
    for (int w = 0; w < 4; ++w)
      if (sh_m[w] > NEG) t += sh_s[w] * __builtin_amdgcn_exp2f((sh_m[w] - m) * a.exp_scale);
    a.stats[slot * 2] = m;
    a.stats[slot * 2 + 1] = t;
  }
  auto push = [&](float v, uint32_t i) {
    const uint32_t pos = atomicAdd(&sh_n, 1u);
    if (pos < CAP)                         // (v + 0: -0 and +0 are one value)
      list[pos] = ((uint64_t)ordered(v + 0.0f) << 32) | (uint32_t)~i;
  };
  // one largest value in every lane (a chunk that is masked throughout): nothing lies above it
  const bool constant = (sh_same[0] & sh_same[1] & sh_same[2] & sh_same[3]) && sh_m[0] == sh_m[1] &&
                        sh_m[0] == sh_m[2] && sh_m[0] == sh_m[3];
  uint32_t n = CAP + 1;
  if (!constant) {
    const float least = shared_bound();
#pragma unroll
    for (int q = 0; q < E / GROUP; ++q)
      if (top[q] >= least) {
#pragma unroll
        for (int e = q * GROUP; e < q * GROUP + GROUP; ++e)
          if (x[e] >= least && (whole || at(e) < V)) push(x[e], at(e));
      }
    __syncthreads();
    n = sh_n;
  }
  if (n > CAP) {
    // Ties overfill the list (a mask, a constant row): the same with the bound to its last bit, what
    // lies above it and, in the order of their indices, K of what equals it.
    float tie = sh_m[0];
    if (!constant) {
      const uint32_t last = wave_bound<0>(key, of_wave);
      __syncthreads();
      if (lane == 0) sh_bound[wave] = last;
      if (tid == 0) sh_n = 0;
      __syncthreads();
      tie = shared_bound();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > tie && (whole || at(e) < V)) push(x[e], at(e));
    }
    int ties = 0;
    for (int v = 0; v < E && ties < a.K; ++v) {
      const uint32_t i = base + v * 256 + tid;
      const bool is = i < V && sane(to_f32(src[i])) == tie;
      const uint64_t on = __ballot(is);
      __syncthreads();
      if (lane == 0) sh_bound[wave] = (uint32_t)__popcll(on);
      __syncthreads();
      int before = ties + (int)__popcll(on & ((1ull << lane) - 1));
      for (int w = 0; w < 4; ++w) {
        if (w < wave) before += (int)sh_bound[w];
        ties += (int)sh_bound[w];
      }
      if (is && before < a.K) push(tie, i);
    }
    __syncthreads();
    n = sh_n;
  }
  if (n <= CAP) {
    for (uint32_t c = tid; c < n; c += 256) {
      const uint64_t key = list[c];
      int rank = 0;
#pragma unroll 4
      for (uint32_t o = 0; o < n; ++o) rank += list[o] > key;
      if (rank < a.K) {
        ox[rank] = unordered((uint32_t)(key >> 32));
        oi[rank] = (int32_t)~(uint32_t)key;
      }
    }
    for (int r = (int)n + tid; r < a.K; r += 256) oi[r] = -1;
    return;
  }
  // still too many (values that differ in their last bits): K times the best of what is left, over
  // the whole workgroup
  __syncthreads();
  float tx = __builtin_inff();
  uint32_t ti = 0;
  float *lx = (float *)list;
  uint32_t *li = (uint32_t *)list + 4;
  for (int r = 0; r < a.K; ++r) {
    float bx = NEG;
    uint32_t bi = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t i = at(e);
      const bool left = i < V && (r == 0 || better(tx, ti, x[e], i));
      if (left && better(x[e], i, bx, bi)) { bx = x[e]; bi = i; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float yx = __shfl_xor(bx, o, 64);
      const uint32_t yi = __shfl_xor(bi, o, 64);
      if (better(yx, yi, bx, bi)) { bx = yx; bi = yi; }
    }
    __syncthreads();
    if (lane == 0) { lx[wave] = bx; li[wave] = bi; }
    __syncthreads();
    tx = lx[0];
    ti = li[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
      if (better(lx[w], li[w], tx, ti)) { tx = lx[w]; ti = li[w]; }
    if (tid == 0) { ox[r] = tx; oi[r] = (int32_t)ti; }   // 0xffffffff: none left
    if (ti == 0xffffffffu) {
      for (int q = r + 1 + tid; q < a.K; q += 256) oi[q] = -1;
      return;
    }
  }
}

__device__ __forceinline__ bool better(double x, int64_t i, double y, int64_t j) {
  return x > y || (x == y && i < j);
}

constexpr int MERGE = 512;                // threads of the merge

__global__ void __launch_bounds__(MERGE) beam_merge_kernel(BeamSelect a) {
  constexpr int LIST = 1024, WAVES = MERGE / 64;
  __shared__ double lse[BEAM_MAX], sx[LIST];     // lse: the maximum of z taken off
  __shared__ float peak[BEAM_MAX];
  __shared__ int64_t si[LIST];
  __shared__ uint32_t live[LIST], sh_n, sh_live, sh_bound[WAVES];
  __shared__ double bx4[WAVES];
  __shared__ int64_t bi4[WAVES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t item = blockIdx.x;
  const int K = a.K;
  const uint8_t *fin = a.finished ? a.finished + item * K : nullptr;
  const float *prevs = a.scores + item * K;
  const int64_t first = item * K * a.chunks;     // of the item's lists
  // list c = beam * chunks + chunk holds up to K candidates, best first; from K chunks on: a
  // finished beam, its own only candidate
  const uint32_t own = K * a.chunks, lists = own + K;
  if (tid == 0) { sh_n = 0; sh_live = 0; }
  // the lists' best candidates, requested before anything waits
  constexpr int AHEAD = 2;
  int32_t hv[AHEAD];
  float hz[AHEAD];
#pragma unroll
  for (int r = 0; r < AHEAD; ++r) {
    const uint32_t c = tid + r * MERGE;
    hv[r] = -1;
    hz[r] = NEG;
    if (c < own) {
      hv[r] = a.cand_i[(first + c) * K];
      hz[r] = a.cand_x[(first + c) * K];
    }
  }
  // ---- logsumexp of each beam from its chunks ----
  for (int k = wave; k < K; k += WAVES) {
    double out = 0;
    float m = 0.f;
    if (a.normalize && !(fin && fin[k])) {
      const float *st = a.stats + (first + k * a.chunks) * 2;
      const uint32_t c0 = lane;
      const float m0 = c0 < a.chunks ? st[2 * c0] : NEG, t0 = c0 < a.chunks ? st[2 * c0 + 1] : 0.f;
      m = m0;
      for (uint32_t c = lane + 64; c < a.chunks; c += 64) m = fmaxf(m, st[2 * c]);
      m = all_max(m);
      double t = m0 > NEG ? (double)(t0 * __builtin_amdgcn_exp2f((m0 - m) * a.exp_scale)) : 0.0;
      for (uint32_t c = lane + 64; c < a.chunks; c += 64)
        if (st[2 * c] > NEG)
          t += (double)(st[2 * c + 1] * __builtin_amdgcn_exp2f((st[2 * c] - m) * a.exp_scale));
      t = all_sum(t);
      if (m > NEG) out = log(t);
      else m = 0.f;
    }
    if (lane == 0) {
      lse[k] = out;
      peak[k] = m;
    }
  }
  double lp_prev = a.lp_prev, lp_new = a.lp_new;
  if (a.step) {
    const double s = (double)load_len(a.step, a.step_dtype, 0);
    lp_prev = pow((a.length_base + s - 1.0) / (a.length_base + 1.0), a.alpha);
    lp_new = pow((a.length_base + s) / (a.length_base + 1.0), a.alpha);
  }
  const double per_lp = 1.0 / lp_new;
  __syncthreads();
  // an index: beam above, token below (finished beams: K above, beam below), in the order of k V + v
  const int64_t none = 0x7fffffffffffffffLL;
  // candidate (token v, logit z) of list c -> score and index (index `none`: there is none)
  auto rate = [&](uint32_t c, int32_t v, float z, double &x, int64_t &i) {
    x = -__builtin_inf();
    i = none;
    const bool self = c >= own;
    const uint32_t k = self ? c - own : c / a.chunks;
    const bool done = fin && fin[k];
    const float prev = prevs[k];
    const bool dead = !(prev > -1e15f);
    if (self) {
      if (done) {
        i = ((int64_t)K << 32) | k;
        if (!dead) x = (double)prev;
      }
    } else if (!done && v >= 0) {
      i = ((int64_t)k << 32) | (uint32_t)v;
      if (z > NEG && !dead)
        x = ((double)prev * lp_prev +
             (((double)z - (double)peak[k]) * a.inv_temperature - lse[k])) * per_lp;
    }
    if (!(x == x)) x = -__builtin_inf();   // (penalties of a step on the device out of range)
  };
  auto get = [&](uint32_t c, int j, double &x, int64_t &i) {
    int32_t v = -1;
    float z = NEG;
    if (c < own) {
      v = a.cand_i[(first + c) * K + j];
      z = a.cand_x[(first + c) * K + j];
    }
    rate(c, v, z, x, i);
    if (c >= own && j > 0) i = none;
  };
  // ---- a bound that K lists' best candidates reach ----
  double mx = -__builtin_inf(), hx[AHEAD];
  bool any = false, has[AHEAD];
#pragma unroll
  for (int r = 0; r < AHEAD; ++r) {
    const uint32_t c = tid + r * MERGE;
    int64_t i = none;
    hx[r] = -__builtin_inf();
    if (c < lists) rate(c, hv[r], hz[r], hx[r], i);
    has[r] = i != none;
    any |= has[r];
    mx = fmax(mx, hx[r]);
  }
  for (uint32_t c = tid + AHEAD * MERGE; c < lists; c += MERGE) {
    double x;
    int64_t i;
    get(c, 0, x, i);
    any |= i != none;
    mx = fmax(mx, x);
  }
  const uint32_t key = any ? (uint32_t)(ordered(mx) >> 32) : 0u, bound = wave_bound<8>(key, K);
  if (lane == 0) sh_bound[wave] = bound;
  __syncthreads();
  uint32_t least = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) least = max(least, sh_bound[w]);
  // ---- the lists whose best candidate reaches it, then all of their candidates at once ----
  auto keep = [&](uint32_t c, double x, bool is) {
    if (is && (uint32_t)(ordered(x) >> 32) >= least) {
      const uint32_t pos = atomicAdd(&sh_live, 1u);
      if (pos < LIST) live[pos] = c;
    }
  };
  uint32_t nlive, found;
  for (int again = 0;; ++again) {
#pragma unroll
    for (int r = 0; r < AHEAD; ++r) keep(tid + r * MERGE, hx[r], has[r]);
    for (uint32_t c = tid + AHEAD * MERGE; c < lists; c += MERGE) {
      double x;
      int64_t i;
      get(c, 0, x, i);
      keep(c, x, i != none);
    }
    __syncthreads();
    nlive = sh_live;
    if (nlive <= LIST)
      for (uint32_t q = tid; q < nlive * (uint32_t)K; q += MERGE) {
        const uint32_t l = q / (uint32_t)K;
        double x;
        int64_t i;
        get(live[l], (int)(q - l * K), x, i);
        if (i != none && (uint32_t)(ordered(x) >> 32) >= least) {
          const uint32_t pos = atomicAdd(&sh_n, 1u);
          if (pos < LIST) { sx[pos] = x; si[pos] = i; }
        }
      }
    __syncthreads();
    found = sh_n;
    // (ranking is quadratic)
    const bool fits = nlive <= LIST && found <= LIST / 4;
    if (again || fits) {
      if (again && found < (uint32_t)K) nlive = LIST + 1;   // (-inf is among the K best)
      break;
    }
    // too many, most likely of -inf (dead beams, masks): once more without those, and above what
    // K / 8 lanes of every wave reach
    const uint32_t every = wave_bound<8>(key, (K + WAVES - 1) / WAVES);
    __syncthreads();
    if (lane == 0) sh_bound[wave] = every;
    if (tid == 0) { sh_n = 0; sh_live = 0; }
    __syncthreads();
    uint32_t shared = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) shared = min(shared, sh_bound[w]);
    least = max(max(least, shared), 0x00100000u);
  }
  auto put = [&](int rank, double x, int64_t i) {
    const int64_t to = item * K + rank;
    const bool was = (i >> 32) == K;
    const int32_t k = was ? (int32_t)i : (int32_t)(i >> 32), v = was ? -1 : (int32_t)i;
    a.out_scores[to] = (float)x;
    a.out_parents[to] = k;
    a.out_tokens[to] = v;
    a.out_finished[to] = was || (a.has_eos && v == a.eos);
  };
  if (nlive <= LIST && found <= LIST) {
    for (uint32_t c = tid; c < found; c += MERGE) {
      const double x = sx[c];
      const int64_t i = si[c];
      int rank = 0;
#pragma unroll 4
      for (uint32_t o = 0; o < found; ++o) rank += better(sx[o], si[o], x, i);
      if (rank < K) put(rank, x, i);
    }
    return;
  }
  // ties overfill a list: K times the best of what is left
  double tx = __builtin_inf();
  int64_t ti = -1;
  for (int r = 0; r < K; ++r) {
    double bx = -__builtin_inf();
    int64_t bi = none;
    for (uint32_t c = tid; c < lists; c += MERGE)
      for (int j = 0; j < K; ++j) {
        double x;
        int64_t i;
        get(c, j, x, i);
        if (i == none) break;
        if (r > 0 && !better(tx, ti, x, i)) continue;      // (taken)
        if (better(x, i, bx, bi)) { bx = x; bi = i; }
        break;                                             // (the best that the list has left)
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double yx = __shfl_xor(bx, o, 64);
      const int64_t yi = __shfl_xor((long long)bi, o, 64);
      if (better(yx, yi, bx, bi)) { bx = yx; bi = yi; }
    }
    __syncthreads();
    if (lane == 0) { bx4[wave] = bx; bi4[wave] = bi; }
    __syncthreads();
    tx = bx4[0];
    ti = bi4[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
      if (better(bx4[w], bi4[w], tx, ti)) { tx = bx4[w]; ti = bi4[w]; }
    if (tid == 0) put(r, tx, ti);
  }
}

// ---- reordering ----
// Pieces of 16 bytes that a thread requests before it writes: 630 MB in 118 us with 4, 120 with 2,
// 193 with 1, 222 with 8.
constexpr int REORDER_UNROLL = 4;

template <int VB> struct Piece;
template <> struct Piece<16> { typedef f32x4 type; };
template <> struct Piece<4> { typedef float type; };
template <> struct Piece<1> { typedef uint8_t type; };

// pieces of a segment that the row's length covers
template <int VB>
__device__ __forceinline__ uint32_t live_pieces(const Reorder &a, const ReorderEntry &e,
                                                int64_t row) {
  const uint32_t all = (uint32_t)(e.seg_bytes / VB);
  if (!a.length || e.slots_per_unit == 0) return all;
  int64_t n = load_len(a.length, a.length_dtype, row);
  n = n < 0 ? 0 : (n > (1LL << 30) ? 1LL << 30 : n);
  const uint32_t units = ((uint32_t)n + (uint32_t)e.slots_per_unit - 1) / (uint32_t)e.slots_per_unit;
  const int64_t used = ((int64_t)units * e.unit_bytes + VB - 1) / VB;
  return used < all ? (uint32_t)used : all;
}
__device__ __forceinline__ int parent_of(const Reorder &a, int64_t row) {
  const int64_t p = load_len(a.parents, a.parents_dtype, row);
  return (int)(p < 0 ? 0 : (p >= a.K ? a.K - 1 : p));
}

// Source and destination apart: a thread moves REORDER_UNROLL pieces of one row, or, where a row's
// segment is short (flat), of a run of pieces over rows.
template <int VB>
__device__ __forceinline__ void reorder_apart(const Reorder &a, const ReorderEntry &e,
                                              uint32_t block) {
  typedef typename Piece<VB>::type P;
  constexpr int UN = REORDER_UNROLL;
  const uint32_t rows = (uint32_t)(a.N * a.K), pieces = (uint32_t)(e.seg_bytes / VB);
  const uint32_t nb = (uint32_t)e.nb;
  uint32_t rest = block / nb;
  const uint32_t first = (block - rest * nb) * (256 * UN) + threadIdx.x;
  P v[UN];
  if (!e.flat) {
    const uint32_t next = rest / rows, row = rest - next * rows;
    const uint32_t outer = next / (uint32_t)e.nseg, seg = next - outer * (uint32_t)e.nseg;
    const int64_t off = outer * e.outer_stride + seg * e.seg_stride;
    const uint32_t from = row / (uint32_t)a.K * (uint32_t)a.K + parent_of(a, row);
    const uint32_t live = live_pieces<VB>(a, e, from);
    const P *src = (const P *)((const char *)e.src + off + from * e.row_stride);
    P *dst = (P *)((char *)e.dst + off + row * e.row_stride);
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (first + u * 256 < live) v[u] = src[first + u * 256];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (first + u * 256 < live) dst[first + u * 256] = v[u];
    return;
  }
  const uint32_t outer = rest / (uint32_t)e.nseg, seg = rest - outer * (uint32_t)e.nseg;
  const int64_t off = outer * e.outer_stride + seg * e.seg_stride;
  int64_t to[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const uint32_t at = first + u * 256, row = at / pieces, p = at - row * pieces;
    to[u] = -1;
    if (row < rows) {
      const uint32_t from = row / (uint32_t)a.K * (uint32_t)a.K + parent_of(a, row);
      if (p < live_pieces<VB>(a, e, from)) {
        v[u] = *(const P *)((const char *)e.src + off + from * e.row_stride + (int64_t)p * VB);
        to[u] = off + row * e.row_stride + (int64_t)p * VB;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < UN; ++u)
    if (to[u] >= 0) *(P *)((char *)e.dst + to[u]) = v[u];
}

// In place: a thread holds one piece of all K <= KM rows of an item before it writes any.
template <int VB, int KM>
__device__ __forceinline__ void reorder_in_place(const Reorder &a, const ReorderEntry &e,
                                                 uint32_t block) {
  typedef typename Piece<VB>::type P;
  const uint32_t items = (uint32_t)a.N, pieces = (uint32_t)(e.seg_bytes / VB);
  const uint32_t nb = (uint32_t)e.nb;
  uint32_t rest = block / nb;
  uint32_t p = (block - rest * nb) * 256 + threadIdx.x, item = 0;
  if (e.flat) {
    item = p / pieces;
    p -= item * pieces;
  } else {
    const uint32_t next = rest / items;
    item = rest - next * items;
    rest = next;
  }
  if (item >= items || p >= pieces) return;
  const uint32_t outer = rest / (uint32_t)e.nseg, seg = rest - outer * (uint32_t)e.nseg;
  const int64_t r0 = (int64_t)item * a.K;
  char *at = (char *)e.dst + outer * e.outer_stride + seg * e.seg_stride + r0 * e.row_stride +
             (int64_t)p * VB;
  P v[KM];
  uint32_t moves = 0;
#pragma unroll
  for (int k = 0; k < KM; ++k)
    if (k < a.K) {
      const int f = parent_of(a, r0 + k);
      if (f != k && p < live_pieces<VB>(a, e, r0 + f)) {
        v[k] = *(const P *)(at + f * e.row_stride);
        moves |= 1u << k;
      }
    }
#pragma unroll
  for (int k = 0; k < KM; ++k)
    if ((moves >> k) & 1) *(P *)(at + k * e.row_stride) = v[k];
}

// KM = 0: source and destination apart
template <int KM>
__global__ void __launch_bounds__(256) reorder_kernel(Reorder a) {
  uint32_t block = blockIdx.x;
  int i = 0;
  while (i + 1 < a.n && block >= (uint32_t)a.e[i].blocks) block -= (uint32_t)a.e[i++].blocks;
  const ReorderEntry &e = a.e[i];
  if (KM == 0) {
    if (e.piece == 16) reorder_apart<16>(a, e, block);
    else if (e.piece == 4) reorder_apart<4>(a, e, block);
    else reorder_apart<1>(a, e, block);
  } else {
    if (e.piece == 16) reorder_in_place<16, KM ? KM : 1>(a, e, block);
    else if (e.piece == 4) reorder_in_place<4, KM ? KM : 1>(a, e, block);
    else reorder_in_place<1, KM ? KM : 1>(a, e, block);
  }
}

}  // namespace

// Values of a thread: 64 bytes, 32 of bfloat16 where that still gives every CU a few workgroups.
// (128 rows of 250112 bfloat16 logits: 20 us, 22 with 16, and the merge 10 us instead of 13; 512
// rows of 32128 float32: 18 us, 20 with 32.)
static int chunk_values(int64_t rows, int64_t V, int dtype) {
  return dtype == GNLP_BF16 && rows * ((V + 8191) / 8192) >= 1024 ? 32 : 16;
}

size_t beam_workspace_bytes(int64_t rows, int64_t V, int K) {     // for either dtype
  const int64_t ch = 256 * 16, slots = rows * ((V + ch - 1) / ch);
  return (size_t)slots * (8 + 8 * (size_t)K);
}

void launch_beam_select(BeamSelect a, int64_t items, int dtype, void *ws, hipStream_t s) {
  const int64_t rows = items * a.K;
  const int values = chunk_values(rows, a.V, dtype);
  a.chunks = (uint32_t)((a.V + 256 * values - 1) / (256 * values));
  a.stats = (float *)ws;
  a.cand_x = a.stats + rows * a.chunks * 2;
  a.cand_i = (int32_t *)(a.cand_x + rows * a.chunks * a.K);
  const int per = dtype == GNLP_BF16 ? 8 : 4;
  const bool vec = ((uintptr_t)a.outputs & 15) == 0 && a.row_stride % per == 0 && a.V % per == 0;
  const dim3 grid(a.chunks, (unsigned)rows), block(256);
#define GO(T, E) \
  do { \
    if (vec) hipLaunchKernelGGL((beam_chunk_kernel<T, true, E>), grid, block, 0, s, a); \
    else hipLaunchKernelGGL((beam_chunk_kernel<T, false, E>), grid, block, 0, s, a); \
  } while (0)
  if (dtype == GNLP_BF16) {
    if (values == 32) GO(bf16, 32);
    else GO(bf16, 16);
  } else {
    GO(float, 16);
  }
#undef GO
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)items), dim3(MERGE), 0, s, a);
}

// The caller has filled everything but piece and blocks.
bool launch_reorder(Reorder a, bool in_place, hipStream_t s) {
  int64_t total = 0;
  for (int i = 0; i < a.n; ++i) {
    ReorderEntry &e = a.e[i];
    // (a length that ends inside a piece copies the whole piece: the slots behind it are free)
    const uint64_t all = (uint64_t)(uintptr_t)e.src | (uint64_t)(uintptr_t)e.dst |
                         (uint64_t)e.outer_stride | (uint64_t)e.row_stride |
                         (uint64_t)e.seg_stride | (uint64_t)e.seg_bytes;
    e.piece = (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : 1;
    const int64_t pieces = e.seg_bytes / e.piece, rows = in_place ? a.N : a.N * a.K;
    const int64_t un = in_place ? 1 : REORDER_UNROLL;
    // short segments (4 time-major states of 64 steps of 512 rows of 1536 bytes, 340 MB moved): 77 us
    // so, 176 with a workgroup for each; in place 51 and 57 with 4 beams, 98 and 185 with 8
    e.flat = pieces < 256 * un && rows * pieces < (1LL << 31);
    const int64_t span = e.flat ? rows * pieces : pieces;
    e.nb = (span + 256 * un - 1) / (256 * un);
    e.blocks = e.nb * (e.flat ? 1 : rows) * e.nseg * e.outer;
    if (pieces >= (1LL << 31) || e.blocks > 0x7fffffffLL) return false;
    total += e.blocks;
  }
  if (total > 0x7fffffffLL) return false;
  const dim3 grid((unsigned)total), block(256);
  if (!in_place) hipLaunchKernelGGL(reorder_kernel<0>, grid, block, 0, s, a);
  else if (a.K <= 4) hipLaunchKernelGGL(reorder_kernel<4>, grid, block, 0, s, a);
  else if (a.K <= 8) hipLaunchKernelGGL(reorder_kernel<8>, grid, block, 0, s, a);
  else if (a.K <= 16) hipLaunchKernelGGL(reorder_kernel<16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(reorder_kernel<BEAM_MAX>, grid, block, 0, s, a);
  return true;
}

}  // namespace gnlp
