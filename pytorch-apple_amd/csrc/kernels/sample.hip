// One token per row of logits from a given uniform number, after temperature, top-k, top-p and min-p.
//
// k_sample_*: one workgroup of 1024 threads per row. With w = exp((l - max) / T), tokens ranked by (logit descending,
// index ascending), the kept ones are those not after the k-th, not after the last whose preceding weights sum to less
// than top_p of them all, and of w >= min_p; the token is the first by index at which the running sum of the kept
// weights passes u times their sum.
//   * Weights are integers: w rounded to 2^-shift (2^-44 up to 2^18 tokens), from a double exponential of relative
//     error below 2^-42. Their sums are exact in any order, so threads, waves and atomics add in whichever order they
//     come and a call gives the same token every time; in 32-bit floats a border between two tokens would move by 1e-7
//     of the sum, and with 150,000 borders a row in a thousand draws another token.
//   * No sort. A token's rank is its 64-bit key, the logit's order-preserving bits over the inverted index (no two
//     alike). The rows's first pass takes the largest; the second counts and weighs tokens in 2048 bins of (max - l)
//     covering 32 T, where weights end (e^-32 rounds to 0: what lies past is in the last bin and weighs nothing). The
//     bin in which the k-th token or the top-p sum falls is then split again by key, 2048 ways a pass, until at most
//     1024 tokens are in it: those are gathered and ranked against each other. Typical rows need no second split; rows
//     of equal logits take two more.
//   * The last passes weigh the kept tokens in groups of 64 sixteen-byte pieces, find the group by a scan and the
//     token within the group by one wave.
#include "common.h"

#define SM_T 1024              // threads
#define SM_BINS 2048
#define SM_LIST 1024           // tokens ranked against each other
#define SM_GROUPS 4096         // groups of 64 pieces: vocab <= SM_GROUPS * 64 * (4 | 8)

typedef unsigned long long u64;

// order-preserving bits of a logit: NaN as -inf, -0 as +0
__device__ __forceinline__ uint32_t sm_order(float v) {
  v = v != v ? -INFINITY : v == 0.f ? 0.f : v;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float sm_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 sm_key(float v, int idx) {
  return ((u64)sm_order(v) << 32) | (uint32_t)~(uint32_t)idx;
}

// 2^(x) for x <= 0 as an integer of 2^-shift, and as a double (0 below 2^-50)
__device__ __forceinline__ double sm_exp2(double x) {
  const double n = __builtin_rint(x), f = (x - n) * 0.69314718055994530942;   // |f| <= 0.347: f^11 / 11! < 2.2e-13
  double p = 2.7557319223985890653e-07;                                       // 1/10!
  p = __builtin_fma(p, f, 2.7557319223985890653e-06);
  p = __builtin_fma(p, f, 2.4801587301587301587e-05);
  p = __builtin_fma(p, f, 1.9841269841269841270e-04);
  p = __builtin_fma(p, f, 1.3888888888888888889e-03);
  p = __builtin_fma(p, f, 8.3333333333333333333e-03);
  p = __builtin_fma(p, f, 4.1666666666666666667e-02);
  p = __builtin_fma(p, f, 1.6666666666666666667e-01);
  p = __builtin_fma(p, f, 0.5);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_fma(p, f, 1.0);
  const bool none = !(x > -50.0);
  const long long e = none ? 0 : (long long)(int)n;
  const double r = __builtin_bit_cast(double, __builtin_bit_cast(long long, p) + (e << 52));
  return none ? 0.0 : r;
}

struct SmRow {
  float max;
  double inv_t2;   // log2(e) / T
  int shift;
  float bin_scale;
  __device__ __forceinline__ double weight(float v) const {
    // (equal to the largest, also where both are infinite: 1)
    return v == max ? 1.0 : sm_exp2(((double)v - (double)max) * inv_t2);
  }
  __device__ __forceinline__ u64 units(double w) const {
    // adding 2^52 rounds to an integer and leaves it in the low bits of the mantissa
    const double s = w * __builtin_bit_cast(double, (u64)(1023 + shift) << 52) + 4503599627370496.0;
    return __builtin_bit_cast(u64, s) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ int bin(float v) const {
    const float d = v == max ? 0.f : (max - v) * bin_scale;
    return d < (float)(SM_BINS - 1) ? (int)d : SM_BINS - 1;   // NaN too: the last
  }
};

__device__ __forceinline__ u64 sm_wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ u64 sm_wave_max(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}
// inclusive scan over the wave
__device__ __forceinline__ u64 sm_wave_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}
// exclusive scan over the workgroup, and the total; red: 16 words
__device__ __forceinline__ u64 sm_block_scan(u64 v, u64* red, u64* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 inc = sm_wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  u64 base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SM_T / 64; ++w) {
    base += w < wave ? red[w] : 0;
    all += red[w];
  }
  *total = all;
  return base + inc - v;
}
__device__ __forceinline__ u64 sm_block_max(u64 v, u64* red) {
  v = sm_wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < SM_T / 64; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

// Pieces of 16 bytes of a row, aligned in memory whatever the vocabulary: piece c holds tokens c * E - skew ..,
// those outside the row given as -inf with an index past 2^31 (key below every token's).
template <int DT>
struct SmPieces {
  static constexpr int E = DT == HS_F32 ? 4 : 8;
  const char* base;   // aligned address at or before the row's start
  int skew, vocab, count;
  __device__ __forceinline__ SmPieces(const SampleArgs& a, int row) {
    constexpr int SZ = DT == HS_F32 ? 4 : 2;
    const char* p = (const char*)a.logits + (long long)row * a.vocab * SZ;
    skew = (int)(((uintptr_t)p & 15) / SZ);
    base = p - skew * SZ;
    vocab = a.vocab;
    count = (skew + vocab + E - 1) / E;
  }
  __device__ __forceinline__ int first(int c) const { return c * E - skew; }
  __device__ __forceinline__ void load(int c, float (&v)[E]) const {
    const int i0 = first(c);
    if (i0 >= 0 && i0 + E <= vocab) {
      const uint4 q = *(const uint4*)(base + (long long)c * 16);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      if constexpr (DT == HS_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = gm_lo<DT>(w[j]), v[2 * j + 1] = gm_hi<DT>(w[j]);
      }
    } else {   // the row's ends, and nothing past them
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = i0 + j;
        v[j] = i >= 0 && i < vocab ? ld_f(base, (long long)c * E + j, DT) : -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = v[j] != v[j] ? -INFINITY : v[j];
  }
  // f(value, index) for every token of the row, by all threads
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int c = threadIdx.x; c < count; c += SM_T) {
      float v[E];
      load(c, v);
      const int i0 = first(c);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i0 + j >= 0 && i0 + j < vocab) f(v[j], i0 + j);
    }
  }
};

template <int DT>
__device__ __forceinline__ void sample_body(const SampleArgs& a) {
  __shared__ u64 red[16];
  __shared__ u64 wsum[SM_GROUPS];        // bins' weights, then groups'
  __shared__ unsigned cnt[SM_BINS];
  __shared__ u64 lkey[SM_LIST], lw[SM_LIST];
  __shared__ unsigned ln;
  __shared__ u64 pick[3];
  static_assert(SM_GROUPS >= SM_BINS, "");
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SmPieces<DT> x(a, row);

  u64 best = 0;
  x.each([&](float v, int i) {
    const u64 k = sm_key(v, i);
    best = k > best ? k : best;
  });
  best = sm_block_max(best, red);
  const float T = a.temperature[row], top_p = a.top_p[row], min_p = a.min_p[row], u = a.u[row];
  const int top_k = a.top_k[row];
  SmRow r;
  r.max = sm_value((uint32_t)(best >> 32));
  if (!(T > 0.f) || r.max == -INFINITY) {   // the first ranked
    if (tid == 0) a.out[row] = (int)~(uint32_t)best;
    return;
  }
  r.inv_t2 = 1.4426950408889634074 / (double)T;
  r.shift = a.shift;
  r.bin_scale = (float)SM_BINS / 32.f / T;

  u64 cut = 0;   // kept: keys >= cut
  // One threshold: the smallest key with fewer than `need` before it (counting tokens or weights, of those above the
  // present cut).
  auto threshold = [&](bool weigh, u64 need) {
    // first split, by bins of (max - l); later ones by key bits: members are keys in [lo, hi], bin (hi - key) >> sh
    u64 lo = 0, hi = best, before = 0;
    int sh = -1;
    while (true) {
      for (int i = tid; i < SM_BINS; i += SM_T) cnt[i] = 0, wsum[i] = 0;
      __syncthreads();
      x.each([&](float v, int i) {
        const u64 k = sm_key(v, i);
        if (k < cut || k < lo || k > hi) return;
        const int bin = sh < 0 ? r.bin(v) : (int)((hi - k) >> sh);
        atomicAdd(&cnt[bin], 1u);
        if (weigh) {
          const u64 w = r.units(r.weight(v));
          if (w) atomicAdd(&wsum[bin], w);
        }
      });
      __syncthreads();
      const u64 c0 = cnt[2 * tid], c1 = cnt[2 * tid + 1], w0 = wsum[2 * tid], w1 = wsum[2 * tid + 1];
      const u64 v0 = weigh ? w0 : c0, v1 = weigh ? w1 : c1;
      u64 total;
      const u64 ex = before + sm_block_scan(v0 + v1, red, &total);
      if (tid == 0) pick[0] = ~0ull;
      __syncthreads();
      if (ex < need && ex + v0 >= need) pick[0] = 2 * tid, pick[1] = ex, pick[2] = c0;
      else if (ex + v0 < need && ex + v0 + v1 >= need) pick[0] = 2 * tid + 1, pick[1] = ex + v0, pick[2] = c1;
      __syncthreads();
      const u64 bin = pick[0], at = pick[1], members = pick[2];
      // none, or the last bin, whose tokens weigh nothing: all stay
      if (bin == ~0ull || (sh < 0 && bin == SM_BINS - 1)) return;
      before = at;
      auto in = [&](float v, u64 k) {
        return k >= cut && k >= lo && k <= hi && (sh < 0 ? (u64)r.bin(v) : (hi - k) >> sh) == bin;
      };
      if (members <= SM_LIST) {
        if (tid == 0) ln = 0;
        __syncthreads();
        x.each([&](float v, int i) {
          const u64 k = sm_key(v, i);
          if (!in(v, k)) return;
          const unsigned s = atomicAdd(&ln, 1u);
          lkey[s] = k;
          lw[s] = weigh ? r.units(r.weight(v)) : 1;
        });
        __syncthreads();
        u64 mine = ~0ull;   // the largest of the inverted keys that stay
        const int n = (int)ln;
        if (tid < n) {
          u64 b = before;
          const u64 k = lkey[tid];
          for (int j = 0; j < n; ++j) b += lkey[j] > k ? lw[j] : 0;
          if (b < need) mine = k;
        }
        // the smallest key that stays
        const u64 m = ~sm_block_max(~mine, red);
        cut = m > cut ? m : cut;
        return;
      }
      // the bin's range of keys, and the next split of it
      u64 kmax = 0, kmin = 0;
      x.each([&](float v, int i) {
        const u64 k = sm_key(v, i);
        if (!in(v, k)) return;
        kmax = k > kmax ? k : kmax;
        kmin = ~k > kmin ? ~k : kmin;
      });
      kmax = sm_block_max(kmax, red);
      kmin = ~sm_block_max(kmin, red);
      lo = kmin, hi = kmax;
      const int bits = 64 - __builtin_clzll((hi - lo) | 1);
      sh = bits > 11 ? bits - 11 : 0;
    }
  };
  if (top_k > 0 && top_k < a.vocab) threshold(false, (u64)top_k);
  // groups of 64 pieces: the weights of their kept tokens
  const int groups = (x.count + 63) / 64;
  const double floor_w = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;
  auto kept = [&](float v, int i, double least) -> u64 {
    if (i < 0 || i >= a.vocab || sm_key(v, i) < cut) return 0;
    const double w = r.weight(v);
    return w >= least ? r.units(w) : 0;
  };
  auto weigh_groups = [&](double least) {
    __syncthreads();
    for (int g = wave; g < groups; g += SM_T / 64) {
      u64 s = 0;
      const int c = g * 64 + lane;
      if (c < x.count) {
        float v[SmPieces<DT>::E];
        x.load(c, v);
#pragma unroll
        for (int j = 0; j < SmPieces<DT>::E; ++j) s += kept(v[j], x.first(c) + j, least);
      }
      s = sm_wave_sum(s);
      if (lane == 0) wsum[g] = s;
    }
    __syncthreads();
  };
  auto group_total = [&](u64& ex, u64 (&g)[SM_GROUPS / SM_T]) {
    u64 s = 0, total;
#pragma unroll
    for (int j = 0; j < SM_GROUPS / SM_T; ++j) {
      const int i = tid * (SM_GROUPS / SM_T) + j;
      g[j] = i < groups ? wsum[i] : 0;
      s += g[j];
    }
    ex = sm_block_scan(s, red, &total);
    return total;
  };
  u64 ex, g[SM_GROUPS / SM_T];
  if (top_p < 1.f) {
    if (!(top_p > 0.f)) {
      cut = best;
    } else {
      weigh_groups(0.0);
      const u64 total = group_total(ex, g);
      const u64 need = (u64)__builtin_ceil((double)top_p * (double)total);
      __syncthreads();
      if (need < total) threshold(true, need);
    }
  }
  weigh_groups(floor_w);
  const u64 total = group_total(ex, g);
  const double t = (double)u * (double)total;
  const u64 target = t > 0.0 ? (t < (double)total ? min((u64)t, total - 1) : total - 1) : 0;
  if (tid == 0) pick[0] = 0, pick[1] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < SM_GROUPS / SM_T; ++j) {
    if (ex <= target && ex + g[j] > target) pick[0] = tid * (SM_GROUPS / SM_T) + j, pick[1] = ex;
    ex += g[j];
  }
  __syncthreads();
  if (wave == 0) {
    const int c = (int)pick[0] * 64 + lane;
    u64 w[SmPieces<DT>::E] = {}, s = 0;
    if (c < x.count) {
      float v[SmPieces<DT>::E];
      x.load(c, v);
#pragma unroll
      for (int j = 0; j < SmPieces<DT>::E; ++j) s += w[j] = kept(v[j], x.first(c) + j, floor_w);
    }
    u64 run = pick[1] + sm_wave_scan(s, lane) - s;
#pragma unroll
    for (int j = 0; j < SmPieces<DT>::E; ++j) {
      if (run <= target && run + w[j] > target) a.out[row] = x.first(c) + j;
      run += w[j];
    }
  }
}

extern "C" __global__ void __launch_bounds__(SM_T) k_sample_f32(const SampleArgs a) { sample_body<HS_F32>(a); }
extern "C" __global__ void __launch_bounds__(SM_T) k_sample_f16(const SampleArgs a) { sample_body<HS_F16>(a); }
extern "C" __global__ void __launch_bounds__(SM_T) k_sample_bf16(const SampleArgs a) { sample_body<HS_BF16>(a); }
