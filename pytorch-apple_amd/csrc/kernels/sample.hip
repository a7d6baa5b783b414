// One token per row of logits from a given uniform number, after temperature, top-k, top-p and min-p.
//
// With w = exp((l - max) / T), tokens ranked by (logit descending, index ascending), the kept ones are those not after
// the k-th, not after the last whose preceding weights sum to less than top_p of them all, and of w >= min_p; the token
// is the first by index at which the running sum of the kept weights passes u times their sum.
//   * Weights are integers: w rounded to 2^-shift (2^-44 up to 2^18 tokens), from a double exponential of relative
//     error below 2^-42. Their sums are exact in any order, so threads, waves and atomics add in whichever order they
//     come and a call gives the same token every time; in 32-bit floats a border between two tokens would move by 1e-7
//     of the sum, and with 150,000 borders a row in a thousand draws another token.
//   * No sort. A token's rank is its 64-bit key, the logit's order-preserving bits over the inverted index (no two
//     alike). A cut is a key; what is needed of the row to find it are the tokens near it.
//   * Rows are read twice, by many workgroups each, in four launches: _hist counts and weighs each part's tokens in
//     512 bins of l of width T / 16, on one grid for all parts of a row and down from the part's largest (after 32 T
//     weights round to 0, so the bins hold all that weigh), near enough to say where a cut lies; _merge adds the parts
//     up and finds the bins in which the k-th token and the end of the top-p sum lie; _collect sums the weights before
//     those bins, those that are kept for sure also in groups of 64 sixteen-byte pieces, and lists the tokens of
//     those bins; _pick ranks the listed ones (a few hundred to a few thousand), adds
//     the kept ones to their groups, finds the group by a scan and the token in it by one wave.
//     One row of 151,936 (bf16): 6 + 9 + 10 + 16 us, all waiting on memory and barriers, _pick most (16 waves of one
//     workgroup). 256 rows in float32: 39 + 10 + 58 + 17 us; _hist reads at 4.0 TB/s, _collect does some 45 instructions a
//     token, two thirds of them the double exponential.
//   * _pick alone does a row of few tokens, and one that the bins do not tell apart (more than SM_LIST tokens near the
//     cuts, or more than SM_PART_LIST in one part: equal logits; infinite ones): it splits the range of keys 2048 ways
//     a pass over the row until at most 256 tokens are left around the cut. 4,000 such tokens next to each other in
//     each of 256 rows: 407 us, 136 where they lie all over the row.
#include "common.h"

#define SM_T 1024              // threads of _pick
#define SM_TH 256              // of _hist and _collect
#define SM_MAX_PARTS 1024      // of a row
#define SM_BINS 512            // of width T / 16
#define SM_MAX_PER 8           // pieces of a part per thread, which stay in registers (SampleArgs.per)
#define SM_LIST 16384          // tokens of the bins around the cuts: a tenth of 150,000, as where their spread is T / 4
#define SM_PART_LIST 1024      // of them in one part (up to 2^14 tokens): where that is of 8 pieces in 16 bits, a row of
                               // 151,936 has 10 parts and lists 10,240 at most
#define SM_NEAR 4096           // of a row's list in LDS, if no more
#define SM_RANK 256            // tokens ranked against each other, four threads a token
#define SM_SPLIT 2048
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

// 2^x for -60 <= x <= 0
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
  return __builtin_amdgcn_ldexp(p, (int)n);
}

struct SmRow {
  float max;
  double inv_t2;   // log2(e) / T
  int shift;
  float scale;     // bins per unit of l
  __device__ __forceinline__ void init(float largest, float T, int sh) {
    max = largest, inv_t2 = 1.4426950408889634074 / (double)T, shift = sh, scale = 16.f / T;
  }
  // (2^-60 is 0 units, also for what is further off or no number)
  __device__ __forceinline__ double finite(float v) const { return sm_exp2(fmax(((double)v - (double)max) * inv_t2, -60.0)); }
  // (equal to the largest, also where both are infinite: 1)
  __device__ __forceinline__ double weight(float v) const { return v == max ? 1.0 : finite(v); }
  __device__ __forceinline__ u64 units(double w) const {
    // adding 2^52 rounds to an integer and leaves it in the low bits of the mantissa
    const double s = w * __builtin_bit_cast(double, (u64)(1023 + shift) << 52) + 4503599627370496.0;
    return __builtin_bit_cast(u64, s) & 0xFFFFFFFFFFFFFull;
  }
  // whether the grid tells values apart. Below 2^20 v * scale is off by at most a 16th of a bin, and what is SM_BINS
  // bins from the largest (e^-32 of it) still rounds to 0. A part's own bound is twice the row's, so that every part
  // that reaches into a row's bins has its own.
  __device__ __forceinline__ bool binned(float most) const {
    return scale > 0.f && scale < INFINITY && fabsf(max * scale) < most;
  }
  __device__ __forceinline__ int grid(float v) const {   // non-decreasing in v
    return (int)fminf(fmaxf(floorf(v * scale), -536870912.f), 536870912.f);
  }
};
// whether the row's first ranked token is the answer
__device__ __forceinline__ bool sm_greedy(float max, float T, int top_k, float top_p) {
  return !(T > 0.f) || max == -INFINITY || top_k == 1 || top_p <= 0.f;
}

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
template <typename N>
__device__ __forceinline__ N sm_wave_scan(N v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const N w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}
// exclusive scan over TH threads, and the total; red: TH / 64 words
template <int TH, typename N>
__device__ __forceinline__ N sm_block_scan(N v, N* red, N* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const N inc = sm_wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  N base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) {
    base += w < wave ? red[w] : 0;
    all += red[w];
  }
  *total = all;
  return base + inc - v;
}
template <int TH>
__device__ __forceinline__ u64 sm_block_max(u64 v, u64* red) {
  v = sm_wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

// Pieces of 16 bytes of a row, aligned in memory whatever the vocabulary: piece c holds tokens c * E - skew .., those
// outside the row given as -inf.
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
  __device__ __forceinline__ bool whole(int c) const { return c < count && first(c) >= 0 && first(c) + E <= vocab; }
  // the piece's bits; a piece at the row's ends comes token by token, and nothing past them is read
  __device__ __forceinline__ uint4 bits(int c) const {
    if (whole(c)) return *(const uint4*)(base + (long long)c * 16);
    constexpr uint32_t NINF = DT == HS_F32 ? 0xff800000u : DT == HS_BF16 ? 0xff80u : 0xfc00u;
    uint32_t w[4] = {};
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = first(c) + j;
      const bool in = c < count && i >= 0 && i < vocab;
      if constexpr (DT == HS_F32) w[j] = in ? ((const uint32_t*)base)[(long long)c * E + j] : NINF;
      else w[j / 2] |= (in ? (uint32_t)((const uint16_t*)base)[(long long)c * E + j] : NINF) << (16 * (j & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ static void values(uint4 q, float (&v)[E]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < E; ++j) {
      float x;
      if constexpr (DT == HS_F32) x = __uint_as_float(w[j]);
      else x = j & 1 ? gm_hi<DT>(w[j / 2]) : gm_lo<DT>(w[j / 2]);
      v[j] = x != x ? -INFINITY : x;
    }
  }
  __device__ __forceinline__ bool in(int i) const { return i >= 0 && i < vocab; }
  // f(value, index) for every token of the row, by SM_T threads
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int c = threadIdx.x; c < count; c += SM_T) {
      float v[E];
      values(bits(c), v);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (in(first(c) + j)) f(v[j], first(c) + j);
    }
  }
};

// ------------------------------------------------------------------ counts and weights of a part, by bins

// A token of weight w (<= 1) as what it adds to its bin: 1 above 49 bits for the sum of weights in units of 2^-34, at
// most SM_MAX_PER * SM_TH * 8 = 2^14 tokens of them. (Adding 2^52 + 2^49 rounds to an integer in the mantissa's low bits.)
__device__ __forceinline__ u64 sm_pack(float w) {
  const double s = __builtin_fma((double)w, 17179869184.0, 4503599627370496.0 + 562949953421312.0);
  return __builtin_bit_cast(u64, s) & 0xFFFFFFFFFFFFFull;
}

// grid (parts, rows). The part stays in registers between its maximum and its bins. The bins' weights only say where
// the cuts lie, so 32-bit exponentials do (arguments to -46, 4e-6 off; rounded to 2^-35, at most 2^14 times against a
// largest of 1: 5e-7): one atomic a token, and half the instructions of a double.
template <int DT>
__device__ __forceinline__ void sample_hist_body(const SampleArgs& a) {
  constexpr int E = SmPieces<DT>::E, N = SM_MAX_PER;
  __shared__ u64 red[SM_TH / 64];
  __shared__ u64 bins[SM_BINS];
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const SmPieces<DT> x(a, row);
  const int c0 = part * a.per * SM_TH + tid;
  uint4 q[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < a.per) q[i] = x.bits(c0 + i * SM_TH);
  const float T = a.temperature[row], top_p = a.top_p[row];
  const int top_k = a.top_k[row];
  if (part == 0 && tid == 0) a.listed[row] = 0, a.sums[2 * row] = a.sums[2 * row + 1] = 0;
#pragma unroll
  for (int i = 0; i < SM_BINS / SM_TH; ++i) bins[i * SM_TH + tid] = 0;
  u64 best = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= a.per) break;
    float v[E];
    x.values(q[i], v);
    float m = v[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < E; ++j)
      if (v[j] > m) m = v[j], at = j;
    // (a token outside the row, -inf, wins over none that is in it)
    const int i0 = x.first(c0 + i * SM_TH);
    if (m == -INFINITY) at = max(0, -i0);
    const u64 k = x.in(i0 + at) ? sm_key(m, i0 + at) : 0;
    best = k > best ? k : best;
  }
  best = sm_block_max<SM_TH>(best, red);
  const long long me = (long long)row * a.parts + part;
  if (tid == 0) a.best[me] = best;
  SmRow r;
  r.init(sm_value((uint32_t)(best >> 32)), T, a.shift);
  const bool k = top_k > 0 && top_k < a.vocab, p = top_p < 1.f;
  if (sm_greedy(r.max, T, top_k, top_p) || !(k || p) || !r.binned(2097152.f)) return;
  const int top = r.grid(r.max);
  const float c = 1.44269504088896340736f / T;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= a.per) break;
    float v[E];
    x.values(q[i], v);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int bin = top - r.grid(v[j]);
      if (bin < SM_BINS) atomicAdd(&bins[bin], sm_pack(__builtin_amdgcn_exp2f((v[j] - r.max) * c)));
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SM_BINS / SM_TH; ++i) a.bins[me * SM_BINS + i * SM_TH + tid] = bins[i * SM_TH + tid];
}

// ------------------------------------------------------------------ the bins of the cuts

// grid (rows). Threads i and 512 + i hold the row's bin i, which counts down from its largest value's: one adds up the
// even parts, the other the odd ones, sixteen parts' loads in flight (one at a time takes 0.7 us a part).
extern "C" __global__ void __launch_bounds__(SM_T) k_sample_merge(const SampleArgs a) {
  static_assert(SM_T == 2 * SM_BINS && SM_MAX_PARTS <= SM_T, "");
  __shared__ u64 red[SM_T / 64];
  __shared__ unsigned redc[SM_T / 64];
  __shared__ double redw[SM_T / 64];
  __shared__ int off[SM_MAX_PARTS + 32];    // the parts' first bins, in the row's
  __shared__ double f[SM_MAX_PARTS + 32];   // their largest tokens' weights
  __shared__ unsigned oddc[SM_BINS];
  __shared__ double oddw[SM_BINS];
  __shared__ int kb, kr, kn, plo, phi, pn;
  __shared__ double ahead, in_kb, base;
  const int row = blockIdx.x, tid = threadIdx.x, bin = tid & (SM_BINS - 1), odd = tid / SM_BINS;
  const u64 key = tid < a.parts ? a.best[(long long)row * a.parts + tid] : 0;
  const float T = a.temperature[row], top_p = a.top_p[row];
  const int top_k = a.top_k[row];
  const u64 best = sm_block_max<SM_T>(key, red);
  SmRow r;
  r.init(sm_value((uint32_t)(best >> 32)), T, a.shift);
  const bool k = top_k > 0 && top_k < a.vocab, p = top_p < 1.f;
  SampleRow s;
  s.best = best, s.kb = -1, s.kr = s.kn = s.pn = s.pad = 0, s.plo = s.phi = -1;
  s.mode = sm_greedy(r.max, T, top_k, top_p) ? 0 : !r.binned(1048576.f) ? 3 : k || p ? 2 : 1;
  if (s.mode != 2) {
    if (tid == 0) a.row[row] = s;
    return;
  }
  const int top = r.grid(r.max);
  const float most = sm_value((uint32_t)(key >> 32));
  const bool any = key != 0 && most != -INFINITY;
  off[tid] = any ? min(top - r.grid(most), SM_BINS) : SM_BINS;
  f[tid] = any ? r.weight(most) : 0.0;
  if (tid < 32) off[SM_MAX_PARTS + tid] = SM_BINS, f[SM_MAX_PARTS + tid] = 0.0;
  if (tid == 0) kb = -1, kr = kn = pn = 0, ahead = in_kb = 0.0, plo = phi = SM_BINS;
  __syncthreads();
  unsigned c = 0;
  double w = 0.0;
  for (int q0 = odd; q0 < a.parts; q0 += 32) {
    u64 n[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {   // (a part that does not reach the bin is read at its first and left out)
      const long long at = ((long long)row * a.parts + min(q0 + 2 * j, a.parts - 1)) * SM_BINS;
      const int i = max(bin - off[q0 + 2 * j], 0);
      n[j] = a.bins[at + i];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (bin >= off[q0 + 2 * j]) c += (unsigned)(n[j] >> 49), w += f[q0 + 2 * j] * (double)(n[j] & ((1ull << 49) - 1));
  }
  if (odd) oddc[bin] = c, oddw[bin] = w;
  __syncthreads();
  c = odd ? 0 : c + oddc[bin];
  w = odd ? 0.0 : w + oddw[bin];
  unsigned call;
  double wall;
  const unsigned c0 = sm_block_scan<SM_T>(c, redc, &call);
  const double w0 = sm_block_scan<SM_T>(w, redw, &wall);
  if (k && c0 < (unsigned)top_k && c0 + c >= (unsigned)top_k) {
    kb = bin, kr = top_k - (int)c0, kn = (int)c, ahead = w0;
    // the bin's first kr tokens weigh at least their share of it, and at most all
    in_kb = w, base = w * (double)kr / (double)c;
  }
  __syncthreads();
  s.kb = kb, s.kr = kr, s.kn = kn;
  s.plo = s.phi = kb;
  if (p) {
    // (the slack is several times the error of the bins' weights)
    const double lo = kb < 0 ? wall : ahead + base, up = kb < 0 ? wall : ahead + in_kb;
    const double plow = (double)top_p * lo * (1.0 - 2e-5), pup = (double)top_p * up * (1.0 + 2e-5);
    if (!odd && w0 < plow && w0 + w >= plow) atomicMin(&plo, bin);
    if (!odd && w0 < pup && w0 + w >= pup) atomicMin(&phi, bin);
    __syncthreads();
    const int last = kb < 0 ? SM_BINS - 1 : kb;
    s.plo = min(plo, last), s.phi = min(phi, last);
    if (c && bin >= s.plo && bin <= s.phi) atomicAdd(&pn, (int)c);
    __syncthreads();
    s.pn = pn;
  } else if (kb < 0) {
    s.mode = 1;   // (fewer tokens weigh anything than k)
  }
  if (tid == 0) a.row[row] = s;
}

// ------------------------------------------------------------------ kept weights by groups, tokens near the cuts

// grid (parts, rows): wave i of a part takes its groups i, i + 4, ..., all loads in flight together.
template <int DT>
__device__ __forceinline__ void sample_collect_body(const SampleArgs& a) {
  constexpr int E = SmPieces<DT>::E, N = SM_MAX_PER;
  __shared__ u64 list[SM_PART_LIST];
  __shared__ unsigned n, at;
  __shared__ u64 red[2 * SM_TH / 64];
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SmPieces<DT> x(a, row);
  const int c0 = part * a.per * SM_TH + tid;
  uint4 q[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < a.per) q[i] = x.bits(c0 + i * SM_TH);
  const SampleRow s = a.row[row];
  if (s.mode == 0 || s.mode == 3) return;
  const float T = a.temperature[row], min_p = a.min_p[row];
  const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;
  SmRow r;
  r.init(sm_value((uint32_t)(s.best >> 32)), T, a.shift);
  const int top = r.grid(r.max), sure = s.mode == 1 ? SM_BINS : s.plo;
  // top-p needs the weights of the bins before plo, and of those before the k-th token's
  const bool p = s.mode == 2 && a.top_p[row] < 1.f;
  const int before = !p ? sure : s.kb < 0 ? SM_BINS : s.kb;   // (>= sure)
  u64 base = 0, ahead = 0;
  if (tid == 0) n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= a.per) break;
    const int c = c0 + i * SM_TH;
    float v[E];
    x.values(q[i], v);
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int bin = top - r.grid(v[j]);   // (outside the row: -inf, past every bin)
      if (bin < before) {
        const double w = r.finite(v[j]);
        const u64 in = r.units(w);
        ahead += in;
        if (bin < sure) base += in, sum += w >= least ? in : 0;
      }
      if (bin >= sure && s.mode == 2 && bin < SM_BINS && (bin <= s.phi || bin == s.kb)) {
        const unsigned k = atomicAdd(&n, 1u);
        if (k < SM_PART_LIST) list[k] = sm_key(v[j], x.first(c) + j);
      }
    }
    sum = sm_wave_sum(sum);
    const int g = (part * a.per + i) * (SM_TH / 64) + wave;
    if (lane == 0 && g < a.ngroups) a.groups[(long long)row * a.ngroups + g] = sum;
  }
  if (p) {
    base = sm_wave_sum(base), ahead = sm_wave_sum(ahead);
    if (lane == 0) red[wave] = base, red[SM_TH / 64 + wave] = ahead;
  }
  __syncthreads();
  if (p && tid < 2) {
    u64 w = 0;
#pragma unroll
    for (int i = 0; i < SM_TH / 64; ++i) w += red[tid * (SM_TH / 64) + i];
    if (w) atomicAdd(&a.sums[2 * row + tid], w);
  }
  if (n == 0) return;
  // (more than the part lists: the row's count goes past SM_LIST, and k_sample_pick does it without the list)
  if (tid == 0) at = atomicAdd(&a.listed[row], n > SM_PART_LIST ? SM_LIST + 1 : n);
  __syncthreads();
  for (int i = tid; i < (int)min(n, (unsigned)SM_PART_LIST); i += SM_TH)
    if (at + i < SM_LIST) a.list[(long long)row * SM_LIST + at + i] = list[i];
}

// ------------------------------------------------------------------ the token

struct SmCut {
  u64 red[SM_T / 64];
  unsigned cnt[SM_SPLIT];
  u64 sum[SM_SPLIT];
  u64 key[SM_RANK], w[SM_RANK];
  unsigned n;
  u64 pick[3];
};

// The smallest key in [lo, hi] with less than `need` before it: `before`, and the weights (1 each where `weigh` is
// false) of the larger keys in [lo, hi]. `members`: no less than there are (their range is then
// [lo, hi] as given), or 0, not known. each(f) calls f(key) for the keys of its thread; 0: none has it.
template <typename F>
__device__ __forceinline__ u64 sm_cut(SmCut& t, F each, const SmRow& r, bool weigh, u64 need, u64 before, u64 lo, u64 hi,
                                  u64 members) {
  const int tid = threadIdx.x;
  auto units = [&](u64 k) { return weigh ? r.units(r.weight(sm_value((uint32_t)(k >> 32)))) : 1ull; };
  __syncthreads();
  if (members == 0) {
    u64 least = ~0ull, most = 0;
    each([&](u64 k) {
      if (k < lo || k > hi) return;
      least = k < least ? k : least, most = k > most ? k : most, ++members;
    });
    members = sm_wave_sum(members), least = ~sm_wave_max(~least), most = sm_wave_max(most);
    if ((tid & 63) == 0) {
      const int w = tid >> 6;
      t.key[w] = least, t.key[SM_T / 64 + w] = most, t.w[w] = members;
    }
    __syncthreads();
    members = 0;
#pragma unroll
    for (int w = 0; w < SM_T / 64; ++w) {
      least = t.key[w] < least ? t.key[w] : least, most = t.key[SM_T / 64 + w] > most ? t.key[SM_T / 64 + w] : most;
      members += t.w[w];
    }
    if (members == 0) return 0;
    lo = least, hi = most;
    __syncthreads();
  }
  while (members > SM_RANK) {
    const int bits = 64 - __builtin_clzll((hi - lo) | 1), sh = max(bits - 11, 0);
    for (int i = tid; i < SM_SPLIT; i += SM_T) t.cnt[i] = 0, t.sum[i] = 0;
    __syncthreads();
    each([&](u64 k) {
      if (k < lo || k > hi) return;
      const int bin = (int)((hi - k) >> sh);
      atomicAdd(&t.cnt[bin], 1u);
      const u64 w = weigh ? units(k) : 0;
      if (w) atomicAdd(&t.sum[bin], w);
    });
    __syncthreads();
    const u64 c0 = t.cnt[2 * tid], c1 = t.cnt[2 * tid + 1];
    const u64 v0 = weigh ? t.sum[2 * tid] : c0, v1 = weigh ? t.sum[2 * tid + 1] : c1;
    u64 total;
    const u64 ex = before + sm_block_scan<SM_T>(v0 + v1, t.red, &total);
    if (tid == 0) t.pick[0] = ~0ull;
    __syncthreads();
    if (ex < need && ex + v0 >= need) t.pick[0] = 2 * tid, t.pick[1] = ex, t.pick[2] = c0;
    else if (ex + v0 < need && ex + v0 + v1 >= need) t.pick[0] = 2 * tid + 1, t.pick[1] = ex + v0, t.pick[2] = c1;
    __syncthreads();
    const u64 bin = t.pick[0];
    if (bin == ~0ull) return 0;
    members = t.pick[2];
    before = t.pick[1];
    const u64 h = hi - (bin << sh);
    lo = hi - lo >= ((bin + 1) << sh) ? h - ((1ull << sh) - 1) : lo;
    hi = h;
    __syncthreads();
  }
  if (tid == 0) t.n = 0;
  __syncthreads();
  each([&](u64 k) {
    if (k < lo || k > hi) return;
    const unsigned s = atomicAdd(&t.n, 1u);
    t.key[s] = k;
    t.w[s] = units(k);
  });
  __syncthreads();
  // four threads a key, each over a quarter of the others
  static_assert(SM_T == 4 * SM_RANK, "");
  u64 mine = ~0ull;
  const int n = (int)t.n, me = tid >> 2;
  if (me < n) {
    u64 b = 0;
    const u64 k = t.key[me];
#pragma unroll 4
    for (int j = tid & 3; j < n; j += 4) b += t.key[j] > k ? t.w[j] : 0;
    b += __shfl_xor(b, 1, 64);
    b += __shfl_xor(b, 2, 64);
    if (before + b < need) mine = k;
  }
  const u64 found = ~sm_block_max<SM_T>(~mine, t.red);
  return found == ~0ull ? 0 : found;
}

// A key below those of the grid's place g, and not below those of place g - 2 (whose values are off by a 16th, and the
// quotient by an 8th, of a place).
__device__ __forceinline__ u64 sm_low(const SmRow& r, int g) { return (u64)sm_order(((float)g - 0.5f) / r.scale) << 32; }

// grid (rows)
template <int DT>
__device__ __forceinline__ void sample_pick_body(const SampleArgs& a) {
  constexpr int E = SmPieces<DT>::E, PER = SM_GROUPS / SM_T;
  __shared__ SmCut t;
  __shared__ u64 groups[SM_GROUPS];
  __shared__ u64 near[SM_NEAR];
  static_assert(SM_SPLIT == 2 * SM_T && SM_RANK <= SM_T, "");
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SmPieces<DT> x(a, row);
  const float T = a.temperature[row], top_p = a.top_p[row], min_p = a.min_p[row], u = a.u[row];
  const int top_k = a.top_k[row];
  const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;
  const bool k = top_k > 0 && top_k < a.vocab;
  SampleRow s;
  unsigned n = 0;
  if (a.best) {
    s = a.row[row];
    n = a.listed[row];
  } else {
    u64 best = 0;
    x.each([&](float v, int i) {
      const u64 key = sm_key(v, i);
      best = key > best ? key : best;
    });
    s.best = sm_block_max<SM_T>(best, t.red);
    s.mode = sm_greedy(sm_value((uint32_t)(s.best >> 32)), T, top_k, top_p) ? 0 : 3;
  }
  if (s.mode == 0) {
    if (tid == 0) a.out[row] = (int)~(uint32_t)s.best;
    return;
  }
  SmRow r;
  r.init(sm_value((uint32_t)(s.best >> 32)), T, a.shift);
  const int ng = (x.count + 63) / 64;
  u64 cut = 0;   // kept: keys >= cut
  auto kept = [&](float v, int i, double at_least) -> u64 {
    if (!x.in(i) || sm_key(v, i) < cut) return 0;
    const double w = r.weight(v);
    return w >= at_least ? r.units(w) : 0;
  };
  const bool listed = s.mode == 1 || (s.mode == 2 && n <= SM_LIST);
  if (listed) {
    for (int g = tid; g < ng; g += SM_T) groups[g] = a.groups[(long long)row * a.ngroups + g];
    if (s.mode == 2) {
      const u64* far = a.list + (long long)row * SM_LIST;
      const bool in = n <= SM_NEAR;
      if (in)
        for (int i = tid; i < (int)n; i += SM_T) near[i] = far[i];
      __syncthreads();
      auto list = [&](int i) { return in ? near[i] : far[i]; };
      const int top = r.grid(r.max);
      auto each = [&](int b0, int b1, auto f) {   // keys of bins b0 .. b1
        for (int i = tid; i < (int)n; i += SM_T) {
          const u64 key = list(i);
          const int bin = top - r.grid(sm_value((uint32_t)(key >> 32)));
          if (bin >= b0 && bin <= b1) f(key);
        }
      };
      u64 total = a.sums[2 * row + 1];
      if (s.kb >= 0) {
        cut = sm_cut(t, [&](auto f) { each(s.kb, s.kb, f); }, r, false, (u64)s.kr, 0, sm_low(r, top - s.kb),
                     min(s.best, sm_low(r, top - s.kb + 2)), (u64)s.kn);
        if (top_p < 1.f) {
          u64 w = 0, all;
          each(s.kb, s.kb, [&](u64 key) { w += key >= cut ? r.units(r.weight(sm_value((uint32_t)(key >> 32)))) : 0; });
          sm_block_scan<SM_T>(w, t.red, &all);
          total += all;
        }
      }
      if (top_p < 1.f) {
        const u64 need = (u64)__builtin_ceil((double)top_p * (double)total);
        const u64 c = sm_cut(t, [&](auto f) { each(s.plo, s.phi, f); }, r, true, need, a.sums[2 * row],
                             max(cut, sm_low(r, top - s.phi)), min(s.best, sm_low(r, top - s.plo + 2)), (u64)s.pn);
        cut = c > cut ? c : cut;
      }
      __syncthreads();
      for (int i = tid; i < (int)n; i += SM_T) {
        const u64 key = list(i);
        const int idx = (int)~(uint32_t)key;
        const u64 w = kept(sm_value((uint32_t)(key >> 32)), idx, least);
        if (w) atomicAdd(&groups[(idx + x.skew) / E / 64], w);
      }
    }
  } else {
    auto each = [&](auto f) { x.each([&](float v, int i) { f(sm_key(v, i)); }); };
    auto weigh = [&](double at_least) {
      __syncthreads();
      for (int g = wave; g < ng; g += SM_T / 64) {
        u64 w = 0;
        float v[E];
        x.values(x.bits(g * 64 + lane), v);
#pragma unroll
        for (int j = 0; j < E; ++j) w += kept(v[j], x.first(g * 64 + lane) + j, at_least);
        w = sm_wave_sum(w);
        if (lane == 0) groups[g] = w;
      }
      __syncthreads();
    };
    if (k) cut = sm_cut(t, each, r, false, (u64)top_k, 0, 0, s.best, 0);
    if (top_p < 1.f) {
      weigh(0.0);
      u64 w = 0, total;
      for (int g = tid; g < ng; g += SM_T) w += groups[g];
      sm_block_scan<SM_T>(w, t.red, &total);
      const u64 need = (u64)__builtin_ceil((double)top_p * (double)total);
      const u64 c = sm_cut(t, each, r, true, need, 0, cut, s.best, 0);
      cut = c > cut ? c : cut;
    }
    weigh(least);
  }
  __syncthreads();
  // the group in which the running sum passes u times the whole, and the token in it
  u64 g[PER], w = 0, total;
#pragma unroll
  for (int j = 0; j < PER; ++j) w += g[j] = tid * PER + j < ng ? groups[tid * PER + j] : 0;
  u64 ex = sm_block_scan<SM_T>(w, t.red, &total);
  const double want = (double)u * (double)total;
  const u64 target = want > 0.0 ? (want < (double)total ? min((u64)want, total - 1) : total - 1) : 0;
  if (tid == 0) t.pick[0] = 0, t.pick[1] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (ex <= target && ex + g[j] > target) t.pick[0] = tid * PER + j, t.pick[1] = ex;
    ex += g[j];
  }
  __syncthreads();
  if (wave == 0) {
    const int c = (int)t.pick[0] * 64 + lane;
    float v[E];
    x.values(x.bits(c), v);
    u64 p[E], sum = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) sum += p[j] = kept(v[j], x.first(c) + j, least);
    u64 run = t.pick[1] + sm_wave_scan(sum, lane) - sum;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (run <= target && run + p[j] > target) a.out[row] = x.first(c) + j;
      run += p[j];
    }
  }
}

#define SM_KERNELS(NAME, DT)                                                                                                  \
  extern "C" __global__ void __launch_bounds__(SM_TH) k_sample_hist_##NAME(const SampleArgs a) { sample_hist_body<DT>(a); }     \
  extern "C" __global__ void __launch_bounds__(SM_TH) k_sample_collect_##NAME(const SampleArgs a) { sample_collect_body<DT>(a); } \
  extern "C" __global__ void __launch_bounds__(SM_T) k_sample_pick_##NAME(const SampleArgs a) { sample_pick_body<DT>(a); }
SM_KERNELS(f32, HS_F32)
SM_KERNELS(f16, HS_F16)
SM_KERNELS(bf16, HS_BF16)
