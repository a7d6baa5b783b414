// Paged K/V caches: append with rotation, and causal attention of packed rows over the pages.
//
// Rows of the packed new tokens belong to sequences (q_start), sequences hold kv_len positions, position p of
// sequence b lies in row p % page_size of page table[b][p / page_size]. Pages hold the queries' type, or e4m3 bytes
// with a power of two per position and K/V head (F8 in what follows). The metadata lies on the device and is
// taken as it comes: whatever it holds, no kernel here reads or writes outside its tensors (a row of no
// sequence is padding; a position before 0, past the table or in a page outside the pool has no place).
#include "common.h"

// Sequence of row `row` (B for none), by one wave: the number of q_start[1 ..] that are <= row.
__device__ __forceinline__ int pg_sequence(const int* q_start, int B, int row, int lane) {
  int n = 0;
  for (int i = 0; i < B; i += 64) n += __popcll(__ballot(i + lane < B && q_start[1 + min(i + lane, B - 1)] <= row));
  return n;
}

// Whether q_start descends somewhere (no batch), by one wave.
__device__ __forceinline__ bool pg_descends(const int* q_start, int B, int lane) {
  bool down = false;
  for (int i = lane; i < B; i += 64) down |= q_start[i + 1] < q_start[i];
  return __ballot(down) != 0;
}

// Position of row `row` of a sequence of `kv` positions whose rows end before `end`. Both may be any number: a position
// far below 0 stays there.
__device__ __forceinline__ int pg_position(int kv, int end, int row) {
  return (int)max((long long)kv - ((long long)end - row), -(1ll << 30));
}

// Page of position pos of sequence b, or -1 where it has no place.
__device__ __forceinline__ int pg_page(const int* table, int b, int M, int page_size, long long pages, int pos) {
  if (pos < 0 || pos / page_size >= M) return -1;
  const int page = table[(long long)b * M + pos / page_size];
  return page >= 0 && page < pages ? page : -1;
}

// place of a position's power of two in pages of 8 bits
__device__ __forceinline__ long long pg_scale_at(long long page, int h, int KVH, int page_size, int row) {
  return (page * KVH + h) * page_size + row;
}

// 2^(b - 127); 255 is NaN, 0 is 0
__device__ __forceinline__ float pg_scale(unsigned b) { return __uint_as_float(b == 255u ? 0x7fc00000u : b << 23); }

// The byte of the power of two with which a head of largest finite magnitude `most` is quantised: the smallest s >= 2^-100
// with most <= 448 s = 1.75 2^8 s. With most = 1.m 2^x it is 2^(x - 8), or twice that where 1.m > 1.75.
__device__ __forceinline__ unsigned pg_quant_byte(float most) {
  const unsigned u = __float_as_uint(fmaxf(most, 2.0194839e-28f));   // 2^-92
  return (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
}
// its inverse (27 <= byte <= 247)
__device__ __forceinline__ float pg_quant_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
// |x| of a finite x, else 0
__device__ __forceinline__ float pg_finite(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

// ------------------------------------------------------------------ append

#define PG_APPEND_R 256   // rotated dims of k_paged_append_bf16, _f16

// k_paged_append_any: one workgroup per row, one element pair (or one element past R) per thread and step; any
// type, head size and strides. x'_j = x_j c - x_{j + R/2} d, x'_{j + R/2} = x_{j + R/2} c + x_j d with c, d the scaled
// cosine and sine of position * inv_freq_j, the product in double: in fp32 the angle of position 100,000 is off by
// 4e-3. One rounding, of the result.
extern "C" __global__ void __launch_bounds__(256) k_paged_append_any(const PagedAppendArgs a) {
  __shared__ int place[3];   // sequence, position, page
  const int row = blockIdx.x, tid = threadIdx.x;
  if (tid < 64) {
    const int b = pg_sequence(a.q_start, a.B, row, tid);
    const bool real = b < a.B && row >= a.q_start[0];
    const int pos = real ? pg_position(a.kv_len[b], a.q_start[b + 1], row) : 0;
    if (tid == 0) place[0] = real ? b : -1, place[1] = pos, place[2] = real ? pg_page(a.table, b, a.M, a.page_size, a.pages, pos) : -1;
  }
  __syncthreads();
  const int pos = place[1], page = place[2], half = a.R / 2;
  const bool real = place[0] >= 0;
  const long long slot = page < 0 ? 0 : page * a.page_stride + (pos % a.page_size) * a.row_stride;
  const int per = half + a.D - a.R;   // steps of one head: pairs, then single elements
  for (int i = tid; i < (a.H + a.KVH) * per; i += 256) {
    const int h = i / per, e = i % per;
    const bool isq = h < a.H;
    const int hk = h - a.H;
    const void* src = isq ? a.q : a.k;
    void* dst = isq ? a.q_out : a.k_pages;
    const long long so = isq ? row * a.q_rs + h * a.q_hs : row * a.k_rs + hk * a.k_hs;
    const long long to = isq ? ((long long)row * a.H + h) * a.D : slot + hk * a.head_stride;
    if (!isq && page < 0) continue;
    if (e < half) {
      float s, c;
      sincos_rot_d((double)pos * (double)a.inv_freq[e], &s, &c);
      c *= a.scaling, s *= a.scaling;
      const float lo = ld_f(src, so + e, a.dtype), hi = ld_f(src, so + half + e, a.dtype);
      st_f(dst, to + e, a.dtype, real ? lo * c - hi * s : 0.f);
      st_f(dst, to + half + e, a.dtype, real ? hi * c + lo * s : 0.f);
    } else {
      const int d = a.R + e - half;
      st_f(dst, to + d, a.dtype, real ? ld_f(src, so + d, a.dtype) : 0.f);
    }
  }
  if (page < 0) return;
  for (int i = tid; i < a.KVH * a.D; i += 256) {
    const int h = i / a.D, d = i % a.D;
    st_f(a.v_pages, slot + h * a.head_stride + d, a.dtype, ld_f(a.v, row * a.v_rs + h * a.v_hs + d, a.dtype));
  }
}

// k_paged_append_*: rows of 16-byte pieces (16-bit types, whole pieces on both sides of every rotated pair, 16-byte
// aligned rows). A wave per row, or the four waves of a workgroup where rows are few (_row): one row's chain of lookups
// (q_start, kv_len, block_table, each waiting for the one before) is what it takes then, and its heads are done in one
// step instead of three. Cosines and sines are taken once per row, for all heads, by a lane each. Bound by the bytes: each
// row is read once and written once (5963 rows of 32 + 8 heads, 147 MB: 33 us, 4.4 TB/s; 34 with the loads of one step in
// flight rather than two).
template <int DT, int WAVES>
__device__ __forceinline__ void append_body(const PagedAppendArgs& a) {
  constexpr int ROWS = 4 / WAVES, TH = 64 * WAVES;
  __shared__ __attribute__((aligned(16))) float cs[ROWS][2][PG_APPEND_R / 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = wave / WAVES, tid = (wave % WAVES) * 64 + lane;
  const int row = blockIdx.x * ROWS + mine, half = a.R / 2;
  const bool in = row < a.N;
  const int b = in ? pg_sequence(a.q_start, a.B, row, lane) : a.B;
  const bool real = b < a.B && row >= a.q_start[0];
  const int pos = real ? pg_position(a.kv_len[b], a.q_start[b + 1], row) : 0;
  const int page = real ? pg_page(a.table, b, a.M, a.page_size, a.pages, pos) : -1;
  if (real)
    for (int j = tid; j < half; j += TH) {
      float s, c;
      sincos_rot_d((double)pos * (double)a.inv_freq[j], &s, &c);
      cs[mine][0][j] = c * a.scaling, cs[mine][1][j] = s * a.scaling;
    }
  __syncthreads();
  if (!in) return;
  const long long slot = page < 0 ? 0 : page * a.page_stride + (pos % a.page_size) * a.row_stride;
  // steps: pairs of pieces, then the pieces past R, then v's
  const int pairs = half / 8, rest = (a.D - a.R) / 8, qk = a.H + a.KVH;
  const int n0 = qk * pairs, n1 = n0 + qk * rest, n2 = n1 + a.KVH * (a.D / 8);
  struct Step {
    uint4 x, y;
    uint16_t* dst;   // null: nothing to write
    int e;
    bool pair;
  };
  auto get = [&](int i) {
    Step t;
    const bool v = i >= n1;
    t.pair = i < n0;
    const int k = t.pair ? i : v ? i - n1 : i - n0, per = t.pair ? pairs : v ? a.D / 8 : rest;
    const int h = k / per;
    t.e = (t.pair ? 0 : v ? 0 : a.R) + k % per * 8;
    const bool isq = !v && h < a.H;
    const int hk = v ? h : h - a.H;
    const uint16_t* src = isq ? (const uint16_t*)a.q + row * a.q_rs + h * a.q_hs
                         : v  ? (const uint16_t*)a.v + row * a.v_rs + hk * a.v_hs
                              : (const uint16_t*)a.k + row * a.k_rs + hk * a.k_hs;
    t.dst = isq ? (uint16_t*)a.q_out + ((long long)row * a.H + h) * a.D
            : page < 0 ? nullptr
                       : (uint16_t*)(v ? a.v_pages : a.k_pages) + slot + hk * a.head_stride;
    t.x = *(const uint4*)(src + t.e);
    t.y = *(const uint4*)(src + t.e + (t.pair ? half : 0));
    return t;
  };
  auto put = [&](const Step& t) {
    if (!t.dst) return;
    if (!t.pair) {
      *(uint4*)(t.dst + t.e) = real ? t.x : make_uint4(0, 0, 0, 0);
      return;
    }
    const uint32_t xw[4] = {t.x.x, t.x.y, t.x.z, t.x.w}, yw[4] = {t.y.x, t.y.y, t.y.z, t.y.w};
    uint32_t lo[4], up[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 c = *(const float2*)&cs[mine][0][t.e + 2 * j], d = *(const float2*)&cs[mine][1][t.e + 2 * j];
      const float x0 = gm_lo<DT>(xw[j]), x1 = gm_hi<DT>(xw[j]), y0 = gm_lo<DT>(yw[j]), y1 = gm_hi<DT>(yw[j]);
      lo[j] = real ? gm_pack2<DT>(x0 * c.x - y0 * d.x, x1 * c.y - y1 * d.y) : 0u;
      up[j] = real ? gm_pack2<DT>(y0 * c.x + x0 * d.x, y1 * c.y + x1 * d.y) : 0u;
    }
    *(uint4*)(t.dst + t.e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    *(uint4*)(t.dst + half + t.e) = make_uint4(up[0], up[1], up[2], up[3]);
  };
  for (int i = tid; i < n2; i += 2 * TH) {   // two steps' loads in flight
    const bool two = i + TH < n2;
    const Step s = get(i), t = get(two ? i + TH : i);
    put(s);
    if (two) put(t);
  }
}
extern "C" __global__ void __launch_bounds__(256) k_paged_append_bf16(const PagedAppendArgs a) { append_body<HS_BF16, 1>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_append_bf16_row(const PagedAppendArgs a) { append_body<HS_BF16, 4>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_append_f16(const PagedAppendArgs a) { append_body<HS_F16, 1>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_append_f16_row(const PagedAppendArgs a) { append_body<HS_F16, 4>(a); }

// ------------------------------------------------------------------ append of normed heads, and into pages of 8 bits
//
// y = rotation of x / sqrt(mean(x^2) + eps) weight (NORM), of x otherwise; pages of 8 bits (F8) take k and v as e4m3
// with pg_quant_byte's power of two. fp32 up to the one rounding of each result.

// k_paged_*_append_any: one workgroup per row, a wave per head; any type, head size and strides. A head is read again for
// each thing that is needed of the whole of it (sum of squares, largest magnitude).
template <bool NORM, bool F8>
__device__ __forceinline__ void append_heads_any(const PagedAppendArgs& a) {
  __shared__ int place[3];   // sequence, position, page
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  if (tid < 64) {
    const int b = pg_sequence(a.q_start, a.B, row, tid);
    const bool real = b < a.B && row >= a.q_start[0];
    const int pos = real ? pg_position(a.kv_len[b], a.q_start[b + 1], row) : 0;
    if (tid == 0) place[0] = real ? b : -1, place[1] = pos, place[2] = real ? pg_page(a.table, b, a.M, a.page_size, a.pages, pos) : -1;
  }
  __syncthreads();
  const int pos = place[1], page = place[2], half = a.R / 2, per = half + a.D - a.R;
  const bool real = place[0] >= 0;
  const long long slot = page < 0 ? 0 : page * a.page_stride + (pos % a.page_size) * a.row_stride;
  for (int h = tid >> 6; h < a.H + 2 * a.KVH; h += 4) {
    const bool isq = h < a.H, isv = h >= a.H + a.KVH;
    const int hk = isv ? h - a.H - a.KVH : h - a.H;
    if (!isq && page < 0) continue;
    const void* src = isq ? a.q : isv ? a.v : a.k;
    const long long so = isq ? row * a.q_rs + h * a.q_hs : isv ? row * a.v_rs + hk * a.v_hs : row * a.k_rs + hk * a.k_hs;
    const void* weight = isq ? a.q_weight : a.k_weight;
    float r = 1.f;
    if (NORM && !isv) {
      float ss = 0.f;
      for (int d = lane; d < a.D; d += 64) {
        const float x = ld_f(src, so + d, a.dtype);
        ss = fmaf(x, x, ss);
      }
      r = 1.f / sqrtf(wave_sum(ss) / (float)a.D + a.eps);
    }
    auto get = [&](int d) {
      const float x = ld_f(src, so + d, a.dtype);
      return NORM && !isv ? x * r * ld_f(weight, d, a.dtype) : x;
    };
    // f(dim, value) for the lane's results
    auto each = [&](auto f) {
      for (int e = lane; e < per; e += 64) {
        if (e < half) {
          float s = 0.f, c = 1.f;
          if (!isv) {
            sincos_rot_d((double)pos * (double)a.inv_freq[e], &s, &c);
            c *= a.scaling, s *= a.scaling;
          }
          const float lo = get(e), hi = get(half + e);
          f(e, isv ? lo : lo * c - hi * s);
          f(half + e, isv ? hi : hi * c + lo * s);
        } else {
          f(a.R + e - half, get(a.R + e - half));
        }
      }
    };
    if (isq || !F8) {
      void* dst = isq ? a.q_out : isv ? a.v_pages : a.k_pages;
      const long long to = isq ? ((long long)row * a.H + h) * a.D : slot + hk * a.head_stride;
      each([&](int d, float y) { st_f(dst, to + d, a.dtype, real ? y : 0.f); });
      continue;
    }
    float most = 0.f;
    each([&](int, float y) { most = fmaxf(most, pg_finite(y)); });
    const unsigned byte = pg_quant_byte(wave_max(most));
    const float inv = pg_quant_inverse(byte);
    unsigned char* dst = (unsigned char*)(isv ? a.v_pages : a.k_pages) + slot + hk * a.head_stride;
    each([&](int d, float y) { dst[d] = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(y * inv, 0.f, 0, false); });
    if (lane == 0) (isv ? a.v_scales : a.k_scales)[pg_scale_at(page, hk, a.KVH, a.page_size, pos % a.page_size)] = (unsigned char)byte;
  }
}
extern "C" __global__ void __launch_bounds__(256) k_paged_norm_append_any(const PagedAppendArgs a) { append_heads_any<true, false>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_quant_append_any(const PagedAppendArgs a) { append_heads_any<false, true>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_norm_quant_append_any(const PagedAppendArgs a) { append_heads_any<true, true>(a); }

// k_paged_*_append_*: 16-bit types, D and R multiples of 16, D <= 256, 16-byte aligned rows. A head lies in LP lanes of a row
// of 16 (the power of two from D / 16, at least 4), 16 dims each in two pieces of 8: those that rotate together, or past R
// two neighbours. So what is needed of a whole head (sum of squares, largest magnitude) takes two to four steps across
// lanes, and a lane's cosines, sines and weights are the same for all heads of its row and stay in registers. Two waves
// per row, or the four of a workgroup where rows are few (_row). Few rows are bound by the chain of loads to a row's place, so
// its first heads are loaded beside that; many by memory: 5,963 rows of 32 + 8 heads of 128, normed and in 8 bits, 32 us for
// 134 MB (4.2 TB/s; 36 with a wave's number in a vector register, 34 with two heads at a time, whose registers leave room
// for fewer waves).
template <bool MAX>
__device__ __forceinline__ float pg_heads(float v, int LP) {
  auto join = [](float x, float y) { return MAX ? fmaxf(x, y) : x + y; };
  v = join(v, HS_DPP(v, HS_QUAD_XOR1));
  v = join(v, HS_DPP(v, HS_QUAD_XOR2));
  if (LP > 4) v = join(v, HS_DPP(v, HS_ROW_HALF_MIRROR));
  if (LP > 8) v = join(v, HS_DPP(v, HS_ROW_MIRROR));
  return v;
}

// four values times inv as e4m3, the first in the lowest byte; NaN where they are not finite
__device__ __forceinline__ uint32_t pg_e4m3(const float* v, float inv) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
}

template <int DT, int WAVES, bool NORM, bool F8>
__device__ __forceinline__ void append_heads(const PagedAppendArgs& a) {
  constexpr int ROWS = 4 / WAVES, TH = 64 * WAVES;
  __shared__ __attribute__((aligned(16))) float cs[ROWS][2][PG_APPEND_R / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = wave / WAVES, tid = (wave % WAVES) * 64 + lane;
  const int row = blockIdx.x * ROWS + mine, half = a.R / 2, heads = a.H + 2 * a.KVH;
  const bool in = row < a.N;
  const int need = a.D / 16, shift = need <= 4 ? 2 : need <= 8 ? 3 : 4, LP = 1 << shift, sub = tid & (LP - 1), step = TH >> shift;
  const bool has = sub < need, turns = has && sub < a.R / 16;
  const int e0 = !has ? 0 : turns ? sub * 8 : a.R + (sub - a.R / 16) * 16, e1 = !has ? 0 : turns ? half + sub * 8 : e0 + 8;
  struct Step {
    uint4 x, y;
    int h;
  };
  auto get = [&](int h) {
    Step t;
    t.h = h;
    const bool isq = h < a.H, isv = h >= a.H + a.KVH;
    const int hk = isv ? h - a.H - a.KVH : h - a.H;
    const uint16_t* src = isq ? (const uint16_t*)a.q + row * a.q_rs + h * a.q_hs
                        : isv ? (const uint16_t*)a.v + row * a.v_rs + hk * a.v_hs
                              : (const uint16_t*)a.k + row * a.k_rs + hk * a.k_hs;
    t.x = *(const uint4*)(src + e0);
    t.y = *(const uint4*)(src + e1);
    return t;
  };
  // the first two heads and the weights are on their way while the row's place and angles are found
  const int h0 = tid >> shift;
  Step t0{}, t1{};
  if (in && h0 < heads) t0 = get(h0);
  if (in && h0 + step < heads) t1 = get(h0 + step);
  uint4 wq0, wq1, wk0, wk1;
  if constexpr (NORM) {
    const uint16_t *wq = (const uint16_t*)a.q_weight, *wk = (const uint16_t*)a.k_weight;
    wq0 = *(const uint4*)(wq + e0), wq1 = *(const uint4*)(wq + e1);
    wk0 = *(const uint4*)(wk + e0), wk1 = *(const uint4*)(wk + e1);
  }
  const int b = __builtin_amdgcn_readfirstlane(in ? pg_sequence(a.q_start, a.B, row, lane) : a.B);
  const bool real = b < a.B && row >= a.q_start[0];
  const int pos = real ? pg_position(a.kv_len[b], a.q_start[b + 1], row) : 0;
  const int page = real ? pg_page(a.table, b, a.M, a.page_size, a.pages, pos) : -1;
  if (real)
    for (int j = tid; j < half; j += TH) {
      float s, c;
      sincos_rot_d((double)pos * (double)a.inv_freq[j], &s, &c);
      cs[mine][0][j] = c * a.scaling, cs[mine][1][j] = s * a.scaling;
    }
  __syncthreads();
  if (!in) return;
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = 1.f, s[j] = 0.f;
  if (turns && real) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = cs[mine][0][e0 + j], s[j] = cs[mine][1][e0 + j];
  }
  const int off = page < 0 ? 0 : pos % a.page_size;
  const long long slot = page < 0 ? 0 : page * a.page_stride + off * a.row_stride;
  auto put = [&](const Step& t) {
    const bool isq = t.h < a.H, isv = t.h >= a.H + a.KVH;
    const int hk = isv ? t.h - a.H - a.KVH : t.h - a.H;
    const uint32_t xw[4] = {t.x.x, t.x.y, t.x.z, t.x.w}, yw[4] = {t.y.x, t.y.y, t.y.z, t.y.w};
    float x[8], y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[2 * j] = gm_lo<DT>(xw[j]), x[2 * j + 1] = gm_hi<DT>(xw[j]), y[2 * j] = gm_lo<DT>(yw[j]), y[2 * j + 1] = gm_hi<DT>(yw[j]);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
      ss = pg_heads<false>(has ? ss : 0.f, LP);
      if (!isv) {
        const float r = 1.f / sqrtf(ss / (float)a.D + a.eps);
        const uint4 w0 = isq ? wq0 : wk0, w1 = isq ? wq1 : wk1;
        const uint32_t uw[4] = {w0.x, w0.y, w0.z, w0.w}, vw[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // (x r first: r times a weight may pass 32 bits where the result does not)
          x[2 * j] = x[2 * j] * r * gm_lo<DT>(uw[j]), x[2 * j + 1] = x[2 * j + 1] * r * gm_hi<DT>(uw[j]);
          y[2 * j] = y[2 * j] * r * gm_lo<DT>(vw[j]), y[2 * j + 1] = y[2 * j + 1] * r * gm_hi<DT>(vw[j]);
        }
      }
    }
    if (!isv && turns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[j] * c[j] - y[j] * s[j], up = y[j] * c[j] + x[j] * s[j];
        x[j] = lo, y[j] = up;
      }
    }
    if (F8 && !isq) {
      if (page < 0) return;
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fmaxf(pg_finite(x[j]), pg_finite(y[j])));
      const unsigned byte = pg_quant_byte(pg_heads<true>(has ? most : 0.f, LP));
      const float inv = pg_quant_inverse(byte);
      if (!has) return;
      unsigned char* dst = (unsigned char*)(isv ? a.v_pages : a.k_pages) + slot + hk * a.head_stride;
      *(uint2*)(dst + e0) = make_uint2(pg_e4m3(x, inv), pg_e4m3(x + 4, inv));
      *(uint2*)(dst + e1) = make_uint2(pg_e4m3(y, inv), pg_e4m3(y + 4, inv));
      if (sub == 0) (isv ? a.v_scales : a.k_scales)[pg_scale_at(page, hk, a.KVH, a.page_size, off)] = (unsigned char)byte;
      return;
    }
    uint16_t* dst = isq ? (uint16_t*)a.q_out + ((long long)row * a.H + t.h) * a.D
                        : (uint16_t*)(isv ? a.v_pages : a.k_pages) + slot + hk * a.head_stride;
    if (!has || (!isq && page < 0)) return;
    uint32_t lo[4], up[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = real ? gm_pack2<DT>(x[2 * j], x[2 * j + 1]) : 0u;
      up[j] = real ? gm_pack2<DT>(y[2 * j], y[2 * j + 1]) : 0u;
    }
    *(uint4*)(dst + e0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    *(uint4*)(dst + e1) = make_uint4(up[0], up[1], up[2], up[3]);
  };
  for (int h = h0; h < heads; h += step) {   // two heads' loads are in flight while one is written
    put(t0);
    t0 = t1;
    if (h + 2 * step < heads) t1 = get(h + 2 * step);
  }
}

#define PG_APPENDS(NAME, NORM, F8)                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) k_paged_##NAME##_append_bf16(const PagedAppendArgs a) { append_heads<HS_BF16, 2, NORM, F8>(a); }     \
  extern "C" __global__ void __launch_bounds__(256) k_paged_##NAME##_append_bf16_row(const PagedAppendArgs a) { append_heads<HS_BF16, 4, NORM, F8>(a); } \
  extern "C" __global__ void __launch_bounds__(256) k_paged_##NAME##_append_f16(const PagedAppendArgs a) { append_heads<HS_F16, 2, NORM, F8>(a); }       \
  extern "C" __global__ void __launch_bounds__(256) k_paged_##NAME##_append_f16_row(const PagedAppendArgs a) { append_heads<HS_F16, 4, NORM, F8>(a); }
PG_APPENDS(norm, true, false)
PG_APPENDS(quant, false, true)
PG_APPENDS(norm_quant, true, true)

// ------------------------------------------------------------------ attention
//
// k_paged_attn_any: one wave per (row, query head), 64 positions a step: a lane scores one position (its key's row
// against q in LDS), the wave takes maximum and sum, then every lane adds its dims of 64 values. Any type, page size
// and head size up to 256; fp32 throughout. Closed positions are never loaded, so what lies there (NaN) does not enter.
#define PG_ANY_D 256
// number i of a pool of 8 bits, without its power of two
__device__ __forceinline__ float pg_number(const void* p, long long i) { return __builtin_amdgcn_cvt_f32_fp8(((const unsigned char*)p)[i], 0); }
template <bool F8>
struct PtArgsOf {
  typedef PagedAttnArgs type;
};
template <>
struct PtArgsOf<true> {
  typedef PagedQuantAttnArgs type;
};
template <bool F8>
using PtArgs = typename PtArgsOf<F8>::type;

// (A: the record, by value over 16-bit pages, where by reference one token over 2,048 positions, 12 + 2 heads of 96, took 1,513 us
// for 1,455, and by reference over pages of 8 bits, 919 by value for 897.)
template <bool F8, typename A>
__device__ __forceinline__ void attn_any_body(A a) {
  __shared__ float q[PG_ANY_D], p[64];
  __shared__ int at[64];   // page of each of the step's positions, -1: closed
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / (a.H / a.KVH);
  const int b = pg_sequence(a.q_start, a.B, row, lane);
  const bool real = b < a.B && row >= a.q_start[0] && !pg_descends(a.q_start, a.B, lane);
  const int pos = real ? pg_position(a.kv_len[b], a.q_start[b + 1], row) : -1;
  for (int d = lane; d < a.D; d += 64) q[d] = ld_f(a.q, row * a.q_rs + h * a.q_hs + d, a.dtype);
  float m = -INFINITY, l = 0.f, o[PG_ANY_D / 64] = {};
  const int end = min((long long)pos + 1, (long long)a.M * a.page_size);
  for (int p0 = 0; p0 < end; p0 += 64) {
    const int mine = p0 + lane, page = mine < end ? pg_page(a.table, b, a.M, a.page_size, a.pages, mine) : -1;
    __syncthreads();
    at[lane] = page;
    float s = -INFINITY;
    if (page >= 0) {
      const long long ko = page * a.page_stride + kvh * a.head_stride + (mine % a.page_size) * a.row_stride;
      s = 0.f;
      for (int d = 0; d < a.D; ++d) {
        if constexpr (F8) s = fmaf(q[d], pg_number(a.k_pages, ko + d), s);
        else s = fmaf(q[d], ld_f(a.k_pages, ko + d, a.dtype), s);
      }
      if constexpr (F8) s *= pg_scale(a.k_scales[pg_scale_at(page, kvh, a.KVH, a.page_size, mine % a.page_size)]);
      s *= a.scale;
    }
    // (wave_max's fmaxf drops a NaN score: its exponential below keeps it)
    const float mn = fmaxf(m, wave_max(page >= 0 ? s : -INFINITY));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float e = page >= 0 ? expf(s - mu) : 0.f, alpha = m == -INFINITY ? 0.f : expf(m - mu);
    l = l * alpha + wave_sum(e);
    m = mn;
    p[lane] = e;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PG_ANY_D / 64; ++i) {
      if (i * 64 + lane >= a.D) continue;
      float x = o[i] * alpha;
      for (int j = 0; j < min(64, end - p0); ++j) {
        if (at[j] < 0) continue;
        const long long vo = at[j] * a.page_stride + kvh * a.head_stride + ((p0 + j) % a.page_size) * a.row_stride;
        if constexpr (F8)
          x = fmaf(p[j], pg_number(a.v_pages, vo + i * 64 + lane) *
                             pg_scale(a.v_scales[pg_scale_at(at[j], kvh, a.KVH, a.page_size, (p0 + j) % a.page_size)]), x);
        else x = fmaf(p[j], ld_f(a.v_pages, vo + i * 64 + lane, a.dtype), x);
      }
      o[i] = x;
    }
  }
#pragma unroll
  for (int i = 0; i < PG_ANY_D / 64; ++i)
    if (i * 64 + lane < a.D)
      st_f(a.out, ((long long)row * a.H + h) * a.D + i * 64 + lane, a.dtype, l == 0.f ? 0.f : o[i] / l);
}
extern "C" __global__ void __launch_bounds__(64) k_paged_attn_any(const PagedAttnArgs a) { attn_any_body<false, const PagedAttnArgs>(a); }
extern "C" __global__ void __launch_bounds__(64) k_paged_quant_attn_any(const PagedQuantAttnArgs a) { attn_any_body<true, const PagedQuantAttnArgs&>(a); }

// ------------------------------------------------------------------ attention on matrix cores
//
// Types of 16 bits, head sizes 64 and 128, pages of a multiple of 16 positions. The G = H / KVH query heads of a K/V
// head are packed with the tokens into rows (row = token * G + head), so K and V are read once for all of them. A
// wave holds 32 rows: S^T = K Q^T on v_mfma_f32_32x32x16 leaves each lane the scores of ONE row, so maximum, exponentials
// and the rescaling of that row's outputs stay in the lane (two lanes, 32 apart, share a row's positions), and
// O^T += V^T P^T takes P as it lies. Two forms of a workgroup of four waves:
//   * narrow tile, sequences of up to 32 rows (decoding, a few speculated tokens): the four waves hold the SAME rows
//     and take every fourth block of positions, each streaming K and V through LDS of its own with no barrier: while a
//     block's scores are taken the next K is on its way, while its outputs are, the next V. Bound by memory.
//   * wide tile, longer chunks: 128 rows, each wave 32 of them, all sharing blocks of 64 positions staged one block
//     ahead. Bound by the matrix cores and the softmax's vector instructions, which a SIMD's two waves overlap in part:
//     409 tokens over 30,409 positions (12 + 2 heads) take 93 us, 0.81 PFLOP/s, 0.65 of a large matrix product.
// K and V go from the pages to LDS directly (a load covers 4 or 8 rows of one page), K swizzled for the fragment
// reads, V for the transposing ones.
//
// Work is dealt out on the device: lengths are tensors, the launch is the same for every batch. Narrow tiles' blocks form
// one list (sequence, head, tile, block), of which every workgroup takes an equal range, so that at most the tiles at
// its ends are split. Wide tiles longer than an even share of all blocks are split evenly; their items are dealt to the
// XCDs in ranges of equal cost, so that the tiles that read the same blocks share an L2. A part of a split tile leaves
// unnormalised outputs with their maximum and sum; k_paged_combine_* joins them.

#define PT_MAXB 1024             // sequences
#define PT_NARROW 32             // rows
#define PT_WIDE 128
#define PT_NARROW_LEAST 4        // fewest blocks of a narrow workgroup: one per wave
// Fewest blocks of a wave over pages of 8 bits. us at 1 / 2 / 4: one token over 2,048 positions (12 + 2 heads of 128) 13.5 / 15.0 /
// 18.7, over 8,000 14.6 / 15.8 / 21.9, 16 over 2,000 (32 + 8) 28.8 / 27.5 / 27.2, 64 over 500 (12 + 2) 16.5 / 19.7 / 23.6.
#define PT_WAVE_LEAST 1
#define PT_WIDE_ITEMS 480        // items that wide tiles are split towards: one round of two workgroups per CU
#define PT_WIDE_LEAST 8          // fewest blocks of a split

typedef __attribute__((ext_vector_type(16))) float pt_f32x16;
typedef __attribute__((ext_vector_type(4))) short pt_s16x4;

template <int DT>
__device__ __forceinline__ pt_f32x16 pt_mfma(const uint4 a, const uint4 b, pt_f32x16 c) {
  if constexpr (DT == HS_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(__attribute__((ext_vector_type(8))) __bf16, a),
                                                   __builtin_bit_cast(__attribute__((ext_vector_type(8))) __bf16, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(__attribute__((ext_vector_type(8))) _Float16, a),
                                                  __builtin_bit_cast(__attribute__((ext_vector_type(8))) _Float16, b), c,
                                                  0, 0, 0);
}

// lanes 32-63 of a and lanes 0-31 of b change places
__device__ __forceinline__ void pt_swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// Transposing LDS read: lanes 4r + c of each 16-lane group address row r, columns 4c .. 4c + 3 (8 bytes);
// lane i gets column i of rows 0 .. 3.
__device__ __forceinline__ uint2 pt_read_tr(const char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) pt_s16x4*)(__attribute__((address_space(3))) char*)p));
}

// uniform load from memory that no kernel in flight writes
__device__ __forceinline__ int pt_ldc(const int* p, long long i) {
  return ((const __attribute__((address_space(4))) int*)p)[i];
}

// A sequence's share of the work: its rows that the tensor has (start, n), their positions (kv - n + i), tiles of R rows,
// blocks of PB positions that its last tile needs.
struct PtSeq {
  int start, n, kv, tiles, blocks;
};
template <int R, int PB>
__device__ __forceinline__ PtSeq pt_seq(const PagedAttnArgs& a, int b, int s0, int s1, int kv, int lo, int hi) {
  const int start = max(s0, 0), stop = min(s1, a.N);
  PtSeq q{start, max(stop, start) - start, pg_position(kv, s1, stop), 0, 0};
  const int G = a.H / a.KVH;
  const long long rows = (long long)q.n * G;
  if (rows <= lo || rows > hi) {
    q.n = 0;
    return q;
  }
  q.tiles = (int)((rows + R - 1) / R);
  const long long end = min((long long)max(q.kv, 1), (long long)a.M * a.page_size);
  q.blocks = (int)((end + PB - 1) / PB);   // (at least one: a tile without positions writes its zeros)
  return q;
}

// The sequences' work, in LDS: running sums over them. Narrow: blocks in items, rows and heads in cost. Wide: items,
// partial slots, and cost (JOIN: rows and heads of split tiles).
struct PtList {
  int items[PT_MAXB];
  int slots[PT_MAXB];
  int cost[PT_MAXB];
  int red[3][4];
  int share;   // blocks per split
};

// inclusive scans of three values over 256 threads, added to the running totals
__device__ __forceinline__ void pt_scan3(int (&v)[3], int (&total)[3], int (&red)[3][4]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int w = __shfl_up(v[j], o, 64);
      if (lane >= o) v[j] += w;
    }
  __syncthreads();
  if (lane == 63)
#pragma unroll
    for (int j = 0; j < 3; ++j) red[j][wave] = v[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    int base = total[j], all = total[j];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      base += w < wave ? red[j][w] : 0;
      all += red[j][w];
    }
    v[j] += base;
    total[j] = all;
  }
}

// splits of a sequence's tiles
__device__ __forceinline__ int pt_splits(const PtSeq& q, int share) { return max(1, (q.blocks + share - 1) / share); }

// Narrow sequences' blocks (by 256 threads; ends with a barrier); returns their number, and that of rows and heads.
// None where q_start descends: sequences then overlap, and their tiles could be more than the launch has room for.
template <int PB>
__device__ __forceinline__ int pt_build_narrow(const PagedAttnArgs& a, PtList& t, int hi, int* rows) {
  int total[3] = {0, 0, 0};
  for (int c = 0; c < a.B; c += 256) {
    const int b = c + threadIdx.x;
    int v[3] = {0, 0, 0};
    if (b < a.B) {
      const int s0 = a.q_start[b], s1 = a.q_start[b + 1];
      const PtSeq q = pt_seq<PT_NARROW, PB>(a, b, s0, s1, a.kv_len[b], 0, hi);
      v[2] = s1 < s0;
      v[0] = q.tiles * q.blocks * a.KVH;
      v[1] = q.n * a.H;
    }
    pt_scan3(v, total, t.red);
    if (b < a.B) t.items[b] = v[0], t.cost[b] = v[1];
  }
  __syncthreads();
  *rows = total[2] ? 0 : total[1];
  return total[2] ? 0 : total[0];
}

// Workgroups that share `all` narrow blocks, of at most `most`, and the first block of workgroup w
template <int LEAST = PT_NARROW_LEAST>
__device__ __forceinline__ int pt_workers(int all, int most) {
  return max(1, min(most, (all + LEAST - 1) / LEAST));
}
__device__ __forceinline__ int pt_first(int all, int workers, int w) { return (int)((long long)all * w / workers); }

// Wide sequences' items (by 256 threads; ends with a barrier); returns their number.
template <bool JOIN>
__device__ __forceinline__ int pt_build_wide(const PagedAttnArgs& a, PtList& t, int* cost) {
  constexpr int PB = 64, ANY = 0x7fffffff;
  const int tid = threadIdx.x;
  int work[3] = {0, 0, 0};
  for (int b = tid; b < a.B; b += 256) {
    const int s0 = a.q_start[b], s1 = a.q_start[b + 1];
    const PtSeq q = pt_seq<PT_WIDE, PB>(a, b, s0, s1, a.kv_len[b], PT_NARROW, ANY);
    work[1] |= s1 < s0;
    work[0] += q.tiles * q.blocks * a.KVH;
  }
  int total[3] = {0, 0, 0};
  pt_scan3(work, total, t.red);
  const int share = max((total[0] + PT_WIDE_ITEMS - 1) / PT_WIDE_ITEMS, PT_WIDE_LEAST);
  const bool down = total[1] != 0;
  total[0] = total[1] = total[2] = 0;
  for (int c = 0; c < a.B; c += 256) {
    const int b = c + tid;
    int v[3] = {0, 0, 0};
    if (b < a.B && !down) {
      const PtSeq q = pt_seq<PT_WIDE, PB>(a, b, a.q_start[b], a.q_start[b + 1], a.kv_len[b], PT_NARROW, ANY);
      const int S = pt_splits(q, share);
      v[0] = q.tiles * S * a.KVH;
      v[1] = S > 1 ? v[0] : 0;
      // cost of an item, in blocks: the mean of the first and the last tile's, and 2 for starting and ending it
      v[2] = JOIN ? (S > 1 ? q.n * a.H : 0) : v[0] * (max(0, q.blocks - q.n / PB / 2) / S + 2);
    }
    pt_scan3(v, total, t.red);
    if (b < a.B) t.items[b] = v[0], t.slots[b] = v[1], t.cost[b] = v[2];
  }
  if (tid == 0) t.share = share;
  __syncthreads();
  *cost = total[2];
  return total[0];
}

// first sequence whose running sum passes x (the sums are non-decreasing)
__device__ __forceinline__ int pt_find(const int* sums, int B, int x) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// One item: blocks b0 .. b1 - 1 of a tile (of those that its rows see). slot: of the partial output, -1 for a whole tile.
struct PtItem {
  PtSeq q;
  int b, h, tile, b0, b1, slot;
};

// blocks that tile `tile` of R rows sees
template <int R, int PB>
__device__ __forceinline__ int pt_seen(const PagedAttnArgs& a, const PtSeq& q, int tile) {
  const int G = a.H / a.KVH, last = q.kv - q.n + min(tile * R + R - 1, q.n * G - 1) / G;
  return last < 0 ? 0 : min(q.blocks, last / PB + 1);
}

// the item of workgroup w that starts at block `at` of all narrow blocks; `end`: of its range. Returns the next start.
template <int PB>
__device__ __forceinline__ int pt_item_narrow(const PagedAttnArgs& a, const PtList& t, int w, int at, int end, int hi, PtItem& it) {
  it.b = __builtin_amdgcn_readfirstlane(pt_find(t.items, a.B, at));
  it.q = pt_seq<PT_NARROW, PB>(a, it.b, pt_ldc(a.q_start, it.b), pt_ldc(a.q_start, it.b + 1), pt_ldc(a.kv_len, it.b), 0, hi);
  const int i = at - (it.b ? __builtin_amdgcn_readfirstlane(t.items[it.b - 1]) : 0), tl = i / it.q.blocks;
  it.tile = tl % it.q.tiles, it.h = tl / it.q.tiles;
  it.b0 = i % it.q.blocks, it.b1 = min(it.q.blocks, it.b0 + end - at);
  const int next = at + it.b1 - it.b0;
  // the first part of a split tile ends its workgroup's range (slot 2 w + 1), the others begin theirs (2 w)
  it.slot = it.b0 > 0 ? 2 * w : it.b1 < it.q.blocks ? 2 * w + 1 : -1;
  const int seen = pt_seen<PT_NARROW, PB>(a, it.q, it.tile);
  it.b0 = min(it.b0, seen), it.b1 = min(it.b1, seen);
  return next;
}

__device__ __forceinline__ PtItem pt_item_wide(const PagedAttnArgs& a, const PtList& t, int item) {
  PtItem it;
  it.b = __builtin_amdgcn_readfirstlane(pt_find(t.items, a.B, item));
  it.q = pt_seq<PT_WIDE, 64>(a, it.b, pt_ldc(a.q_start, it.b), pt_ldc(a.q_start, it.b + 1), pt_ldc(a.kv_len, it.b),
                             PT_NARROW, 0x7fffffff);
  const int S = pt_splits(it.q, __builtin_amdgcn_readfirstlane(t.share));
  const int i = item - (it.b ? __builtin_amdgcn_readfirstlane(t.items[it.b - 1]) : 0);   // (head, split, tile from the last)
  it.tile = it.q.tiles - 1 - i % it.q.tiles;
  const int split = i / it.q.tiles % S;
  it.h = i / it.q.tiles / S;
  it.slot = S > 1 ? (it.b ? __builtin_amdgcn_readfirstlane(t.slots[it.b - 1]) : 0) + (it.h * it.q.tiles + it.tile) * S + split : -1;
  const int seen = pt_seen<PT_WIDE, 64>(a, it.q, it.tile);
  it.b0 = (int)((long long)seen * split / S), it.b1 = (int)((long long)seen * (split + 1) / S);
  return it;
}

// Rows' swizzles: chunk c (16 bytes) of row r lies in slot c ^ x(r). K: the 32 rows x 2 chunks of a fragment read hit
// every bank; V: so do the transposing reads of 4 rows.
template <int D>
__device__ __forceinline__ int pt_xk(int r) {
  return D == 128 ? r & 15 : (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int pt_xv(int r) {
  return (D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1);
}

// Exponentials go to the second product in the pools' type, half a step of each (its operands have 16 bits; the sum takes
// them unrounded). They are e^(s - m) 2^pt_up, so that float16 holds those far below the largest: a running maximum lags by up
// to 8 in the exponent (softmax), so 2^15 is the most (65504 fits), and its smallest step, 2^-24, is 2^-31 of the largest.
// Without the factor 16 nats below the largest a probability had one or two bits. bfloat16 has the range as it is.
template <int DT>
constexpr float pt_up = DT == HS_F16 ? 7.f : 0.f;

// The state of a wave's 32 rows over the positions seen so far.
template <int DT, int D>
struct PtWave {
  static constexpr int RB = 2 * D;         // bytes of a row
  static constexpr int TD = D / 32;        // output tiles of 32 dims
  uint4 qf[D / 16];                        // B operand of S^T: row fr, dims 16 ks + 8 hi .. + 8
  pt_f32x16 o[TD];                         // O^T: dims 32 t + 8 i + 4 hi + r, row fr
  float m, l;                              // running maximum of the raw scores; the lane's own sum
  float c;                                 // |scale| log2(e)
  int pos;                                 // position of row fr, -1: none open
  int lane, fr, hi;

  // F8: the queries in the order in which a narrow tile reads K, 16 dims of a position at a time
  template <bool F8 = false>
  __device__ __forceinline__ void init(const PagedAttnArgs& a, const PtItem& it, int row0) {
    queries<F8>(a, it, row0);
    begin(a, it, row0);
  }
  template <bool F8 = false>
  __device__ __forceinline__ void queries(const PagedAttnArgs& a, const PtItem& it, int row0) {
    const int ln = threadIdx.x & 63, half = ln >> 5;
    const int G = a.H / a.KVH, rows = it.q.n * G, r = min(row0 + (ln & 31), rows - 1), t = r / G;
    const uint16_t* p = (const uint16_t*)a.q + (long long)(it.q.start + t) * a.q_rs + (long long)(it.h * G + r - t * G) * a.q_hs;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const uint4*)(p + (F8 ? ks / 2 * 32 + half * 16 + ks % 2 * 8 : ks * 16 + half * 8));
  }
  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const PtItem& it, int row0) {
    lane = threadIdx.x & 63, fr = lane & 31, hi = lane >> 5;
    const int G = a.H / a.KVH, rows = it.q.n * G, r = min(row0 + fr, rows - 1), t = r / G;
    pos = it.q.kv - it.q.n + t;
    const long long last = (long long)a.M * a.page_size - 1;
    pos = pos > last ? (int)last : pos;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;   // a negative scale: of -q
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = make_uint4(qf[ks].x ^ flip, qf[ks].y ^ flip, qf[ks].z ^ flip, qf[ks].w ^ flip);
#pragma unroll
    for (int t2 = 0; t2 < TD; ++t2)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[t2][e] = 0.f;
    m = -INFINITY, l = 0.f;
    c = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1e-37f);   // (0: every score counts alike)
  }

  // scores of 32 NB positions from Kt; the operands are read eight (D = 64: four) ahead
  template <int NB>
  __device__ __forceinline__ void scores(const char* Kt, pt_f32x16 (&s)[NB]) const {
    scores_of<NB>([&](int sb, int ks) { return *(const uint4*)(Kt + (sb * 32 + fr) * RB + (((2 * ks + hi) ^ pt_xk<D>(fr)) * 16)); }, s);
  }
  template <int NB, typename F>
  __device__ __forceinline__ void scores_of(F read, pt_f32x16 (&s)[NB]) const {
    constexpr int KS = D / 16;
    uint4 k[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[ks] = read(0, ks);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[sb][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s[sb] = pt_mfma<DT>(k[ks], qf[ks], s[sb]);
        if (sb + 1 < NB) k[ks] = read(sb + 1, ks);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // closed positions' scores to -inf: behind the row, or in one of the 16-position groups of `bad`
  template <int NB>
  __device__ __forceinline__ void mask(pt_f32x16 (&s)[NB], int p0, unsigned bad) const {
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = sb * 32 + 8 * (e >> 2) + 4 * hi + (e & 3);
        if (p0 + j > pos || ((bad >> (j >> 4)) & 1)) s[sb][e] = -INFINITY;
      }
  }

  // Maximum and exponentials (left in s). Outputs are rescaled when a row's maximum has grown by more than 8 in
  // the exponent, not at every new maximum: the exponentials stay below 2^8 (times 2^pt_up), as exact as below 1, and of
  // 32 rows some row's maximum grows in nearly every block.
  template <int NB>
  __device__ __forceinline__ void softmax(pt_f32x16 (&s)[NB]) {
    float bm = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int e = 0; e < 16; ++e) bm = fmaxf(bm, s[sb][e]);
    {
      uint32_t u = __float_as_uint(bm), w = u;
      pt_swap32(u, w);
      bm = fmaxf(__uint_as_float(u), __uint_as_float(w));
    }
    if (__ballot((bm - m) * c > 8.f) != 0ull) {
      const float mn = fmaxf(m, bm);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < TD; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.f : __builtin_fmaf(-m, c, pt_up<DT>);   // nothing open yet: every score is -inf
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[sb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sb][e], c, mc));
  }

  __device__ __forceinline__ uint4 vfrag(const char* Vt, int sb, int hf, int t) const {
    // rows 8 hi + 4 q + vr of the half block's 16, dims 32 t + 16 g + 4 c
    const int vr = (lane & 15) >> 2, r = sb * 32 + hf * 16 + 8 * hi + vr;
    const int ch = 4 * t + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const char* p = Vt + r * RB + (lane & 1) * 8;
    const uint2 lo = pt_read_tr(p + ((ch ^ pt_xv<D>(vr)) * 16));
    const uint2 up = pt_read_tr(p + 4 * RB + ((ch ^ pt_xv<D>(vr + 4)) * 16));
    return make_uint4(lo.x, lo.y, up.x, up.y);
  }

  // P in the B operand's layout: lane half 0 needs positions 0-7 / 16-23 of 32, half 1 8-15 / 24-31
  template <int NB>
  __device__ __forceinline__ void pack(const pt_f32x16 (&s)[NB], uint4 (&p)[2 * NB]) const {
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
      uint32_t g[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[i][0] = gm_pack2<DT>(s[sb][4 * i], s[sb][4 * i + 1]);
        g[i][1] = gm_pack2<DT>(s[sb][4 * i + 2], s[sb][4 * i + 3]);
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        pt_swap32(g[i][0], g[i + 1][0]);
        pt_swap32(g[i][1], g[i + 1][1]);
        p[2 * sb + i / 2] = make_uint4(g[i][0], g[i][1], g[i + 1][0], g[i + 1][1]);
      }
    }
  }

  // Outputs, and the sums of the exponentials s. The operands are read four ahead, in an order that the compiler keeps:
  // left alone it read one, waited for it, multiplied and read the next (98 us for a long chunk's wide tiles; 94 so), or
  // not, depending on code elsewhere.
  template <int NB>
  __device__ __forceinline__ void outputs(const char* Vt, const uint4 (&p)[2 * NB], const pt_f32x16 (&s)[NB]) {
    outputs_of<NB>([&](int i) { return vfrag(Vt, i / TD / 2, i / TD % 2, i % TD); }, p, s);
  }
  template <int NB, typename F>   // (operand i: of 16 positions i / TD, 32 dims i % TD)
  __device__ __forceinline__ void outputs_of(F read, const uint4 (&p)[2 * NB], const pt_f32x16 (&s)[NB]) {
    constexpr int N = 2 * NB * TD, EL = NB * 16 / N;
    uint4 v[4];
    float sum[2] = {l, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i % TD] = pt_mfma<DT>(v[i % 4], p[i / TD], o[i % TD]);
      if (i + 4 < N) v[i % 4] = read(i + 4);
#pragma unroll
      for (int e = i * EL; e < i * EL + EL; ++e) sum[e & 1] += s[e / 16][e % 16];
      __builtin_amdgcn_sched_barrier(0);
    }
    l = sum[0] + sum[1];
  }

  // Closed positions have probability 0, but a value there may be anything, and 0 x NaN is NaN. Those that are closed to
  // every row of the tile (behind its last row's position `end`, or without a page: stale or foreign memory) are zeroed
  // in LDS; for the rest see bad_output.
  template <int NB>
  __device__ __forceinline__ void clear_closed(char* Vt, int p0, int end, unsigned bad) const {
    constexpr int SL = RB / 16;
#pragma unroll 1
    for (int i = lane; i < NB * 32 * SL; i += 64) {
      const int j = i / SL;
      if (p0 + j > end || ((bad >> (j >> 4)) & 1)) *(uint4*)(Vt + i * 16) = make_uint4(0, 0, 0, 0);
    }
  }

  // Whether an output of the wave is not finite: it may come from a position that is open to other rows only
  // (pt_row then takes the rows one by one).
  __device__ __forceinline__ bool bad_output() const {
    bool odd = false;
#pragma unroll
    for (int t = 0; t < TD; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) odd = odd || (__float_as_uint(o[t][e]) & 0x7f800000u) == 0x7f800000u;
    return __ballot(odd) != 0ull;
  }

  // both lanes' sum of the row
  __device__ __forceinline__ float row_sum() const {
    uint32_t u = __float_as_uint(l), w = u;
    pt_swap32(u, w);
    return __uint_as_float(u) + __uint_as_float(w);
  }
};

// The places of 64 consecutive groups of 16 positions, a lane each: byte offset in a pool of the K/V head's row (of page
// 0 where there is no page), and which have a page. Looked up once for 16 (or 32) blocks: a scalar load per block left its
// latency, 700 cycles, in every block's way. The next window's page ids are on their way to the wave's slot of LDS
// meanwhile (to registers, the compiler's wait for them would cover the K and V loads in flight).
template <bool F8>
struct PtWindowT {
  uint32_t lo, hi;
  unsigned long long ok;
  unsigned long long scale;   // 8 bits: place of the group's powers of two
};
typedef PtWindowT<false> PtWindow;
__device__ __forceinline__ unsigned pt_page_of(const PagedAttnArgs& a, int group) {   // may lie past the table
  const unsigned grp = (unsigned)group + (threadIdx.x & 63);
  return a.group_magic ? __umulhi(grp, a.group_magic) : grp;
}
template <bool F8 = false>
__device__ __forceinline__ PtWindowT<F8> pt_window(const PagedAttnArgs& a, const PtItem& it, int group, int id) {
  PtWindowT<F8> w;
  const unsigned grp = (unsigned)group + (threadIdx.x & 63), at = pt_page_of(a, group);
  const bool ok = at < (unsigned)a.M && (unsigned long long)(long long)id < (unsigned long long)a.pages;
  const unsigned long long off = (F8 ? 1ull : 2ull) * ((ok ? id : 0) * a.page_stride + it.h * a.head_stride +
                                         (ok ? (long long)((grp - at * a.page_groups) * 16) * a.row_stride : 0));
  w.lo = (uint32_t)off, w.hi = (uint32_t)(off >> 32);
  w.ok = __ballot(ok);
  if constexpr (F8) w.scale = pg_scale_at(ok ? id : 0, it.h, a.KVH, a.page_size, ok ? (int)((grp - at * a.page_groups) * 16) : 0);
  return w;
}
template <bool F8 = false>
__device__ __forceinline__ PtWindowT<F8> pt_window(const PagedAttnArgs& a, const PtItem& it, int group) {
  return pt_window<F8>(a, it, group, a.table[(long long)it.b * a.M + min(pt_page_of(a, group), (unsigned)a.M - 1)]);
}
// page ids of a window to slot[64]
__device__ __forceinline__ void pt_fetch(const PagedAttnArgs& a, const PtItem& it, int group, int* slot) {
  const unsigned lds = (unsigned)(size_t)(__attribute__((address_space(3))) int*)slot;
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(
                   min(pt_page_of(a, group), (unsigned)a.M - 1) * 4u),
               "s"(a.table + (long long)it.b * a.M), "s"(lds)
               : "memory", "m0");
}

// offset of group i of the window (uniform)
template <bool F8>
__device__ __forceinline__ unsigned long long pt_place(const PtWindowT<F8>& w, int i) {
  return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane(w.hi, i) << 32) | (uint32_t)__builtin_amdgcn_readlane(w.lo, i);
}

// One 1 KiB load of a group to LDS: rows i * (1024 / RB) .. of its 16, swizzled
template <int D, bool V>
__device__ __forceinline__ void pt_load(const char* group, unsigned row_bytes, int i, unsigned lds, int lane) {
  constexpr int RB = 2 * D, PER = 1024 / RB, SL = RB / 16;   // rows per load, slots of a row
  const int r = i * PER + lane / SL, ch = (lane % SL) ^ (V ? pt_xv<D>(r) : pt_xk<D>(r));
  gm_dma16s(group, (unsigned)r * row_bytes + ch * 16, lds);
}

// element i of a pool, without its power of two
template <int DT, bool F8>
__device__ __forceinline__ float pt_cached(const void* p, long long i) {
  if constexpr (F8) return __builtin_amdgcn_cvt_f32_fp8(((const unsigned char*)p)[i], 0);
  else return gm_ld<DT>(p, i);
}

// One row over positions p0 .. p1 - 1 by a wave, 64 at a time, reading open positions only: the row's maximum of the raw
// scores, sum of exponentials and the lane's outputs (dims lane * E ..), times 2^pt_up as the tiles' (they may be joined
// with them). For tiles whose product is not finite.
template <int DT, int D, bool F8>
__device__ __forceinline__ void pt_row(const PtArgs<F8>& a, const PtItem& it, int row, int p0, int p1, float& m,
                                       float& l, float (&x)[D / 64]) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, G = a.H / a.KVH, t = row / G;
  const float flip = a.scale < 0.f ? -1.f : 1.f, c = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1e-37f);
  const uint16_t* q = (const uint16_t*)a.q + (long long)(it.q.start + t) * a.q_rs + (long long)(it.h * G + row - t * G) * a.q_hs;
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
  const int end = min(p1, it.q.kv - it.q.n + t + 1);
#pragma unroll 1
  for (; p0 < end; p0 += 64) {
    const int pos = p0 + lane, page = pos < end ? pg_page(a.table, it.b, a.M, a.page_size, a.pages, pos) : -1;
    const long long at = page < 0 ? 0 : page * a.page_stride + it.h * a.head_stride + (pos % a.page_size) * a.row_stride;
    float s = 0.f, vs = 1.f;
    if (page >= 0) {
#pragma unroll 1
      for (int d = 0; d < D; ++d) s = fmaf(gm_ld<DT>(q, d), pt_cached<DT, F8>(a.k_pages, at + d), s);
      if constexpr (F8) {
        const long long i = pg_scale_at(page, it.h, a.KVH, a.page_size, pos % a.page_size);
        s *= pg_scale(a.k_scales[i]), vs = pg_scale(a.v_scales[i]);
      }
    }
    s = page < 0 ? -INFINITY : s * flip;
    const float mn = fmaxf(m, wave_max(s)), mc = mn == -INFINITY ? 0.f : __builtin_fmaf(-mn, c, pt_up<DT>);
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * c);
    const float e = page < 0 ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, mc));
    m = mn;
    l = l * alpha + wave_sum(e);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] *= alpha;
#pragma unroll 1
    for (int j = 0; j < min(64, end - p0); ++j) {
      const long long aj = __shfl(at, j, 64);
      const float ej = __shfl(e, j, 64), vj = F8 ? __shfl(vs, j, 64) : 1.f;
      if (__shfl(page, j, 64) < 0) continue;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float v = pt_cached<DT, F8>(a.v_pages, aj + lane * E + i);
        x[i] = fmaf(ej, F8 ? v * vj : v, x[i]);
      }
    }
  }
}

// rows r0, r0 + step, ... of a tile one by one, written as the tile's rows are (part: index of its first partial row)
template <int DT, int D, bool F8 = false>
__device__ __forceinline__ void pt_rows(const PtArgs<F8>& a, const PtItem& it, int tile0, int r0, int r1, int step, int p0,
                                     int p1, long long part) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, G = a.H / a.KVH;
#pragma unroll 1
  for (int row = r0; row < r1; row += step) {
    float m, l, x[E];
    pt_row<DT, D, F8>(a, it, row, p0, p1, m, l, x);
    if (it.slot >= 0) {
      const long long at = part + row - tile0;
      if (lane == 0) *(float2*)(a.part_ml + at * 2) = make_float2(m, l);
#pragma unroll
      for (int i = 0; i < E; ++i) a.part_o[at * D + lane * E + i] = x[i];
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int t = row / G;
      uint16_t* out = (uint16_t*)a.out + ((long long)(it.q.start + t) * a.H + it.h * G + row - t * G) * D + lane * E;
#pragma unroll
      for (int i = 0; i < E; ++i) out[i] = gm_pack<DT>(x[i] * inv);
    }
  }
}

// ------------------------------------------------------------------ narrow tiles

struct PtK {
  static constexpr bool value = false;
};
struct PtV {
  static constexpr bool value = true;
};

template <int DT, int D, bool F8 = false>
struct PtNarrow {
  static constexpr int PB = F8 ? 64 : 8192 / (2 * D), NB = PB / 32, NG = PB / 16;   // positions of a block: 8 KiB of K, 8 of V
  static constexpr int LPG = (F8 ? 1 : 2) * D * 16 / 1024;                          // loads per group
  static constexpr int OLD = 64 + 4;                                        // output row in LDS (floats)
};

template <int DT, int D>
__device__ __forceinline__ void pt_narrow(const PagedAttnArgs& a, const PtItem& it, char* lds, float (*ml)[2][32], int (*slots)[64]) {
  using C = PtNarrow<DT, D>;
  constexpr int PB = C::PB, NB = C::NB, NG = C::NG, LPG = C::LPG, OLD = C::OLD;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.H / a.KVH, rows = it.q.n * G, row0 = it.tile * 32;
  PtWave<DT, D> w;
  const unsigned row_bytes = (unsigned)(2 * a.row_stride);
  char* Kt = lds + wave * 16384;
  char* Vt = Kt + 8192;
  const unsigned k0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)Kt, v0 = k0 + 8192;
  const int b0 = it.b0, b1 = it.b1;
  constexpr int WB = 64 / NG;   // blocks of a window
  PtWindow cur;
  int* ids = slots[wave];
  int wi;                       // window of cur
  unsigned bad = 0, bad_next;   // groups of the present and the next block without a page
  auto seek = [&](int blk) {    // cur: the block's window
    if (blk / WB != wi) {
      ++wi;
      cur = pt_window(a, it, wi * 64, ids[lane]);
      pt_fetch(a, it, (wi + 1) * 64, ids);
    }
    return ~(unsigned)(cur.ok >> (blk % WB * NG)) & ((1u << NG) - 1);
  };
  auto load = [&](auto v, int blk) {
    constexpr bool V = decltype(v)::value;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const char* p = (const char*)(V ? a.v_pages : a.k_pages) + pt_place(cur, blk % WB * NG + g);
#pragma unroll
      for (int i = 0; i < LPG; ++i) pt_load<D, V>(p, row_bytes, i, (V ? v0 : k0) + (g * LPG + i) * 1024, lane);
    }
  };
  int blk = b0 + wave;
  if (blk < b1) {
    wi = blk / WB;
    cur = pt_window(a, it, wi * 64);
    pt_fetch(a, it, (wi + 1) * 64, ids);
    bad = seek(blk);
    load(PtK{}, blk);
    load(PtV{}, blk);
  }
  w.init(a, it, row0);
  // the queries are waited for here: at their first use the wait would cover the loads in flight of every block
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" ::"v"(w.qf[ks].x), "v"(w.qf[ks].y), "v"(w.qf[ks].z), "v"(w.qf[ks].w));
  // positions that the tile's first row has open, and its last
  const int pmin = __builtin_amdgcn_readfirstlane(w.pos), pend = __builtin_amdgcn_readlane(w.pos, 31);
  for (; blk < b1; blk += 4) {
    const bool more = blk + 4 < b1;
    const bool open = blk * PB + PB - 1 <= pmin && bad == 0;
    gm_vmcnt<8>();   // K has landed; V's eight loads may be on their way
    asm volatile("" ::: "memory");
    pt_f32x16 s[NB];
    w.template scores<NB>(Kt, s);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K's rows are in registers
    if (more) {
      bad_next = seek(blk + 4);
      load(PtK{}, blk + 4);
    }
    if (!open) w.template mask<NB>(s, blk * PB, bad);
    w.template softmax<NB>(s);
    uint4 p[2 * NB];
    w.template pack<NB>(s, p);
    if (more) gm_vmcnt<8>();   // V has landed; the next K's eight loads may be on their way
    else gm_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (blk * PB + PB - 1 > pend || bad) w.template clear_closed<NB>(Vt, blk * PB, pend, bad);
    w.template outputs<NB>(Vt, p, s);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) load(PtV{}, blk + 4);
    bad = bad_next;
  }
  // join the four waves: sum over waves of e^(m_w - M) o_w, e^(m_w - M) l_w
  const float l = w.row_sum();
  if (w.hi == 0) ml[wave][0][w.fr] = w.m, ml[wave][1][w.fr] = l;
  if (__syncthreads_or(w.bad_output())) {
    pt_rows<DT, D>(a, it, row0, row0 + wave, min(row0 + 32, rows), 4, b0 * PB, b1 * PB, (long long)it.slot * 32);
    __syncthreads();
    return;
  }
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) M = fmaxf(M, ml[i][0][w.fr]);
  const float f = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((w.m - M) * w.c);
  float* ob = (float*)lds;
  const int valid = min(32, rows - row0);
#pragma unroll
  for (int half = 0; half < D / 64; ++half) {   // dims 64 half .. + 64
    if (half) __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const pt_f32x16& o = w.o[2 * half + t];
        float4 v;
        v.x = o[4 * i] * f, v.y = o[4 * i + 1] * f, v.z = o[4 * i + 2] * f, v.w = o[4 * i + 3] * f;
        *(float4*)&ob[(wave * 32 + w.fr) * OLD + t * 32 + 8 * i + 4 * w.hi] = v;
      }
    __syncthreads();
    for (int idx = tid; idx < valid * 8; idx += 256) {   // (row, 8 dims)
      const int ch = idx & 7, r = idx >> 3;
      float Mr = -INFINITY, L = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) Mr = fmaxf(Mr, ml[i][0][r]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        L += ml[i][0][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i][0][r] - Mr) * w.c) * ml[i][1][r];
      float x[8] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4* p = (const float4*)&ob[(i * 32 + r) * OLD + 8 * ch];
        const float4 u = p[0], v = p[1];
        x[0] += u.x, x[1] += u.y, x[2] += u.z, x[3] += u.w;
        x[4] += v.x, x[5] += v.y, x[6] += v.z, x[7] += v.w;
      }
      if (it.slot >= 0) {
        float* po = a.part_o + ((long long)it.slot * 32 + r) * D + 64 * half + 8 * ch;
        *(float4*)po = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(po + 4) = make_float4(x[4], x[5], x[6], x[7]);
        if (half == 0 && ch == 0) *(float2*)(a.part_ml + ((long long)it.slot * 32 + r) * 2) = make_float2(Mr, L);
      } else {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int row = row0 + r, t = row / G;
        uint16_t* out = (uint16_t*)a.out + ((long long)(it.q.start + t) * a.H + it.h * G + row - t * G) * D + 64 * half + 8 * ch;
        *(uint4*)out = make_uint4(gm_pack2<DT>(x[0] * inv, x[1] * inv), gm_pack2<DT>(x[2] * inv, x[3] * inv),
                                  gm_pack2<DT>(x[4] * inv, x[5] * inv), gm_pack2<DT>(x[6] * inv, x[7] * inv));
      }
    }
  }
  __syncthreads();   // the next item's loads go to the same LDS
}

// ------------------------------------------------------------------ wide tiles

template <int DT, int D>
__device__ __forceinline__ void pt_wide(const PagedAttnArgs& a, const PtItem& it, char* lds, int (*slots)[64]) {
  constexpr int PB = 64, NB = 2, NG = 4, RB = 2 * D, BYTES = PB * RB;   // bytes of a block's K, and of its V
  constexpr int LPG = RB * 16 / 1024;                                   // loads per group: each wave takes its group's
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.H / a.KVH, rows = it.q.n * G, tile0 = it.tile * PT_WIDE, row0 = tile0 + wave * 32;
  const unsigned row_bytes = (unsigned)(2 * a.row_stride);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
  const int first = it.q.kv - it.q.n;   // position of token 0
  const int tlast = min(tile0 + PT_WIDE - 1, rows - 1) / G;
  const int b0 = it.b0, b1 = it.b1;
  constexpr int WB = 64 / NG;   // blocks of a window
  PtWindow cur;
  int* ids = slots[wave];
  int wi = b0 / WB;             // window of cur
  unsigned bad = 0, bad_next = 0;   // groups of the present and the next block without a page
  auto issue = [&](int blk) {
    if (blk / WB != wi) {
      ++wi;
      cur = pt_window(a, it, wi * 64, ids[lane]);
      pt_fetch(a, it, (wi + 1) * 64, ids);
    }
    bad_next = ~(unsigned)(cur.ok >> (blk % WB * NG)) & ((1u << NG) - 1);
    const unsigned dst = lds0 + (unsigned)(blk & 1) * 2 * BYTES + (unsigned)wave * LPG * 1024;
    const unsigned long long at = pt_place(cur, blk % WB * NG + wave);
    const char *k = (const char*)a.k_pages + at, *v = (const char*)a.v_pages + at;
#pragma unroll
    for (int i = 0; i < LPG; ++i) pt_load<D, false>(k, row_bytes, i, dst + i * 1024, lane);
#pragma unroll
    for (int i = 0; i < LPG; ++i) pt_load<D, true>(v, row_bytes, i, dst + BYTES + i * 1024, lane);
  };
  if (b0 < b1) {
    cur = pt_window(a, it, wi * 64);
    pt_fetch(a, it, (wi + 1) * 64, ids);
    issue(b0);
  }
  PtWave<DT, D> w;
  w.init(a, it, row0);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" ::"v"(w.qf[ks].x), "v"(w.qf[ks].y), "v"(w.qf[ks].z), "v"(w.qf[ks].w));
  // positions that every row of the wave has open, and that any has
  const int pmin = __builtin_amdgcn_readfirstlane(w.pos);
  const int pmax = row0 < rows ? __builtin_amdgcn_readlane(w.pos, 31) : -1;
  const int pend = (int)min((long long)first + tlast, (long long)a.M * a.page_size - 1);   // the tile's last row's
  for (int blk = b0; blk < b1; ++blk) {
    gm_vmcnt<0>();
    __syncthreads();   // the block is in LDS, and every wave is done with the other stage
    bad = bad_next;
    if (blk + 1 < b1) issue(blk + 1);
    if (blk * PB > pmax) continue;   // wave-uniform
    const bool open = blk * PB + PB - 1 <= pmin && bad == 0;
    char* Kt = lds + (blk & 1) * 2 * BYTES;
    char* Vt = Kt + BYTES;
    pt_f32x16 s[NB];
    w.template scores<NB>(Kt, s);
    if (!open) w.template mask<NB>(s, blk * PB, bad);
    __builtin_amdgcn_s_setprio(1);   // vector instructions first: the other workgroup's matrix instructions run on beside them
    w.template softmax<NB>(s);
    uint4 p[2 * NB];
    w.template pack<NB>(s, p);
    __builtin_amdgcn_s_setprio(0);
    if (blk * PB + PB - 1 > pend || bad) w.template clear_closed<NB>(Vt, blk * PB, pend, bad);
    w.template outputs<NB>(Vt, p, s);
  }
  const float l = w.row_sum();
  const int row = row0 + w.fr;
  const long long part = (long long)2 * a.grid_narrow * PT_NARROW + (long long)it.slot * PT_WIDE;
  if (row0 < rows && w.bad_output()) {
    pt_rows<DT, D>(a, it, tile0, row0, min(row0 + 32, rows), 1, b0 * PB, b1 * PB, part);
  } else if (row < rows) {
    if (it.slot >= 0) {
      const long long at = part + row - tile0;
      if (w.hi == 0) *(float2*)(a.part_ml + at * 2) = make_float2(w.m, l);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(float4*)(a.part_o + at * D + 32 * t + 8 * i + 4 * w.hi) =
              make_float4(w.o[t][4 * i], w.o[t][4 * i + 1], w.o[t][4 * i + 2], w.o[t][4 * i + 3]);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int t0 = row / G;
      uint16_t* out = (uint16_t*)a.out + ((long long)(it.q.start + t0) * a.H + it.h * G + row - t0 * G) * D;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(uint2*)(out + 32 * t + 8 * i + 4 * w.hi) =
              make_uint2(gm_pack2<DT>(w.o[t][4 * i] * inv, w.o[t][4 * i + 1] * inv),
                         gm_pack2<DT>(w.o[t][4 * i + 2] * inv, w.o[t][4 * i + 3] * inv));
    }
  }
  __syncthreads();   // the next item's loads go to the same LDS
}

// ------------------------------------------------------------------ pages of 8 bits
//
// The same tiles over e4m3 numbers K_jd 2^ke_j and V_jd 2^ve_j. The products stay in 16 bits: e4m3 queries or probabilities
// would carry 3 bits of mantissa into every output. Numbers of 4 bits are exact in bfloat16, and in float16 while they are
// multiples of 2^-24, which e4m3 numbers times 2^-15 (byte 112) are. Keys of smaller powers enter float16 products without
// them, and their scores are multiplied by them in 32 bits: whether a block (wide: a group of 16 positions) has such is one
// test of its bytes (a wide tile's waves tell each other in LDS: a mixed step in float16 67.8 -> 69.5 us).
//   * Narrow: half the bytes come to LDS, and become 16 bits on the way from there to the matrix instructions. A lane of
//     K's operand holds one position, so 2^ke_j comes with the conversion. A lane of V's holds eight positions of one dim:
//     2^ve_j goes to the probabilities, which are therefore taken in bfloat16 (whose range holds any power of two) whatever the
//     queries' type, for float16 in two parts, the second the first's rounding error, each with its product: float16's own
//     11 bits at least, where bfloat16's outputs have 8 bits as its probabilities do. Bound by memory, which hides the second
//     product: 64 decodes of up to 4,096 positions (32 + 8 heads of 128, 412 MB) take 88 us, 4.7 TB/s (153 from 16-bit pages),
//     four of up to 131,071 (12 + 2) 40 (76).
//   * Wide: bound by the matrix cores, so each block is converted once for all four waves, powers of two included, by way of
//     registers one block ahead, into the LDS layout of 16-bit pages; the rest is the 16-bit tile. The conversion's vector
//     instructions and LDS writes come on top of the softmax's: 409 tokens over 30,409 positions (12 + 2 heads) take 106 us, 0.72
//     PFLOP/s, rather than 93. (Softmax of one block between the products of another within a wave: 4.4 us a block rather than
//     2.3 at head size 128, since its registers spill; three workgroups a CU at head size 64 spill too: 78 us rather than 70 for a
//     mixed step.)
// K in float16 can overflow where 2^ke is 2^8 or more (keys above 57,344), bfloat16 where a power is 2^120; probabilities times
// powers below 2^-100 reach the end of bfloat16; byte 255 is NaN: tiles that see such a byte in an open place are done row
// by row, like those with outputs that are not finite. (0, what was never written, is none of them: it counts as 0.
// A wide tile holds V in float16, in steps of 2^-24 below 2^-14: half a step, 2^-25, is as much as the rounding of outputs so
// small is off.)

template <int DT>
constexpr unsigned pt_least_odd = DT == HS_F16 ? 135u : 247u;   // odd power bytes: 1 .. 26, and from here on
__device__ __forceinline__ bool pt_odd(unsigned byte, unsigned least) { return byte - 1u < 26u || byte >= least; }

// whether one of four bytes is odd: bit 7 of a byte's sum says whether it is at least the number that takes 128 to it
__device__ __forceinline__ bool pt_any_odd(uint32_t w, unsigned least) {
  constexpr uint32_t ONES = 0x01010101u;
  const uint32_t low = w & (0x7f * ONES), top = w & (0x80 * ONES);
  const uint32_t from_least = (low + (256u - least) * ONES) & top, from_1 = low + 0x7f * ONES, from_27 = low + (128u - 27u) * ONES;
  return (from_least | (from_1 & ~from_27 & ~w & (0x80 * ONES))) != 0;
}

// The first power byte from which the conversion to DT is exact for every number, which are multiples of 2^-9 (bfloat16: for all
// that are not odd, but 0, which the conversion would take as 2^-127).
template <int DT>
constexpr unsigned pt_exact_from = DT == HS_F16 ? 112u : 1u;
// whether one of four bytes is below `from` (1 .. 128)
__device__ __forceinline__ bool pt_any_below(uint32_t w, unsigned from) {
  constexpr uint32_t ONES = 0x01010101u;
  return ((((w & (0x7f * ONES)) + (128u - from) * ONES) | w) & (0x80 * ONES)) != 0x80 * ONES;
}

// four e4m3 numbers times 0: NaN (0x7f, 0xff) or 0
__device__ __forceinline__ uint32_t pt_times_0(uint32_t w) {
  constexpr uint32_t ONES = 0x01010101u;
  return ((((w & (0x7f * ONES)) + ONES) >> 7) & ONES) * 0x7f;
}

// four scores, s[at ..], times the powers of four bytes
__device__ __forceinline__ void pt_times_powers(pt_f32x16& s, int at, uint32_t u) {
  s[at] *= __uint_as_float((u << 23) & 0x7f800000u);
  s[at + 1] *= __uint_as_float((u << 15) & 0x7f800000u);
  s[at + 2] *= __uint_as_float((u << 7) & 0x7f800000u);
  s[at + 3] *= __uint_as_float((u >> 1) & 0x7f800000u);
}

// eight e4m3 numbers times 2^(power - 127) as DT
template <int DT>
__device__ __forceinline__ uint4 pt_widen(uint32_t a, uint32_t b, float power) {
  uint4 r;
  if constexpr (DT == HS_BF16) {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, true));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, power, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, power, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, power, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, power, true));
  }
  return r;
}

// pack for 16 positions: the lane's eight values in the B operand's layout
template <int DT>
__device__ __forceinline__ uint4 pt_pack16(const float (&e)[8]) {
  uint32_t g[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) g[i] = gm_pack2<DT>(e[2 * i], e[2 * i + 1]);
  pt_swap32(g[0], g[2]);
  pt_swap32(g[1], g[3]);
  return make_uint4(g[0], g[1], g[2], g[3]);
}

// Transposing LDS read of bytes: lanes 2r + c of each 16-lane group address row r, columns 8c .. 8c + 7; lane i gets column i
// of rows 0 .. 7.
__device__ __forceinline__ uint2 pt_read_tr8(const char* p) {
  typedef __attribute__((ext_vector_type(2))) int i32x2;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                       (__attribute__((address_space(3))) i32x2*)(__attribute__((address_space(3))) char*)p));
}

// Rows' swizzles, as pt_xk and pt_xv, for rows of D bytes: the 32 rows of K's 16-byte reads, and the 8 rows x 2 chunks of V's
// transposing reads by 32 lanes, hit every bank.
template <int D>
__device__ __forceinline__ int pt_xk8(int r) {
  return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int pt_xv8(int r) {
  return D == 128 ? ((r >> 1) & 3) << 1 : ((r >> 2) & 1) << 1;
}
template <int D, bool V>
__device__ __forceinline__ void pt_load8(const char* group, unsigned row_bytes, int i, unsigned lds, int lane) {
  constexpr int PER = 1024 / D, SL = D / 16;   // rows per load, slots of a row
  const int r = i * PER + lane / SL, ch = (lane % SL) ^ (V ? pt_xv8<D>(r) : pt_xk8<D>(r));
  gm_dma16s(group, (unsigned)r * row_bytes + ch * 16, lds);
}

// Writes the rows row0 .. of one wave, of a tile that begins at row tile0: as outputs, or as a part (whose first row is
// `part`). `odd` (uniform): the wave's outputs are not to be used, as where they are not finite. (For these pages: with pt_wide's
// end as this function the 16-bit kernel takes other registers, and one token 13.9 us rather than 13.6.)
template <int DT, int D>
__device__ __forceinline__ void pt_end(const PagedQuantAttnArgs& a, const PtItem& it, const PtWave<DT, D>& w, int tile0, int row0,
                                       int rows, int p0, int p1, long long part, bool odd) {
  const int G = a.H / a.KVH;
  const float l = w.row_sum();
  const int row = row0 + w.fr;
  if (row0 < rows && (odd || w.bad_output())) {
    pt_rows<DT, D, true>(a, it, tile0, row0, min(row0 + 32, rows), 1, p0, p1, part);
  } else if (row < rows) {
    if (it.slot >= 0) {
      const long long at = part + row - tile0;
      if (w.hi == 0) *(float2*)(a.part_ml + at * 2) = make_float2(w.m, l);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(float4*)(a.part_o + at * D + 32 * t + 8 * i + 4 * w.hi) =
              make_float4(w.o[t][4 * i], w.o[t][4 * i + 1], w.o[t][4 * i + 2], w.o[t][4 * i + 3]);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int t0 = row / G;
      uint16_t* out = (uint16_t*)a.out + ((long long)(it.q.start + t0) * a.H + it.h * G + row - t0 * G) * D;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(uint2*)(out + 32 * t + 8 * i + 4 * w.hi) =
              make_uint2(gm_pack2<DT>(w.o[t][4 * i] * inv, w.o[t][4 * i + 1] * inv),
                         gm_pack2<DT>(w.o[t][4 * i + 2] * inv, w.o[t][4 * i + 3] * inv));
    }
  }
}

// Work, dealt out in equal ranges to the last block: narrow tiles' blocks to waves, wide tiles' to workgroups. A range begins
// and ends inside tiles, whose parts its slots 2 w (a part behind another) and 2 w + 1 (a tile's first part) take.
struct PtItem8 : PtItem {
  int parts;   // a tile's first part: how many there are. 0: a later one
};

// A tile's first part tells k_paged_quant_combine where each of its rows' parts are: [first part's row, 2 parts + kind].
__device__ __forceinline__ void pt_tell(const PagedQuantAttnArgs& a, const PtItem8& it, int row, int rows, long long part, int wide) {
  const int G = a.H / a.KVH, t = row / G;
  if (it.parts && row < rows && (threadIdx.x & 63) < 32)
    ((int2*)a.joins)[(long long)(it.q.start + t) * a.H + it.h * G + row - t * G] = make_int2((int)part, 2 * it.parts + wide);
}

// Of a block of a wide tile in float16: whether the keys' powers of its groups of 16 positions enter by the scores (a byte
// each), and those powers
struct PtPowers {
  uint32_t after, k[16];
};

struct PtList8 {
  union {
    int items[PT_MAXB];                  // narrow: running sums of blocks
    unsigned long long cost[PT_MAXB];    // wide: of costs (pt_cost)
  };
  int red[3][4];
  unsigned long long red64[4];
};

// Narrow sequences' blocks, as pt_build_narrow.
__device__ __forceinline__ int pt_build_narrow8(const PagedAttnArgs& a, PtList8& t, int hi) {
  int total[3] = {0, 0, 0};
  for (int c = 0; c < a.B; c += 256) {
    const int b = c + threadIdx.x;
    int v[3] = {0, 0, 0};
    if (b < a.B) {
      const int s0 = a.q_start[b], s1 = a.q_start[b + 1];
      const PtSeq q = pt_seq<PT_NARROW, 64>(a, b, s0, s1, a.kv_len[b], 0, hi);
      v[0] = q.tiles * q.blocks * a.KVH;
      v[1] = s1 < s0;
    }
    pt_scan3(v, total, t.red);
    if (b < a.B) t.items[b] = v[0];
  }
  __syncthreads();
  return total[1] ? 0 : total[0];
}

// The item of wave w that starts at block `at` of all narrow blocks; `end`: of its range. Returns the next start.
__device__ __forceinline__ int pt_item_narrow8(const PagedAttnArgs& a, const PtList8& t, int w, int at, int end, int hi, int all,
                                               int workers, PtItem8& it) {
  it.b = __builtin_amdgcn_readfirstlane(pt_find(t.items, a.B, at));
  it.q = pt_seq<PT_NARROW, 64>(a, it.b, pt_ldc(a.q_start, it.b), pt_ldc(a.q_start, it.b + 1), pt_ldc(a.kv_len, it.b), 0, hi);
  const int i = at - (it.b ? __builtin_amdgcn_readfirstlane(t.items[it.b - 1]) : 0), tl = i / it.q.blocks;
  it.tile = tl % it.q.tiles, it.h = tl / it.q.tiles;
  it.b0 = i % it.q.blocks, it.b1 = min(it.q.blocks, it.b0 + end - at);
  const int next = at + it.b1 - it.b0;
  const bool split = it.b1 < it.q.blocks;
  it.slot = it.b0 > 0 ? 2 * w : split ? 2 * w + 1 : -1;
  // (the wave that holds the tile's last block)
  it.parts = it.b0 > 0 ? 0 : split ? (int)((((long long)at + it.q.blocks) * workers - 1) / all) - w + 1 : 1;
  const int seen = pt_seen<PT_NARROW, 64>(a, it.q, it.tile);
  it.b0 = min(it.b0, seen), it.b1 = min(it.b1, seen);
  return next;
}

// What wide tiles cost, in positions times G: tile i of a sequence sees about the positions before its first token and
// those of (i + 1/2) 128 / G tokens, and begins and ends in the time of two blocks.
struct PtCost {
  long long c0, head;   // of tile 0 (tile i: c0 + 128 i), and of all tiles of a K/V head
  __device__ __forceinline__ PtCost(const PagedAttnArgs& a, const PtSeq& q) {
    const int G = a.H / a.KVH;
    c0 = (min((long long)max(q.kv - q.n, 0), (long long)a.M * a.page_size) + 128) * G + 64;
    head = before(q.tiles);
  }
  __device__ __forceinline__ long long before(int i) const { return i * c0 + 64ll * i * (i - 1); }
};

// Wide sequences' costs (by 256 threads; ends with a barrier); returns their sum, 0 where q_start descends.
__device__ __forceinline__ unsigned long long pt_build_wide8(const PagedAttnArgs& a, PtList8& t) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned long long total = 0;
  bool down = false;
  for (int c = 0; c < a.B; c += 256) {
    const int b = c + tid;
    unsigned long long v = 0;
    if (b < a.B) {
      const int s0 = a.q_start[b], s1 = a.q_start[b + 1];
      const PtSeq q = pt_seq<PT_WIDE, 64>(a, b, s0, s1, a.kv_len[b], PT_NARROW, 0x7fffffff);
      down |= s1 < s0;
      if (q.n) v = (unsigned long long)PtCost(a, q).head * a.KVH;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long w = __shfl_up(v, o, 64);
      if (lane >= o) v += w;
    }
    __syncthreads();
    if (lane == 63) t.red64[wave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) v += w < wave ? t.red64[w] : 0;
    v += total;
    if (b < a.B) t.cost[b] = v;
#pragma unroll
    for (int w = 0; w < 4; ++w) total += t.red64[w];
  }
  return __syncthreads_or(down) ? 0 : total;
}

// A place in the wide tiles' list: block blk of a tile of a K/V head of sequence b (B: the end).
struct PtCut {
  int b, h, tile, blk;
  __device__ __forceinline__ bool in(const PtCut& o) const { return b == o.b && h == o.h && tile == o.tile; }
};
// Fewest blocks that a range is worth, about those of a tile of one: us of 16 prompts of 16 tokens (32 + 8 heads of 128) at 8 / 4 /
// 2 / 1 31 / 20 / 16 / 17, of 64 tokens 36 / 24 / 20 / 21, one of 256 35 / 26 / 20 / 20; 64 tokens behind 2,000 33 / 28 / 28 / 29.
#define PT_RANGE_LEAST 2
struct PtRanges {
  unsigned long long total;
  unsigned long long range;   // of a workgroup
  int workers;
};

__device__ __forceinline__ unsigned long long pt_cost_at(const PtList8& t, int b) { return b < 0 ? 0 : t.cost[b]; }   // of the sequences up to b
// the tile behind c's, at its first block
__device__ __forceinline__ PtCut pt_behind(const PagedAttnArgs& a, const PtList8& t, int tiles, PtCut c) {
  c.blk = 0;
  if (++c.tile < tiles) return c;
  c.tile = 0;
  if (++c.h < a.KVH) return c;
  c.h = 0;
  const unsigned long long here = pt_cost_at(t, c.b);
  while (++c.b < a.B && pt_cost_at(t, c.b) == here) {
  }
  return c;
}
// Where workgroup w's range begins; a lane each may ask for another w. Ranges are of equal cost, but where tiles are short
// against them one that would begin within an eighth of a range from a tile's border begins there, so that fewer tiles have
// parts to be written and read again (of many prompts, else, nearly every range would begin inside a tile).
__device__ __forceinline__ PtCut pt_cut(const PagedAttnArgs& a, const PtList8& t, const PtRanges& r, int w) {
  if (w >= r.workers) return PtCut{a.B, 0, 0, 0};
  const unsigned long long x = r.range * w + r.total % r.workers * w / r.workers;
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (pt_cost_at(t, mid) > x) hi = mid;
    else lo = mid + 1;
  }
  PtCut c{lo, 0, 0, 0};
  const PtSeq q = pt_seq<PT_WIDE, 64>(a, lo, a.q_start[lo], a.q_start[lo + 1], a.kv_len[lo], PT_NARROW, 0x7fffffff);
  const PtCost k(a, q);
  long long z = (long long)(x - pt_cost_at(t, lo - 1));
  c.h = min((int)((double)z / (double)k.head), a.KVH - 1);
  while (z < c.h * k.head) --c.h;
  while (c.h + 1 < a.KVH && z >= (c.h + 1) * k.head) ++c.h;
  z -= c.h * k.head;
  const double p = (double)(k.c0 - 64);
  c.tile = max(0, min((int)((sqrt(p * p + 256.0 * (double)z) - p) * (1.0 / 128.0)), q.tiles - 1));
  while (c.tile > 0 && z < k.before(c.tile)) --c.tile;
  while (c.tile + 1 < q.tiles && z >= k.before(c.tile + 1)) ++c.tile;
  z -= k.before(c.tile);
  const int nb = pt_seen<PT_WIDE, 64>(a, q, c.tile), per = 64 * (a.H / a.KVH);
  const int range = (int)min(r.range / per, 1ull << 30);   // in blocks
  c.blk = min((int)((double)nb * (double)z / (double)(k.c0 + 128ll * c.tile)), nb);
  const int near = nb <= range ? max(1, range / 8) : 1;
  if (c.blk <= near) c.blk = 0;
  else if (nb - c.blk <= near) c = pt_behind(a, t, q.tiles, c);
  return c;
}
__device__ __forceinline__ PtCut pt_cut_of(const PtCut& c, int lane) {
  return PtCut{__builtin_amdgcn_readlane(c.b, lane), __builtin_amdgcn_readlane(c.h, lane), __builtin_amdgcn_readlane(c.tile, lane),
               __builtin_amdgcn_readlane(c.blk, lane)};
}

// Workgroup w's range, and how many begin inside the tile inside which it ends.
struct PtRange {
  PtCut at, end;
  int inside;
  __device__ __forceinline__ bool done() const { return at.in(end) && at.blk == end.blk; }
};
__device__ __forceinline__ PtRange pt_range(const PagedAttnArgs& a, const PtList8& t, const PtRanges& r, int w) {
  const int lane = threadIdx.x & 63;
  PtCut c = pt_cut(a, t, r, w + lane);
  PtRange g{pt_cut_of(c, 0), pt_cut_of(c, 1), 0};
  if (g.end.blk == 0) return g;
  for (int base = w;; base += 64) {   // (they follow each other)
    const int n = __popcll(__ballot(c.in(g.end) && c.blk > 0 && base + lane > w));
    g.inside += n;
    if (__builtin_amdgcn_readlane(c.in(g.end) ? 1 : 0, 63) == 0) return g;
    c = pt_cut(a, t, r, base + 64 + lane);
  }
}

// The item of workgroup w at its range's place, which moves on.
__device__ __forceinline__ PtItem8 pt_item_wide8(const PagedAttnArgs& a, const PtList8& t, int w, PtRange& g) {
  PtItem8 it;
  it.b = g.at.b, it.h = g.at.h, it.tile = g.at.tile;
  it.q = pt_seq<PT_WIDE, 64>(a, it.b, pt_ldc(a.q_start, it.b), pt_ldc(a.q_start, it.b + 1), pt_ldc(a.kv_len, it.b), PT_NARROW, 0x7fffffff);
  const int nb = pt_seen<PT_WIDE, 64>(a, it.q, it.tile);
  const bool split = g.at.in(g.end);   // (the end of a range is its tile's first block, or one inside)
  it.b0 = g.at.blk, it.b1 = split ? g.end.blk : nb;
  it.slot = it.b0 > 0 ? 2 * w : split ? 2 * w + 1 : -1;
  it.parts = it.b0 > 0 ? 0 : split ? g.inside + 1 : 1;
  if (split) {
    g.at = g.end;
  } else {
    const PtCut c = pt_behind(a, t, it.q.tiles, g.at);
    g.at = PtCut{__builtin_amdgcn_readfirstlane(c.b), c.h, c.tile, 0};
  }
  return it;
}

template <int DT, int D>
__device__ __forceinline__ void pt_narrow8(const PagedQuantAttnArgs& a, const PtItem8& it, char* lds, int (*slots)[64], uint32_t (*powers)[64]) {
  using C = PtNarrow<DT, D, true>;
  constexpr int PB = C::PB, NB = C::NB, NG = C::NG, LPG = C::LPG, TD = D / 32;
  constexpr int LD = NG * LPG;   // loads of a block's K, and of its V
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = it.tile * 32;
  PtWave<DT, D> w;
  const unsigned row_bytes = (unsigned)a.row_stride;
  char* Kt = lds + wave * 16384;
  char* Vt = Kt + 8192;
  const unsigned k0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)Kt, v0 = k0 + 8192;
  uint32_t* pw = powers[wave];   // the block's powers of two: K's 64 bytes, then V's
  const unsigned pw0 = (unsigned)(size_t)(__attribute__((address_space(3))) uint32_t*)pw;
  const int b0 = it.b0, b1 = it.b1;
  constexpr int WB = 64 / NG;   // blocks of a window
  PtWindowT<true> cur;
  int* ids = slots[wave];
  int wi;                       // window of cur
  unsigned bad = 0, bad_next;   // groups of the present and the next block without a page
  bool odd = false;
  auto seek = [&](int blk) {    // cur: the block's window
    if (blk / WB != wi) {
      ++wi;
      cur = pt_window<true>(a, it, wi * 64, ids[lane]);
      pt_fetch(a, it, (wi + 1) * 64, ids);
    }
    return ~(unsigned)(cur.ok >> (blk % WB * NG)) & ((1u << NG) - 1);
  };
  auto load = [&](auto v, int blk) {
    constexpr bool V = decltype(v)::value;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const char* p = (const char*)(V ? a.v_pages : a.k_pages) + pt_place(cur, blk % WB * NG + g);
#pragma unroll
      for (int i = 0; i < LPG; ++i) pt_load8<D, V>(p, row_bytes, i, (V ? v0 : k0) + (g * LPG + i) * 1024, lane);
    }
  };
  auto load_powers = [&](int blk) {   // lane i of 32: four bytes of K's (i < 16) or V's; the upper half repeats them
    const int g = blk % WB * NG + ((lane & 15) >> 2);
    const unsigned long long at = ((unsigned long long)(uint32_t)__shfl((int)(cur.scale >> 32), g, 64) << 32) |
                                  (uint32_t)__shfl((int)(uint32_t)cur.scale, g, 64);
    const unsigned char* p = ((lane & 16) ? a.v_scales : a.k_scales) + at + (lane & 3) * 4;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(pw0) : "memory", "m0");
  };
  int blk = b0;
  if (blk < b1) {
    wi = blk / WB;
    cur = pt_window<true>(a, it, wi * 64);
    pt_fetch(a, it, (wi + 1) * 64, ids);
    bad = seek(blk);
    load_powers(blk);
    load(PtK{}, blk);
    load(PtV{}, blk);
  }
  w.template init<true>(a, it, row0);
  // the queries are waited for here: at their first use the wait would cover the loads in flight of every block
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" ::"v"(w.qf[ks].x), "v"(w.qf[ks].y), "v"(w.qf[ks].z), "v"(w.qf[ks].w));
  // positions that the tile's first row has open, and its last
  const int pmin = __builtin_amdgcn_readfirstlane(w.pos), pend = __builtin_amdgcn_readlane(w.pos, 31);
  for (; blk < b1; ++blk) {
    const bool more = blk + 1 < b1;
    const bool open = blk * PB + PB - 1 <= pmin && bad == 0;
    gm_vmcnt<LD>();   // powers and K have landed; V's loads may be on their way
    asm volatile("" ::: "memory");
    if (blk * PB + PB - 1 > pend || bad) {   // the powers of places closed to every row: anything (0 x NaN)
      if (lane < 32) {
        const int j = (lane & 15) * 4;
        uint32_t p = pw[lane];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (blk * PB + j + i > pend || ((bad >> (j >> 4)) & 1)) p = (p & ~(255u << (8 * i))) | (127u << (8 * i));
        pw[lane] = p;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    const uint32_t four = pw[lane & 31];
    odd = odd || pt_any_odd(four, pt_least_odd<DT>);
    // K's powers enter with the conversion where it is exact, else by the scores (uniform)
    const bool after = (__ballot(pt_any_below(four, pt_exact_from<DT>)) & 0xffffull) != 0;
    uint32_t vp[NB][4];   // V's powers, at the places of the lane's scores
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int i = 0; i < 4; ++i) vp[sb][i] = pw[16 + sb * 8 + 2 * i + w.hi];
    // S^T = K Q^T
    pt_f32x16 s[NB];
    {
      constexpr int KS = D / 32;   // 16-byte reads of a position
      uint4 k[KS];
      auto read = [&](int sb, int ks) { return *(const uint4*)(Kt + (sb * 32 + w.fr) * D + (((2 * ks + w.hi) ^ pt_xk8<D>(w.fr)) * 16)); };
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) k[ks] = read(0, ks);
#pragma unroll
      for (int sb = 0; sb < NB; ++sb) {
        const float power = after ? 1.f : __uint_as_float((uint32_t)((const unsigned char*)pw)[sb * 32 + w.fr] << 23);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[sb][e] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s[sb] = pt_mfma<DT>(pt_widen<DT>(k[ks].x, k[ks].y, power), w.qf[2 * ks], s[sb]);
          s[sb] = pt_mfma<DT>(pt_widen<DT>(k[ks].z, k[ks].w, power), w.qf[2 * ks + 1], s[sb]);
          if (sb + 1 < NB) k[ks] = read(sb + 1, ks);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (after)
#pragma unroll
      for (int sb = 0; sb < NB; ++sb)
#pragma unroll
        for (int i = 0; i < 4; ++i) pt_times_powers(s[sb], 4 * i, pw[sb * 8 + 2 * i + w.hi]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K's rows and the powers are in registers
    if (more) {
      bad_next = seek(blk + 1);
      load_powers(blk + 1);
      load(PtK{}, blk + 1);
    }
    if (!open) w.template mask<NB>(s, blk * PB, bad);
    w.template softmax<NB>(s);
    if (more) gm_vmcnt<LD + 1>();   // V has landed; the next powers' and K's loads may be on their way
    else gm_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (blk * PB + PB - 1 > pend || bad) {
      constexpr int SL = D / 16;
#pragma unroll 1
      for (int i = lane; i < PB * SL; i += 64) {
        const int j = i / SL;
        if (blk * PB + j > pend || ((bad >> (j >> 4)) & 1)) *(uint4*)(Vt + i * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    // O^T += V^T P^T, 32 positions at a time, the operands read four ahead
    float sum[2] = {w.l, 0.f};
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
      constexpr int N = 2 * TD;
      auto read = [&](int i) {   // rows 8 hi + r of half block i / TD, dims 32 t + 16 g + 8 c
        const int r = sb * 32 + (i / TD) * 16 + 8 * w.hi + ((lane & 15) >> 1), ch = 2 * (i % TD) + ((lane >> 4) & 1);
        return pt_read_tr8(Vt + r * D + ((ch ^ pt_xv8<D>(r)) * 16) + (lane & 1) * 8);
      };
      uint2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = read(i);
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // 16 positions
        float e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float x = s[sb][8 * h + k];
          sum[k & 1] += x;
          const uint32_t u = vp[sb][2 * h + (k >> 2)];
          const uint32_t f = (k & 3) == 0 ? u << 23 : (k & 3) == 1 ? u << 15 : (k & 3) == 2 ? u << 7 : u >> 1;
          e[k] = x * __uint_as_float(f & 0x7f800000u);
        }
        const uint4 p = pt_pack16<HS_BF16>(e);
        uint4 p2;
        if constexpr (DT == HS_F16) {   // the rounding errors, in turn
#pragma unroll
          for (int k = 0; k < 8; ++k) e[k] -= gm_round<HS_BF16>(e[k]);
          p2 = pt_pack16<HS_BF16>(e);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = h * TD; i < h * TD + TD; ++i) {
          const uint4 vf = pt_widen<HS_BF16>(v[i % 4].x, v[i % 4].y, 1.f);
          w.o[i % TD] = pt_mfma<HS_BF16>(vf, p, w.o[i % TD]);
          if constexpr (DT == HS_F16) w.o[i % TD] = pt_mfma<HS_BF16>(vf, p2, w.o[i % TD]);
          if (i + 4 < N) v[i % 4] = read(i + 4);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    w.l = sum[0] + sum[1];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) load(PtV{}, blk + 1);
    bad = bad_next;
  }
  const int rows = it.q.n * (a.H / a.KVH);
  const long long part = (long long)it.slot * PT_NARROW;
  pt_tell(a, it, row0 + w.fr, rows, part + w.fr, 0);
  pt_end<DT, D>(a, it, w, row0, row0, rows, b0 * PB, b1 * PB, part, __ballot(odd) != 0ull);
}

// A workgroup's range of the wide tiles. The next item's first block is on its way while the last of the present one is
// computed, its pages' ids before that. XCD i (workgroups i, i + 8, ...) takes neighbouring ranges: they read the same blocks.
template <int DT, int D>
__device__ __forceinline__ void pt_wide8(const PagedQuantAttnArgs& a, PtList8& t, char* lds, int (*slots)[64], PtPowers* kpw) {
  constexpr int PB = 64, NB = 2, NG = 4, RB = 2 * D, BYTES = PB * RB;   // bytes of a block's K, and of its V, in 16 bits
  constexpr int PCS = D / 64;                                           // 16-byte pieces of a row that a thread takes, of K and of V
  constexpr int WB = 64 / NG, TD = D / 32;                              // blocks of a window; output tiles
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.H / a.KVH;
  if (DT == HS_F16 && tid < 2) kpw[tid].after = 0;
  PtRanges r;
  r.total = pt_build_wide8(a, t);   // (a barrier)
  r.workers = (int)max(1ull, min((unsigned long long)a.grid_wide, r.total / (PT_RANGE_LEAST * PB * G)));
  r.range = r.total / r.workers;
  const int each = (r.workers + 7) >> 3, me = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if (r.total == 0 || (int)(blockIdx.x >> 3) >= each || me >= r.workers) return;
  PtRange range = pt_range(a, t, r, me);
  if (range.done() && range.at.blk == 0) return;   // (inside a tile: an empty part, since the others count it)
  int* ids = slots[wave];
  PtWindowT<true> cur;
  int wi = 0;                       // window of cur
  unsigned bad = 0, bad_next = 0;   // groups of the present and the next block without a page
  // A wave converts its group of 16 positions, four lanes a position. LDS takes the writes of 8 lanes at a time, two positions'
  // here: K's swizzle sends those to different banks (D = 64: of positions 0 and 2), for V every other position writes its
  // odd chunk first.
  const int gr = D == 128 ? lane >> 2 : (lane >> 4) << 2 | ((lane >> 2) & 1) << 1 | ((lane >> 3) & 1), part = lane & 3;
  const bool turn = (lane >> 2) & 1;
  const unsigned ko = (unsigned)gr * (unsigned)a.row_stride + part * 16;   // 16-byte pieces part + 4 i of a row
  // Places in LDS. A swizzle is an exclusive or, so a fragment's place is another's with a constant: one instruction each from
  // a place that changes with the block, where the compiler would keep thirty in registers (and spill: a reload waits
  // for the loads in flight). Fragments as PtWave's: chunk 2 ks + hi of K's row fr; of V's, two times four rows, 4 apart.
  const int fr = lane & 31, hi = lane >> 5, vrow = (lane & 15) >> 2, sr = wave * 16 + gr;
  const unsigned krd = fr * RB + ((hi ^ pt_xk<D>(fr)) * 16);
  const unsigned vrd = BYTES + (8 * hi + vrow) * RB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ pt_xv<D>(vrow)) * 16) + (lane & 1) * 8;
  const unsigned kwr = sr * RB + (((2 * part) ^ pt_xk<D>(sr & 31)) * 16), vwr = BYTES + sr * RB + (((2 * part + turn) ^ pt_xv<D>(sr)) * 16);
  uint4 kr[PCS], vr[PCS];
  unsigned kb = 127, vb = 127;
  auto issue = [&](int blk) {   // (a block of the window cur)
    bad_next = ~(unsigned)(cur.ok >> (blk % WB * NG)) & ((1u << NG) - 1);
    const int g = blk % WB * NG + wave;
    const unsigned long long at = pt_place(cur, g);
    const unsigned long long sc = ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(cur.scale >> 32), g) << 32) |
                                  (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)cur.scale, g);
    const char *k = (const char*)a.k_pages + at, *v = (const char*)a.v_pages + at;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      kr[i] = *(const uint4*)(k + (ko + i * 64));
      vr[i] = *(const uint4*)(v + (ko + i * 64));
    }
    kb = (a.k_scales + sc)[gr], vb = (a.v_scales + sc)[gr];
    __builtin_amdgcn_sched_barrier(0);
  };
  // page id of the lane's group in the window of an item's first block, and that block's loads
  auto first_id = [&](const PtItem& x) {
    return a.table[(long long)x.b * a.M + min(pt_page_of(a, x.b0 / WB * 64), (unsigned)a.M - 1)];
  };
  auto begin = [&](const PtItem& x, int id) {
    if (x.b0 >= x.b1) return;
    wi = x.b0 / WB;
    cur = pt_window<true>(a, x, wi * 64, id);
    pt_fetch(a, x, (wi + 1) * 64, ids);
    issue(x.b0);
  };
  int st = 0;   // LDS stage of the present block
  unsigned told = 0;
  // what was loaded, as 16 bits, to the other stage; zeros in the places that are closed to every row of the tile
  auto stage = [&](int blk, int pend) {   // returns whether a power is odd
    if (blk * PB + PB - 1 > pend || bad_next) {
      if (blk * PB + sr > pend || ((bad_next >> wave) & 1)) {
        kb = vb = 127;
#pragma unroll
        for (int i = 0; i < PCS; ++i) kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      }
    }
    if (__ballot(kb == 0 || vb == 0)) {   // (the conversion takes a byte of 0 as 2^-127)
#pragma unroll
      for (int i = 0; i < PCS; ++i) {
        if (kb == 0) kr[i] = make_uint4(pt_times_0(kr[i].x), pt_times_0(kr[i].y), pt_times_0(kr[i].z), pt_times_0(kr[i].w));
        if (vb == 0) vr[i] = make_uint4(pt_times_0(vr[i].x), pt_times_0(vr[i].y), pt_times_0(vr[i].z), pt_times_0(vr[i].w));
      }
    }
    const int odd = pt_odd(kb, pt_least_odd<DT>) | pt_odd(vb, pt_least_odd<DT>);
    float kp = __uint_as_float(kb << 23);
    const float vp = __uint_as_float(vb << 23);
    if constexpr (DT == HS_F16) {   // a group whose keys float16 does not hold exactly: its powers enter by the scores
      const bool after = __ballot(kb < pt_exact_from<DT>) != 0;
      if (after || (told >> st & 1)) {   // (told: of the stages that say so, bit 0 is of stage 1)
        PtPowers& to = kpw[st ^ 1];
        if (lane == 0) ((unsigned char*)&to.after)[wave] = after;
        if (after) kp = 1.f;
        if (part == 0) ((unsigned char*)to.k)[sr] = (unsigned char)kb;
        told = (told & (2u >> st)) | (unsigned)after << st;
      }
    }
    const unsigned kat = kwr + (st ^ 1) * 2 * BYTES, vat = vwr + (st ^ 1) * 2 * BYTES;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const uint4 k = kr[i], v = vr[i];
      *(uint4*)(lds + (kat ^ (i * 128))) = pt_widen<DT>(k.x, k.y, kp);
      *(uint4*)(lds + (kat ^ (i * 128 + 16))) = pt_widen<DT>(k.z, k.w, kp);
      *(uint4*)(lds + (vat ^ (i * 128))) = pt_widen<DT>(turn ? v.z : v.x, turn ? v.w : v.y, vp);
      *(uint4*)(lds + (vat ^ (i * 128 + 16))) = pt_widen<DT>(turn ? v.x : v.z, turn ? v.y : v.w, vp);
    }
    return odd;
  };
  auto last_pos = [&](const PtItem& x) {   // the tile's last row's position
    const int tlast = min(x.tile * PT_WIDE + PT_WIDE - 1, x.q.n * G - 1) / G;
    return (int)min((long long)x.q.kv - x.q.n + tlast, (long long)a.M * a.page_size - 1);
  };
  PtItem8 it = pt_item_wide8(a, t, me, range);
  PtWave<DT, D> w;
  int odd = 0;
  begin(it, first_id(it));
  w.queries(a, it, it.tile * PT_WIDE + wave * 32);
  if (it.b0 < it.b1) odd = stage(it.b0, last_pos(it));
  for (;;) {
    const int rows = it.q.n * G, tile0 = it.tile * PT_WIDE, row0 = tile0 + wave * 32;
    const int b0 = it.b0, b1 = it.b1, pend = last_pos(it);
    const bool last = range.done();
    int odd_next = 0;
    PtItem8 nx = it;
    int id = 0;
    if (!last) {
      nx = pt_item_wide8(a, t, me, range);
      id = first_id(nx);
    }
    const int pend_next = last_pos(nx);
    w.begin(a, it, row0);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) asm volatile("" ::"v"(w.qf[ks].x), "v"(w.qf[ks].y), "v"(w.qf[ks].z), "v"(w.qf[ks].w));
    // positions that every row of the wave has open, and that any has
    const int pmin = __builtin_amdgcn_readfirstlane(w.pos);
    const int pmax = row0 < rows ? __builtin_amdgcn_readlane(w.pos, 31) : -1;
    for (int blk = b0; blk < b1; ++blk) {
      const bool here = blk + 1 < b1;   // whether the next block is this item's
      bad = bad_next;
      __syncthreads();   // the block is in LDS, and every wave is done with the other stage
      st ^= 1;
      if (here) {
        if ((blk + 1) / WB != wi) {
          ++wi;
          cur = pt_window<true>(a, it, wi * 64, ids[lane]);
          pt_fetch(a, it, (wi + 1) * 64, ids);
        }
        issue(blk + 1);
      } else if (!last) {
        begin(nx, id);
      }
      const bool some = blk * PB <= pmax;   // wave-uniform
      const uint32_t groups = DT == HS_F16 ? kpw[st].after : 0;
      const unsigned kat = krd + st * 2 * BYTES, vat = vrd + st * 2 * BYTES;
      pt_f32x16 s[NB];
      if (some) w.template scores_of<NB>([&](int sb, int ks) { return *(const uint4*)(lds + (kat ^ (ks * 32)) + sb * 32 * RB); }, s);
      if constexpr (DT == HS_F16) {
        const unsigned after = __builtin_amdgcn_readfirstlane(groups);
        if (some && after)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if ((after >> (8 * g)) & 1)
#pragma unroll
              for (int i = 0; i < 2; ++i) pt_times_powers(s[g / 2], 8 * (g % 2) + 4 * i, kpw[st].k[g * 4 + 2 * i + hi]);
      }
      if (!here && !last) w.queries(a, nx, nx.tile * PT_WIDE + wave * 32);   // (this item's are done with)
      if (some) {
        if (!(blk * PB + PB - 1 <= pmin && bad == 0)) w.template mask<NB>(s, blk * PB, bad);
        w.template softmax<NB>(s);
        uint4 p[2 * NB];
        w.template pack<NB>(s, p);
        w.template outputs_of<NB>([&](int i) {
          const char* q = lds + i / TD * 16 * RB;
          const uint2 lo = pt_read_tr(q + (vat ^ (i % TD * 64))), up = pt_read_tr(q + 4 * RB + (vat ^ (i % TD * 64 + 32)));
          return make_uint4(lo.x, lo.y, up.x, up.y);
        }, p, s);
      }
      if (here || (!last && nx.b0 < nx.b1)) {
        const int more = stage(here ? blk + 1 : nx.b0, here ? pend : pend_next);
        odd |= here ? more : 0, odd_next |= here ? 0 : more;
      }
    }
    if (b0 >= b1 && !last) {   // (an item without blocks)
      begin(nx, id);
      w.queries(a, nx, nx.tile * PT_WIDE + wave * 32);
      if (nx.b0 < nx.b1) odd_next = stage(nx.b0, pend_next);
    }
    odd = __syncthreads_or(odd);
    const long long part = (long long)8 * a.grid_narrow * PT_NARROW + (long long)it.slot * PT_WIDE;   // (behind the narrow tiles')
    pt_tell(a, it, row0 + w.fr, rows, part + row0 + w.fr - tile0, 1);
    pt_end<DT, D>(a, it, w, tile0, row0, rows, b0 * PB, b1 * PB, part, odd);
    if (last) return;
    it = nx, odd = odd_next;
  }
}

// ------------------------------------------------------------------ kernels

// grid_wide = 0: sequences of any number of rows on narrow tiles (batches that are nearly all single tokens)
template <int DT, int D>
__device__ __forceinline__ void pt_attn_body(const PagedAttnArgs& a) {
  constexpr int ANY = 0x7fffffff, NPB = PtNarrow<DT, D>::PB;
  __shared__ __attribute__((aligned(1024))) char lds[65536];
  __shared__ float ml[4][2][32];
  __shared__ int ids[4][64];
  __shared__ PtList t;
  const int nw = a.grid_wide;
  int x;
  if ((int)blockIdx.x >= nw) {
    const int hi = nw ? PT_NARROW : ANY, w = blockIdx.x - nw;
    const int all = pt_build_narrow<NPB>(a, t, hi, &x), workers = pt_workers(all, gridDim.x - nw);
    if (w >= workers) return;
    const int end = pt_first(all, workers, w + 1);
    for (int at = pt_first(all, workers, w); at < end;) {
      PtItem it;
      at = pt_item_narrow<NPB>(a, t, w, at, end, hi, it);
      pt_narrow<DT, D>(a, it, lds, ml, ids);
    }
    return;
  }
  const int n = pt_build_wide<false>(a, t, &x);
  // XCD i (workgroups i, i + 8, ...) takes the items whose running cost falls into its eighth of the whole
  auto bound = [&](int i) {
    if (i >= 8) return n;
    const int at = (int)((long long)x * i / 8);
    const int b = pt_find(t.cost, a.B, at);
    const int c0 = b ? t.cost[b - 1] : 0, i0 = b ? t.items[b - 1] : 0;
    const int ci = t.cost[b] - c0, ii = t.items[b] - i0;
    return ci ? i0 + (int)((long long)(at - c0) * ii / ci) : i0;
  };
  const int xcd = blockIdx.x & 7, i0 = bound(xcd), i1 = bound(xcd + 1);
  for (int item = i0 + (blockIdx.x >> 3); item < i1; item += nw >> 3) pt_wide<DT, D>(a, pt_item_wide(a, t, item), lds, ids);
}

// Over pages of 8 bits: wide tiles' workgroups first, then the narrow ones', each wave of which takes blocks of its own.
template <int DT, int D>
__device__ __forceinline__ void pt_attn8_body(const PagedQuantAttnArgs& a) {
  constexpr int ANY = 0x7fffffff;
  __shared__ __attribute__((aligned(1024))) char lds[65536];
  __shared__ int ids[4][64];
  __shared__ uint32_t powers[4][64];
  __shared__ PtList8 t;
  __shared__ PtPowers kpw[2];
  const int nw = a.grid_wide;
  if ((int)blockIdx.x < nw) {
    pt_wide8<DT, D>(a, t, lds, ids, kpw);
    return;
  }
  const int hi = nw ? PT_NARROW : ANY, w = (blockIdx.x - nw) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all = pt_build_narrow8(a, t, hi), workers = pt_workers<PT_WAVE_LEAST>(all, (gridDim.x - nw) * 4);
  if (w >= workers) return;
  const int end = pt_first(all, workers, w + 1);
  for (int at = pt_first(all, workers, w); at < end;) {
    PtItem8 it;
    at = pt_item_narrow8(a, t, w, at, end, hi, all, workers, it);
    pt_narrow8<DT, D>(a, it, lds, ids, powers);
  }
}

// Adds S parts of one row to its maximum, sum and the lane's 4 dims (by a wave): part s lies `rel(s)` slots of R
// rows after row `first` of the parts. L and x are then the lane's own, to be summed over lanes (pt_gathered).
template <int D, int R, typename F>
__device__ __forceinline__ void pt_gather(const PagedAttnArgs& a, long long first, int S, F rel, float& M, float& L,
                                          float (&x)[4]) {
  // a load covers PER parts: lane (part, 4 dims); a batch is eight of them
  constexpr int LN = D / 4, PER = 64 / LN;
  const int lane = threadIdx.x & 63;
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1e-37f);
  const float* mls = a.part_ml + first * 2;
  const float* os = a.part_o + first * D;
  for (int s0 = 0; s0 < S; s0 += 64) {
    const int n = min(64, S - s0);
    const float2 ml = *(const float2*)(mls + rel(s0 + min(lane, n - 1)) * R * 2);
    float4 v[8];
    auto fetch = [&](int j) {   // (past the last part: it again, weighed 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (j + i * PER >= n) break;
        const int s = min(j + i * PER + lane / LN, n - 1);
        v[i] = *(const float4*)(os + rel(s0 + s) * R * D + (lane % LN) * 4);
      }
    };
    fetch(0);   // in flight with the statistics
    const float m = lane < n ? ml.x : -INFINITY, most = fmaxf(M, wave_max(m));
    const float old = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - most) * c);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - most) * c);
    M = most;
    L = L * old + (lane < n ? f * ml.y : 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= old;
    for (int j = 0; j < n; j += 8 * PER) {
      if (j) fetch(j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (j + i * PER >= n) break;
        const int k = j + i * PER + lane / LN;
        const float fs = __shfl(f, min(k, n - 1), 64), g = k < n ? fs : 0.f;
        x[0] += g * v[i].x, x[1] += g * v[i].y, x[2] += g * v[i].z, x[3] += g * v[i].w;
      }
    }
  }
}
// sums over the lanes of a wave: L, and x of the lanes that hold the same dims
template <int D>
__device__ __forceinline__ void pt_gathered(float& L, float (&x)[4]) {
  L = wave_sum(L);
#pragma unroll
  for (int o = D / 4; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o, 64);
}
template <int DT, int D>
__device__ __forceinline__ void pt_put(uint16_t* out, float L, const float (&x)[4]) {
  const int lane = threadIdx.x & 63;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (lane < D / 4) *(uint2*)(out + lane * 4) = make_uint2(gm_pack2<DT>(x[0] * inv, x[1] * inv), gm_pack2<DT>(x[2] * inv, x[3] * inv));
}
// Joins S parts of one row (by a wave).
template <int DT, int D, int R, typename F>
__device__ __forceinline__ void pt_join(const PagedAttnArgs& a, long long first, int S, F rel, uint16_t* out) {
  float M = -INFINITY, L = 0.f, x[4] = {};
  pt_gather<D, R>(a, first, S, rel, M, L, x);
  pt_gathered<D>(L, x);
  pt_put<DT, D>(out, L, x);
}
// k_paged_combine: joins the parts of split tiles, a wave per row and head, and zeroes the rows of no sequence.
// (A part without open positions has maximum -inf and outputs of zero.)
template <int DT, int D>
__device__ __forceinline__ void pt_combine_body(const PagedAttnArgs& a) {
  constexpr int ANY = 0x7fffffff, NPB = PtNarrow<DT, D>::PB;
  __shared__ PtList t;
  __shared__ int start[PT_MAXB + 1], kv[PT_MAXB];   // (a row looks its sequence up in LDS: from memory it is 1 us)
  for (int b = threadIdx.x; b <= a.B; b += 256) {
    start[b] = a.q_start[b];
    if (b < a.B) kv[b] = a.kv_len[b];
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.H / a.KVH, waves = gridDim.x * 4, me = blockIdx.x * 4 + wave, hi = a.grid_wide ? PT_NARROW : ANY;
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  // Each wave takes a run of rows and looks up where they lie only where a sequence, head or tile begins: looked up
  // row by row (binary search, divisions) a batch of 7,100 rows takes 18 us rather than 15.
  auto runs = [&](int rows, auto seq, auto tile, auto join) {
    const int per = (rows + waves - 1) / waves, end = min(rows, (me + 1) * per);
    for (int u = me * per; u < end;) {
      const int b = uniform(pt_find(t.cost, a.B, u));
      const int s0 = uniform(start[b]), i = u - (b ? uniform(t.cost[b - 1]) : 0);
      const PtSeq q = seq(b, s0, uniform(start[b + 1]), uniform(kv[b]));
      const int of = q.n * G, stop = min(end, u - i + of * a.KVH);   // (rows of the sequence, per head)
      int h = i / of, row = i - h * of;
      bool fresh = true;
      for (; u < stop; ++u, ++row) {
        if (row == of) row = 0, ++h, fresh = true;
        if (fresh || tile(row)) join(b, q, h, row, true);
        else join(b, q, h, row, false);
        fresh = false;
      }
    }
  };
  auto out = [&](const PtSeq& q, int h, int row) {
    const int tk = row / G;
    return (uint16_t*)a.out + ((long long)(q.start + tk) * a.H + h * G + row - tk * G) * D;
  };
  int rows;
  const int all = pt_build_narrow<NPB>(a, t, hi, &rows), workers = pt_workers(all, a.grid_narrow);
  int w0 = 0, w1 = 0;   // workgroups that hold the tile's first and last block
  runs(
      uniform(rows), [&](int b, int s0, int s1, int kv) { return pt_seq<PT_NARROW, NPB>(a, b, s0, s1, kv, 0, hi); },
      [](int row) { return row % PT_NARROW == 0; },
      [&](int b, const PtSeq& q, int h, int row, bool fresh) {
        if (fresh) {
          const int g0 = (b ? uniform(t.items[b - 1]) : 0) + (h * q.tiles + row / PT_NARROW) * q.blocks;
          w0 = uniform((int)((((long long)g0 + 1) * workers - 1) / all));
          w1 = uniform((int)((((long long)g0 + q.blocks) * workers - 1) / all));
        }
        if (w0 != w1)
          pt_join<DT, D, PT_NARROW>(a, (long long)2 * w0 * PT_NARROW + row % PT_NARROW, w1 - w0 + 1,
                                    [](int s) { return 2 * s + (s == 0); }, out(q, h, row));
      });
  if (a.grid_wide) {
    __syncthreads();
    pt_build_wide<true>(a, t, &rows);
    const int share = uniform(t.share);
    runs(
        uniform(rows), [&](int b, int s0, int s1, int kv) { return pt_seq<PT_WIDE, 64>(a, b, s0, s1, kv, PT_NARROW, ANY); },
        [](int) { return false; },
        [&](int b, const PtSeq& q, int h, int row, bool) {
          const int S = pt_splits(q, share), slot = (b ? uniform(t.slots[b - 1]) : 0) + (h * q.tiles + row / PT_WIDE) * S;
          pt_join<DT, D, PT_WIDE>(a, (long long)(2 * a.grid_narrow * PT_NARROW) + (long long)slot * PT_WIDE + row % PT_WIDE, S,
                                  [](int s) { return s; }, out(q, h, row));
        });
  }
  int down = 0;   // (no batch: every row)
  for (int b = lane; b < a.B; b += 64) down |= start[b + 1] < start[b];
  const bool none = __ballot(down) != 0;
  const int s0 = none ? 0 : start[0], s1 = none ? 0 : start[a.B];
  for (int row = me; row < a.N; row += waves) {
    if (row >= s0 && row < s1) continue;
    uint4* o = (uint4*)((uint16_t*)a.out + (long long)row * a.H * D);
    for (int i = lane; i < a.H * D / 8; i += 64) o[i] = make_uint4(0, 0, 0, 0);
  }
}

// k_paged_quant_combine: the same over pages of 8 bits. What a row is joined of stands in a.joins, where the wave (workgroup)
// that began its tile has put it, so nothing is looked up here. Rows are D / 4 lanes each, so a wave has the loads of several
// rows in flight at once. _join, for few rows: a workgroup of 16 waves joins a row, which over long caches has hundreds of
// parts (4 requests over up to 131,071 positions: 6.6 us, 8.9 by 4 waves). Bound by the latency of dependent loads: 4 to 5 us
// for decodes, 9 for 1,553 rows of 14 heads of 64, 11 for 5,963 rows of 32 heads of 128.
template <int DT, int D, bool JOIN>
__device__ __forceinline__ void pt_combine8_body(const PagedQuantAttnArgs& a) {
  constexpr int LN = D / 4, PER = 64 / LN, W = JOIN ? 16 : 1;
  __shared__ float shares[W][4][LN + 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LN;
  const int s0 = a.q_start[0], s1 = a.q_start[a.B], rows = a.N * a.H;
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1e-37f);
  const bool none = pg_descends(a.q_start, a.B, lane);   // no batch: every row is zero
  auto far = [&](const int2 j, int s) { return s ? (2 * s - 1) * (j.y & 1 ? PT_WIDE : PT_NARROW) : 0; };   // rows from the first part's
  auto zero = [&](int u) {
    const int row = u / a.H;
    return none || row < s0 || row >= s1;
  };
  uint16_t* out = (uint16_t*)a.out;
  if constexpr (JOIN) {
    for (int u = blockIdx.x; u < rows; u += gridDim.x) {
      if (zero(u)) {
        if (threadIdx.x < D / 4) *(uint2*)(out + (long long)u * D + threadIdx.x * 4) = make_uint2(0, 0);
        continue;
      }
      const int2 j = ((const int2*)a.joins)[u];
      const int S = j.y >> 1;
      if (S < 2) continue;
      float M = -INFINITY, L = 0.f, x[4] = {};
      const int from = S * wave / W;
      pt_gather<D, 1>(a, j.x, S * (wave + 1) / W - from, [&](int s) { return far(j, from + s); }, M, L, x);
      pt_gathered<D>(L, x);
      if (lane < LN)
#pragma unroll
        for (int e = 0; e < 4; ++e) shares[wave][e][lane] = x[e];
      if (lane == 0) shares[wave][0][LN] = M, shares[wave][0][LN + 1] = L;
      __syncthreads();
      if (wave == 0) {
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; ++i) most = fmaxf(most, shares[i][0][LN]);
        L = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float m = shares[i][0][LN], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - most) * c);
          L += f * shares[i][0][LN + 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] += f * shares[i][e][sub];
        }
        pt_put<DT, D>(out + (long long)u * D, L, x);
      }
      __syncthreads();
    }
    return;
  }
  // a wave's run of rows, 64 at a time: a lane each looks whether there is something to do
  const int waves = gridDim.x * 4, each = (rows + waves - 1) / waves, me = blockIdx.x * 4 + wave, stop = min(rows, (me + 1) * each);
  for (int u0 = me * each; u0 < stop; u0 += 64) {
    const int mine = u0 + lane;
    int2 jm = make_int2(0, 0);
    bool blank = false;
    if (mine < stop) {
      jm = ((const int2*)a.joins)[mine];
      blank = zero(mine);
    }
    unsigned long long todo = __ballot(mine < stop && (blank || jm.y >= 4));
    while (todo) {
      // the wave's lane groups take the next PER of them
      int k = -1;
#pragma unroll
      for (int g = 0; g < PER; ++g) {
        const int first = todo ? __ffsll(todo) - 1 : -1;
        if (first >= 0) todo &= todo - 1;
        if (lane / LN == g) k = first;
      }
      const int2 j = make_int2(__shfl(jm.x, max(k, 0), 64), __shfl(jm.y, max(k, 0), 64));
      const bool empty = __shfl((int)blank, max(k, 0), 64);
      if (k < 0) continue;
      uint2* to = (uint2*)(out + (long long)(u0 + k) * D) + sub;
      if (empty) {
        *to = make_uint2(0, 0);
        continue;
      }
      const int S = j.y >> 1;
      const float2* mls = (const float2*)a.part_ml + j.x;
      const float4* os = (const float4*)(a.part_o + (long long)j.x * D) + sub;
      float M = -INFINITY, L = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = 0; p < S; p += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p + i < S) {
            const long long at = far(j, p + i);
            ml[i] = mls[at];
            v[i] = os[at * LN];
          }
        float most = M;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p + i < S) most = fmaxf(most, ml[i].x);
        const float old = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - most) * c);
        M = most, L *= old, x.x *= old, x.y *= old, x.z *= old, x.w *= old;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p + i < S) {
            const float f = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i].x - most) * c);
            L = fmaf(f, ml[i].y, L);
            x.x = fmaf(f, v[i].x, x.x), x.y = fmaf(f, v[i].y, x.y), x.z = fmaf(f, v[i].z, x.z), x.w = fmaf(f, v[i].w, x.w);
          }
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      *to = make_uint2(gm_pack2<DT>(x.x * inv, x.y * inv), gm_pack2<DT>(x.z * inv, x.w * inv));
    }
  }
}

#define PT_KERNELS(NAME, DT, D)                                                                                                  \
  extern "C" __global__ void __launch_bounds__(256, 2) k_paged_attn_##NAME(const PagedAttnArgs a) { pt_attn_body<DT, D>(a); }     \
  extern "C" __global__ void __launch_bounds__(256) k_paged_combine_##NAME(const PagedAttnArgs a) { pt_combine_body<DT, D>(a); }  \
  extern "C" __global__ void __launch_bounds__(256, 2) k_paged_quant_attn_##NAME(const PagedQuantAttnArgs a) { pt_attn8_body<DT, D>(a); } \
  extern "C" __global__ void __launch_bounds__(256) k_paged_quant_combine_##NAME(const PagedQuantAttnArgs a) { pt_combine8_body<DT, D, false>(a); } \
  extern "C" __global__ void __launch_bounds__(1024) k_paged_quant_join_##NAME(const PagedQuantAttnArgs a) { pt_combine8_body<DT, D, true>(a); }
PT_KERNELS(bf16_d128, HS_BF16, 128)
PT_KERNELS(bf16_d64, HS_BF16, 64)
PT_KERNELS(f16_d128, HS_F16, 128)
PT_KERNELS(f16_d64, HS_F16, 64)
