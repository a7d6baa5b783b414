// Paged K/V caches: append with rotation, and causal attention of packed rows over the pages.
//
// Rows of the packed new tokens belong to sequences (q_start), sequences hold kv_len positions, position p of
// sequence b lies in row p % page_size of page table[b][p / page_size]. The metadata lies on the device and is
// taken as it comes: whatever it holds, no kernel here reads or writes outside its tensors (a row of no
// sequence is padding; a position before 0, past the table or in a page outside the pool has no place).
#include "common.h"

// Sequence of row `row` (B for none), by one wave: the number of q_start[1 ..] that are <= row.
__device__ __forceinline__ int pg_sequence(const int* q_start, int B, int row, int lane) {
  int n = 0;
  for (int i = 0; i < B; i += 64) n += __popcll(__ballot(i + lane < B && q_start[1 + min(i + lane, B - 1)] <= row));
  return n;
}

// Page of position pos of sequence b, or -1 where it has no place.
__device__ __forceinline__ int pg_page(const int* table, int b, int M, int page_size, long long pages, int pos) {
  if (pos < 0 || pos / page_size >= M) return -1;
  const int page = table[(long long)b * M + pos / page_size];
  return page >= 0 && page < pages ? page : -1;
}

// ------------------------------------------------------------------ append
//
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
    const int pos = real ? a.kv_len[min(b, a.B - 1)] - a.q_start[b + 1] + row : 0;
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

// ------------------------------------------------------------------ attention
//
// k_paged_attn_any: one wave per (row, query head), 64 positions a step: a lane scores one position (its key's row
// against q in LDS), the wave takes maximum and sum, then every lane adds its dims of 64 values. Any type, page size
// and head size up to 256; fp32 throughout. Closed positions are never loaded, so what lies there (NaN) does not enter.
#define PG_ANY_D 256
extern "C" __global__ void __launch_bounds__(64) k_paged_attn_any(const PagedAttnArgs a) {
  __shared__ float q[PG_ANY_D], p[64];
  __shared__ int at[64];   // page of each of the step's positions, -1: closed
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / (a.H / a.KVH);
  const int b = pg_sequence(a.q_start, a.B, row, lane);
  const bool real = b < a.B && row >= a.q_start[0];
  const int pos = real ? a.kv_len[b] - a.q_start[b + 1] + row : -1;
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
      for (int d = 0; d < a.D; ++d) s = fmaf(q[d], ld_f(a.k_pages, ko + d, a.dtype), s);
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
        x = fmaf(p[j], ld_f(a.v_pages, vo + i * 64 + lane, a.dtype), x);
      }
      o[i] = x;
    }
  }
#pragma unroll
  for (int i = 0; i < PG_ANY_D / 64; ++i)
    if (i * 64 + lane < a.D)
      st_f(a.out, ((long long)row * a.H + h) * a.D + i * 64 + lane, a.dtype, l == 0.f ? 0.f : o[i] / l);
}
