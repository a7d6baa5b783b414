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
__device__ __forceinline__ int pt_workers(int all, int most) {
  return max(1, min(most, (all + PT_NARROW_LEAST - 1) / PT_NARROW_LEAST));
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

  __device__ __forceinline__ void init(const PagedAttnArgs& a, const PtItem& it, int row0) {
    lane = threadIdx.x & 63, fr = lane & 31, hi = lane >> 5;
    const int G = a.H / a.KVH, rows = it.q.n * G, r = min(row0 + fr, rows - 1), t = r / G;
    pos = it.q.kv - it.q.n + t;
    const long long last = (long long)a.M * a.page_size - 1;
    pos = pos > last ? (int)last : pos;
    const uint16_t* p = (const uint16_t*)a.q + (long long)(it.q.start + t) * a.q_rs + (long long)(it.h * G + r - t * G) * a.q_hs;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;   // a negative scale: of -q
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint4 v = *(const uint4*)(p + ks * 16 + hi * 8);
      qf[ks] = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
    }
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
    constexpr int KS = D / 16;
    uint4 k[KS];
    auto read = [&](int sb, int ks) { return *(const uint4*)(Kt + (sb * 32 + fr) * RB + (((2 * ks + hi) ^ pt_xk<D>(fr)) * 16)); };
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
    constexpr int N = 2 * NB * TD, EL = NB * 16 / N;
    auto read = [&](int i) { return vfrag(Vt, i / TD / 2, i / TD % 2, i % TD); };
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
struct PtWindow {
  uint32_t lo, hi;
  unsigned long long ok;
};
__device__ __forceinline__ unsigned pt_page_of(const PagedAttnArgs& a, int group) {   // may lie past the table
  const unsigned grp = (unsigned)group + (threadIdx.x & 63);
  return a.group_magic ? __umulhi(grp, a.group_magic) : grp;
}
__device__ __forceinline__ PtWindow pt_window(const PagedAttnArgs& a, const PtItem& it, int group, int id) {
  PtWindow w;
  const unsigned grp = (unsigned)group + (threadIdx.x & 63), at = pt_page_of(a, group);
  const bool ok = at < (unsigned)a.M && (unsigned long long)(long long)id < (unsigned long long)a.pages;
  const unsigned long long off = 2ull * ((ok ? id : 0) * a.page_stride + it.h * a.head_stride +
                                         (ok ? (long long)((grp - at * a.page_groups) * 16) * a.row_stride : 0));
  w.lo = (uint32_t)off, w.hi = (uint32_t)(off >> 32);
  w.ok = __ballot(ok);
  return w;
}
__device__ __forceinline__ PtWindow pt_window(const PagedAttnArgs& a, const PtItem& it, int group) {
  return pt_window(a, it, group, a.table[(long long)it.b * a.M + min(pt_page_of(a, group), (unsigned)a.M - 1)]);
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
__device__ __forceinline__ unsigned long long pt_place(const PtWindow& w, int i) {
  return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane(w.hi, i) << 32) | (uint32_t)__builtin_amdgcn_readlane(w.lo, i);
}

// One 1 KiB load of a group to LDS: rows i * (1024 / RB) .. of its 16, swizzled
template <int D, bool V>
__device__ __forceinline__ void pt_load(const char* group, unsigned row_bytes, int i, unsigned lds, int lane) {
  constexpr int RB = 2 * D, PER = 1024 / RB, SL = RB / 16;   // rows per load, slots of a row
  const int r = i * PER + lane / SL, ch = (lane % SL) ^ (V ? pt_xv<D>(r) : pt_xk<D>(r));
  gm_dma16s(group, (unsigned)r * row_bytes + ch * 16, lds);
}

// One row over positions p0 .. p1 - 1 by a wave, 64 at a time, reading open positions only: the row's maximum of the raw
// scores, sum of exponentials and the lane's outputs (dims lane * E ..), times 2^pt_up as the tiles' (they may be joined
// with them). For tiles whose product is not finite.
template <int DT, int D>
__device__ __forceinline__ void pt_row(const PagedAttnArgs& a, const PtItem& it, int row, int p0, int p1, float& m,
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
    float s = 0.f;
    if (page >= 0)
#pragma unroll 1
      for (int d = 0; d < D; ++d) s = fmaf(gm_ld<DT>(q, d), gm_ld<DT>(a.k_pages, at + d), s);
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
      const float ej = __shfl(e, j, 64);
      if (__shfl(page, j, 64) < 0) continue;
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = fmaf(ej, gm_ld<DT>(a.v_pages, aj + lane * E + i), x[i]);
    }
  }
}

// rows r0, r0 + step, ... of a tile one by one, written as the tile's rows are (part: index of its first partial row)
template <int DT, int D>
__device__ __forceinline__ void pt_rows(const PagedAttnArgs& a, const PtItem& it, int tile0, int r0, int r1, int step, int p0,
                                     int p1, long long part) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, G = a.H / a.KVH;
#pragma unroll 1
  for (int row = r0; row < r1; row += step) {
    float m, l, x[E];
    pt_row<DT, D>(a, it, row, p0, p1, m, l, x);
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

template <int DT, int D>
struct PtNarrow {
  static constexpr int PB = 8192 / (2 * D), NB = PB / 32, NG = PB / 16;   // positions of a block: 8 KiB of K, 8 of V
  static constexpr int LPG = 2 * D * 16 / 1024;                             // loads per group
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

// Joins S parts of one row (by a wave): part s lies `rel(s)` slots of R rows after row `first` of the parts.
template <int DT, int D, int R, typename F>
__device__ __forceinline__ void pt_join(const PagedAttnArgs& a, long long first, int S, F rel, uint16_t* out) {
  // a load covers PER parts: lane (part, 4 dims); a batch is eight of them
  constexpr int LN = D / 4, PER = 64 / LN;
  const int lane = threadIdx.x & 63;
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1e-37f);
  const float* mls = a.part_ml + first * 2;
  const float* os = a.part_o + first * D;
  float M = -INFINITY, L = 0.f, x[4] = {};
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
  L = wave_sum(L);
#pragma unroll
  for (int o = LN; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o, 64);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (lane < LN) *(uint2*)(out + lane * 4) = make_uint2(gm_pack2<DT>(x[0] * inv, x[1] * inv), gm_pack2<DT>(x[2] * inv, x[3] * inv));
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

#define PT_KERNELS(NAME, DT, D)                                                                                                  \
  extern "C" __global__ void __launch_bounds__(256, 2) k_paged_attn_##NAME(const PagedAttnArgs a) { pt_attn_body<DT, D>(a); }     \
  extern "C" __global__ void __launch_bounds__(256) k_paged_combine_##NAME(const PagedAttnArgs a) { pt_combine_body<DT, D>(a); }
PT_KERNELS(bf16_d128, HS_BF16, 128)
PT_KERNELS(bf16_d64, HS_BF16, 64)
PT_KERNELS(f16_d128, HS_F16, 128)
PT_KERNELS(f16_d64, HS_F16, 64)
