// What the kernels that split the keys share (attn_split.hip, attn_prefix_unit.hip): parameters, scores of a part, and what a part leaves of a row.
#pragma once
#include <math.h>

#include "entmax_rows_kernel.h"

namespace adsp {
namespace split {
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxChunk = 2048;  // keys of a workgroup: 32 scores a lane when a wave holds a row
constexpr int kMaxRows = 64;     // rows of a K/V head
constexpr int kWaves = 4;        // of a part's workgroup
constexpr int kListCap = 2048;   // keys above the bound that the second kernel's list holds: a quarter for each of its waves

struct Entry {
  float z;
  int key;
};
// What a workgroup of the first kernel leaves of a row: its largest score, a lower bound of the row's threshold, the number of keys above it.  Thresholds are
// solved relative to the row's maximum and weights divided by their sum: a threshold at the size of the scores would be off by half a step of that size for
// all members alike, which adds up over them (alpha = 2, scores around 64, 3000 members: 8e-3 of the weights' sum).  For a backward the row's maximum is left in its first part.
struct Part {
  float max, bound;
  int count;
};

struct SplitParams {
  const void *q, *k, *v;
  void* out;
  float* taus;     // [B * Hkv * R], or null: thresholds of the rows less their maxima, for a backward, which also takes the parts and entries
  Part* parts;     // [B * Hkv * R][splits]
  Entry* entries;  // [B * Hkv * R][splits][chunk]
  const int* tables;  // [B][table_stride] pages of a sequence, or null: k and v are [B, Hkv, N, D]
  long long table_stride;
  const void *lens, *lens_q;
  int lens_bits, lens_q_bits;
  long long k_s0, k_sh, k_sn, v_s0, v_sh, v_sn;  // strides in elements: page (or batch item), head, key
  int units, Hkv, R, Nq, N;  // units: heads of K and V of all sequences
  int pages, page, page_shift;  // page_shift: log2(page), or -1
  int splits, chunk;
  // keys [0, prefix) lie in the pages of this table for every request whose own table starts with them: parts [0, prefix_parts); the parts behind them start at key `prefix`
  const int* prefix_table;
  int prefix, prefix_parts, B;
  RowsParams rows;  // (the solver's constants; scale: (alpha - 1) / sqrt(D))
};
// Parts of a row with `len` keys.
__device__ __forceinline__ int parts_of(const SplitParams& p, int len) {
  return len <= p.prefix ? (len + p.chunk - 1) / p.chunk : p.prefix_parts + (len - p.prefix + p.chunk - 1) / p.chunk;
}

__device__ __forceinline__ int length_at(const void* lens, int bits, int b, int most) {
  if (!lens) return most;
  const long long l = bits == 64 ? ((const long long*)lens)[b] : (long long)((const int*)lens)[b];
  return (int)(l < 0 ? 0 : (l > most ? most : l));
}
__device__ __forceinline__ int page_of(const SplitParams& p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page; }
// The page that a table names, or -1: an entry outside the cache is a page without keys.
__device__ __forceinline__ int table_entry(const SplitParams& p, int b, int i) {
  const int id = p.tables[(long long)b * p.table_stride + i];
  return (unsigned)id < (unsigned)p.pages ? id : -1;
}

// Rows of both matrices multiplied: kSteps pieces of 16 bytes a lane.  Single precision: four sums, of every fourth product each, added up at the end.  One sum of D products in turn has
// roundings of its own size D times (against 64 bits, 8 x 16/8 heads, 2386 tokens, D = 128: outputs off by 1.4e-6 with one sum, 6e-7 with four, in the same time).
template <typename T, int kSteps> __device__ __forceinline__ f32x4 rows_product(const u32x4 (&a)[kSteps], const u32x4 (&b)[kSteps]) {
  if constexpr (elem_traits<T>::kVec == 4) {
    f32x4 part[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) part[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = a[s][e], y = b[s][e];
        part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y), part[e], 0, 0, 0);
      }
    return (part[0] + part[1]) + (part[2] + part[3]);
  } else {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (elem_traits<T>::kIsBf16) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[s]), __builtin_bit_cast(bf16x8, b[s]), c, 0, 0, 0);
      else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[s]), __builtin_bit_cast(f16x8, b[s]), c, 0, 0, 0);
    }
    return c;
  }
}

// A row's scores in a wave's registers: lane l holds keys 256 i + 4 l .. + 3.
struct HeldRow {
  f32x4 z[kMaxChunk / 256];
  int n;  // keys
  __device__ __forceinline__ void less(float m) {
#pragma unroll
    for (int i = 0; i < kMaxChunk / 256; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[i][e] -= m;
  }
  template <typename F> __device__ __forceinline__ void for_each(F f) const {
#pragma unroll
    for (int i = 0; i < kMaxChunk / 256; ++i)
      if (i * 256 < n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f(z[i][e]);
      }
  }
};

constexpr int score_stride(int chunk) { return chunk + 4; }  // (16 rows at one key: 16 different groups of banks)
inline size_t scores_lds(int R, int chunk, int page, bool paged) {
  return ((size_t)R * score_stride(chunk) + (paged ? chunk / page + 2 : 0)) * 4;
}

// The scores of keys [key0, key0 + n) of a head, all rows, into LDS: z[row][key - key0], -inf from n up to the next multiple of 64 and in
// pages that are none.  `pages`: LDS for the chunk's part of the block table.
// Operand layout: lane l holds row l % 16 of its matrix, the 16-byte piece l / 16 of every 64 bytes; of the result row (of the
// queries) l % 16 and keys 4 (l / 16) + 0 .. 3.
template <typename T, int D, bool kPaged, int W>
__device__ __forceinline__ void chunk_scores(const SplitParams& p, int b, int kvh, int key0, int n, float* z, const int* pages, int wave, int lane) {
  constexpr int kSteps = D * elem_traits<T>::kBytes / 64, kB = elem_traits<T>::kBytes;
  const int r = lane & 15, g = lane >> 4, zs = score_stride(p.chunk);
  const int first_page = kPaged ? page_of(p, key0) : 0;
  const char* const kbase = (const char*)p.k + ((kPaged ? 0 : b * p.k_s0) + kvh * p.k_sh) * kB;
  const char* const qbase = (const char*)p.q + (size_t)(b * p.Hkv + kvh) * p.R * D * kB;
  u32x4 qf[kSteps];
  auto load_q = [&](int row0) {
    const int row = row0 + r < p.R ? row0 + r : p.R - 1;
    const u32x4* src = reinterpret_cast<const u32x4*>(qbase + (size_t)row * D * kB) + g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = src[s * 4];
  };
  load_q(0);
  for (int k0 = wave * 64; k0 < n; k0 += W * 64) {
    u32x4 kf[4][kSteps];
    int there = 0;  // of the lane's four keys, those in a page
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = k0 + j * 16 + r, key = key0 + (at < n ? at : n - 1);
      long long off;
      if constexpr (kPaged) {
        const int pg = page_of(p, key), id = pages[pg - first_page];
        there |= (id >= 0 ? 1 : 0) << j;
        off = (id >= 0 ? id : 0) * p.k_s0 + (key - pg * p.page) * p.k_sn;
      } else {
        off = key * p.k_sn;
      }
      const u32x4* src = reinterpret_cast<const u32x4*>(kbase + off * kB) + g;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kf[j][s] = src[s * 4];
    }
    for (int row0 = 0; row0 < p.R; row0 += 16) {
      if (row0 > 0 || p.R > 16) load_q(row0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 acc = rows_product<T>(kf[j], qf);
        const int at = k0 + j * 16 + g * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bool see = at + i < n;
          if constexpr (kPaged) see = see && (__shfl(there, g * 4 + i, 64) >> j & 1);
          acc[i] = see ? acc[i] * p.rows.scale : -INFINITY;
        }
        if (row0 + r < p.R) *reinterpret_cast<f32x4*>(z + (row0 + r) * zs + at) = acc;
      }
    }
  }
}

// A lower bound of the threshold that a step of Newton's method gives from another, on (sum u^c0)^(1/c0) - 1, which is convex and falls: a step from below does
// not pass the root.  a0 = sum u^c0, a1 = sum u^(c0 - 1); less some roundings of the sums.
template <int AM> __device__ __forceinline__ float newton_step(float a0, float a1, const RowsParams& rows) {
  float step;
  if constexpr (AM == AM_2) step = a0 - 1.f;
  else if constexpr (AM == AM_15) step = a0 - __builtin_amdgcn_sqrtf(a0);
  else step = a0 - fast_exp2(fast_log2(a0) * (1.f - rows.inv_c0));
  return a1 > 0.f ? step * fast_rcp(a1) : 0.f;
}
template <int AM> __device__ __forceinline__ float raised(float t, float a0, float a1, const RowsParams& rows) {
  const float to = t + newton_step<AM>(a0, a1, rows);
  return fmaxf(t, to - 2e-6f * fmaxf(fabsf(to), 1.f));
}

// Two sums over a wave at once: each half of it adds up one of them.
__device__ __forceinline__ void wave_sums(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  float x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  x += dpp_move<0x111, 0xf>(0.f, x);
  x += dpp_move<0x112, 0xf>(0.f, x);
  x += dpp_move<0x114, 0xf>(0.f, x);
  x += dpp_move<0x118, 0xf>(0.f, x);
  x += dpp_move<0x142, 0xa>(0.f, x);  // (lane 15 of a half's first row into its second)
  a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 31));
  b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
// The threshold, from a lower bound `t` of it, as solve_row finds it from the maximum less 1.
template <int AM, bool kBlock, typename Row> __device__ __forceinline__ float solve_from(const Row& row, float t, const RowsParams& rows, float* sm) {
  for (int it = 0; it < 64; ++it) {
    float a[2] = {0.f, 0.f};
    row.for_each([&](float z) { accum_stats<AM>(z - t, rows.c0, a); });
    if constexpr (kBlock) row_sum<256, 2>(a, sm);
    else wave_sums(a[0], a[1]);
    const float step = newton_step<AM>(a[0], a[1], rows);
    t += step;
    if (fabsf(a[0] - 1.f) <= 2e-6f || !(fabsf(step) > 1.2e-7f * fabsf(t))) break;
  }
  return t;
}

__device__ __forceinline__ float hold_row(HeldRow& held, const float* z, int n, int lane) {
  const int n64 = (n + 63) & ~63;
  float m = -INFINITY;
  held.n = n;
#pragma unroll
  for (int i = 0; i < kMaxChunk / 256; ++i) {
    const int at = i * 256 + lane * 4;
    held.z[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (at < n64) held.z[i] = *reinterpret_cast<const f32x4*>(z + at);
    m = fmaxf(m, fmaxf(fmaxf(held.z[i][0], held.z[i][1]), fmaxf(held.z[i][2], held.z[i][3])));
  }
  return wave_max(m);
}

// What a wave leaves of a row's scores of keys [key0, key0 + n), in LDS: a lower bound of the row's threshold and the keys above it, as part `at`.
template <int AM> __device__ __forceinline__ void leave_part(const SplitParams& p, const float* z, int n, int key0, size_t at, int lane) {
  HeldRow held;
  const float m = hold_row(held, z, n, lane);
  if (!(m > -INFINITY)) {
    if (lane == 0) p.parts[at] = Part{-INFINITY, -INFINITY, 0};
    return;
  }
  // below the maximum less 1 by some roundings; a score of +inf: the bound lies there, above which no key of the row lies, and the row is 0
  float t = m < INFINITY ? m - 1.f - 2e-6f * fmaxf(fabsf(m), 1.f) : m;
  // (of a few keys that leaves few enough)
  for (int it = 0; it < (n <= 256 ? 0 : 4); ++it) {
    float a[2] = {0.f, 0.f};
    held.for_each([&](float x) { accum_stats<AM>(x - t, p.rows.c0, a); });
    wave_sums(a[0], a[1]);
    t = raised<AM>(t, a[0], a[1], p.rows);
  }
  Entry* const list = p.entries + at * p.chunk;
  int count = 0;
  held.for_each([&](float x) { count += x > t ? 1 : 0; });
  const int upto = wave_prefix_sum(count);
  int w = upto - count;
#pragma unroll
  for (int i = 0; i < kMaxChunk / 256; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = held.z[i][e];
      if (x > t) list[w++] = Entry{x, key0 + i * 256 + lane * 4 + e};
    }
  if (lane == 63) p.parts[at] = Part{m, t, upto};
}

// A prefix that requests have in common (attn_prefix_unit.hip): the keys of a wave, which holds them in 64 registers a lane; a part has those of two, four or eight waves, and 64 at least.
constexpr int wave_keys(int row_bytes) { return row_bytes <= 256 ? 64 : (row_bytes == 512 ? 32 : 16); }
// Tiles of sixteen rows of a workgroup: all, up to 64 rows (32 where they are long), but two workgroups to a CU where there are rows to share out.
inline int prefix_row_tiles(long long tiles, long long parts, int row_bytes) {
  int row_tiles = row_bytes <= 512 ? 4 : 2;
  while (row_tiles > 1 && parts * ((tiles + row_tiles - 1) / row_tiles) < 512) row_tiles /= 2;
  return row_tiles > tiles ? (int)tiles : row_tiles;
}
constexpr int kFewRows = 16;  // up to so many there is a kernel of its own
// The first kernel of such a call, for one element type; am: AM_GEN, AM_15 or AM_2.
template <typename T> void prefix_scores_launch(const SplitParams& p, int D, int am, hipStream_t s);
}  // namespace split
}  // namespace adsp
