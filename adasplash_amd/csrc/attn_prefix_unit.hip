// One translation unit per element type (-DADSP_T=...): the first kernel of paged attention where many requests' tables start with the same pages.
//
// A workgroup takes 16 rows (queries of whatever requests) and a part of the prefix: K comes from memory once for all of them, and from L2 once for every 16 rows.  Rows whose
// request does not have these pages, or ends inside the part, are left to other workgroups, which look at the tables in the same way and do a part of the prefix for one request only
// where it was left: the prefix table says what is worth sharing, and no more.
//
// What bounds it: vector instructions, some twelve for each score (with 64 requests a key of the prefix meets 256 rows of each head of K, and comes from memory once).  So the scores
// stay where the matrix product leaves them, 64 of one row to a lane.  The threshold's lower bound comes from 64 of a row's 1024: the largest of every sixteen, which hold most of a
// support, and of which any has a threshold below the whole row's.  Only where that leaves long lists (flat scores) are steps taken on all of them.
#include "attn_split.h"

namespace adsp {
namespace split {
constexpr int kLongList = 160;   // keys above a bound from which on a step on all scores pays
constexpr int kMaxPitch = 68;    // of a row's maxima: 16 lanes of 4, on other banks than the next row's

// LDS of a shared part.
struct PrefixLds {
  float maxima[kPrefixRows][kMaxPitch];
  float top[kPrefixRows], bound[kPrefixRows];
  float sums[kWaves][kPrefixRows][2];
  int counts[2][kWaves][kPrefixRows];
  int differs[kPrefixRows];
};

__device__ __forceinline__ bool entry_differs(const SplitParams& p, int b, int i) { return p.tables[(long long)b * p.table_stride + i] != p.prefix_table[i]; }
// The sum over a row's four lanes of a wave: 16 apart.
__device__ __forceinline__ float row_lanes_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Part `part` of the prefix for rows [row0, row0 + 16) of head `kvh`.
template <typename T, int D, int AM, int kTiles> __device__ __forceinline__ void shared_part(const SplitParams& p, int kvh, int row0, int part, PrefixLds& lds, int* pages) {
  constexpr int kB = elem_traits<T>::kBytes, kSteps = D * kB / 64;
  constexpr int kBatch = kSteps <= 4 ? 2 : 1;  // tiles whose rows of K are under way together
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4, all = p.B * p.R;
  const int key0 = part * p.chunk, end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix, n = end - key0;
  const int first = page_of(p, key0), count = page_of(p, end - 1) - first + 1;
  const int b0 = row0 / p.R, b1 = (row0 + kPrefixRows < all ? row0 + kPrefixRows - 1 : all - 1) / p.R;
  // ---- pages, and the requests that have them ----
  if (tid <= b1 - b0) lds.differs[tid] = length_at(p.lens, p.lens_bits, b0 + tid, p.N) < end ? 1 : 0;
  for (int i = tid; i < count; i += 64 * kWaves) {
    const int id = p.prefix_table[first + i];
    pages[i] = (unsigned)id < (unsigned)p.pages ? id : -1;
  }
  // (asked for now, looked at behind the scores: the first entries of the requests' tables and what the prefix has there)
  const int entries = count * (b1 - b0 + 1);
  constexpr int kAsked = 2;
  int theirs[kAsked], ours[kAsked];
#pragma unroll
  for (int u = 0; u < kAsked; ++u) {
    const int i = tid + u * 64 * kWaves < entries ? tid + u * 64 * kWaves : 0;
    theirs[u] = p.tables[(long long)(b0 + i / count) * p.table_stride + first + i % count];
    ours[u] = p.prefix_table[first + i % count];
  }
  const int row = row0 + r < all ? row0 + r : all - 1, b = row / p.R;
  const int unit_row = (b * p.Hkv + kvh) * p.R + (row - b * p.R);
  u32x4 qf[kSteps];
  {
    const u32x4* const src = reinterpret_cast<const u32x4*>((const char*)p.q + (size_t)unit_row * D * kB) + g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = src[s * 4];
  }
  __syncthreads();
  // ---- scores: tile j of a wave has keys 16 (4 j + wave) .. + 15, a lane 4 g .. + 3 of them for row r; the next tiles' rows of K are under way while these are multiplied ----
  const char* const kbase = (const char*)p.k + kvh * p.k_sh * kB + g * 16;
  f32x4 z[kTiles];
  u32x4 kf[2][kBatch][kSteps];
  int there[2];
  auto load = [&](int j0, int to) {
    there[to] = 0;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = ((j0 + j) * kWaves + wave) * 16 + r, key = key0 + (at < n ? at : n - 1);
      const int pg = page_of(p, key), id = pages[pg - first];
      there[to] |= (id >= 0 && at < n ? 1 : 0) << j;
      const long long off = (id >= 0 ? id : 0) * p.k_s0 + (key - pg * p.page) * p.k_sn;
      const u32x4* const src = reinterpret_cast<const u32x4*>(kbase + off * kB);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kf[to][j][s] = src[s * 4];
    }
  };
  load(0, 0);
#pragma unroll
  for (int j0 = 0; j0 < kTiles; j0 += kBatch) {
    const int now = j0 / kBatch & 1;
    if (j0 + kBatch < kTiles) load(j0 + kBatch, 1 - now);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      z[j0 + j] = rows_product<T>(kf[now][j], qf);
#pragma unroll
      for (int i = 0; i < 4; ++i) z[j0 + j][i] *= p.rows.scale;
    }
    if (__builtin_amdgcn_ballot_w64(there[now] != (1 << kBatch) - 1) != 0) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[j0 + j][i] = __shfl(there[now], g * 4 + i, 64) >> j & 1 ? z[j0 + j][i] : -INFINITY;
    }
  }
#pragma unroll
  for (int u = 0; u < kAsked; ++u)
    if (tid + u * 64 * kWaves < entries && theirs[u] != ours[u]) lds.differs[(tid + u * 64 * kWaves) / count] = 1;
  for (int i = tid + kAsked * 64 * kWaves; i < entries; i += 64 * kWaves)
    if (entry_differs(p, b0 + i / count, first + i % count)) lds.differs[i / count] = 1;
  // ---- a lower bound of each row's threshold from the largest scores of its runs of sixteen ----
  f32x4 most = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < kTiles; ++j) most[j % 4] = fmaxf(most[j % 4], fmaxf(fmaxf(z[j][0], z[j][1]), fmaxf(z[j][2], z[j][3])));
  *reinterpret_cast<f32x4*>(&lds.maxima[r][(wave * 4 + g) * 4]) = most;
  __syncthreads();
  {
    const int solved = wave * 4 + g;  // sixteen lanes to a row
    const f32x4 x = *reinterpret_cast<const f32x4*>(&lds.maxima[solved][r * 4]);
    const float m = group16_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    // (below the maximum less 1 by some roundings; a score of +inf: the bound lies there, above which no key of the row lies, and the row is 0)
    float t = m > -INFINITY && m < INFINITY ? m - 1.f - 2e-6f * fmaxf(fabsf(m), 1.f) : m;
    for (int it = 0; it < 5; ++it) {
      float a[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) accum_stats<AM>(x[e] - t, p.rows.c0, a);
      a[0] = group16_sum(a[0]);
      a[1] = group16_sum(a[1]);
      if (m > -INFINITY && m < INFINITY) t = raised<AM>(t, a[0], a[1], p.rows);
    }
    if (r == 0) {
      lds.top[solved] = m;
      lds.bound[solved] = t;
    }
  }
  __syncthreads();
  // ---- the keys above it, in the order of the lanes that have them ----
  const bool mine = row0 + r < all && !lds.differs[b - b0];
  const float m = lds.top[r];
  const bool solvable = m > -INFINITY && m < INFINITY;
  float t = lds.bound[r];
  int upto, total;
  for (int pass = 0;; ++pass) {
    const float above = mine && m > -INFINITY ? t : INFINITY;
    int c = 0;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) c += z[j][i] > above ? 1 : 0;
    int s = c, y = __shfl_up(s, 16, 64);
    s += g >= 1 ? y : 0;
    y = __shfl_up(s, 32, 64);
    s += g >= 2 ? y : 0;
    if (g == 3) lds.counts[pass & 1][wave][r] = s;
    __syncthreads();
    upto = s - c;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int in_wave = lds.counts[pass & 1][w][r];
      upto += w < wave ? in_wave : 0;
      total += in_wave;
    }
    if (pass == 4 || __builtin_amdgcn_ballot_w64(total > kLongList) == 0) break;
    // a step of Newton's method on all scores
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) accum_stats<AM>(z[j][i] - t, p.rows.c0, a);
    a[0] = row_lanes_sum(a[0]);
    a[1] = row_lanes_sum(a[1]);
    if (g == 0) {
      lds.sums[wave][r][0] = a[0];
      lds.sums[wave][r][1] = a[1];
    }
    __syncthreads();
    a[0] = a[1] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      a[0] += lds.sums[w][r][0];
      a[1] += lds.sums[w][r][1];
    }
    if (solvable) t = raised<AM>(t, a[0], a[1], p.rows);
  }
  if (!mine) return;
  const uint32_t at = (uint32_t)unit_row * p.splits + part;
  if (m > -INFINITY) {
    // (the entries' bytes are below 2^32: one register of an address to a lane)
    uint32_t to = (at * p.chunk + upto) * (uint32_t)sizeof(Entry);
    const int key = key0 + wave * 16 + g * 4;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (z[j][i] > t) {
          *reinterpret_cast<Entry*>((char*)p.entries + to) = Entry{z[j][i], key + j * kWaves * 16 + i};
          to += sizeof(Entry);
        }
  }
  if (wave == 0 && g == 0) p.parts[at] = m > -INFINITY ? Part{m, t, total} : Part{-INFINITY, -INFINITY, 0};
}

// A request's keys [key0, end) as part `part`, by its own workgroup.
template <typename T, int D, int AM> __device__ __forceinline__ void own_part(const SplitParams& p, int unit, int key0, int end, int part, float* z) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), zs = score_stride(p.chunk), b = unit / p.Hkv;
  int* const pages = reinterpret_cast<int*>(z + p.R * zs);
  const int first = page_of(p, key0), last = page_of(p, end - 1);
  __syncthreads();  // (the part before has been read)
  for (int i = first + tid; i <= last; i += 64 * kWaves) pages[i - first] = table_entry(p, b, i);
  __syncthreads();
  chunk_scores<T, D, true, kWaves>(p, b, unit % p.Hkv, key0, end - key0, z, pages, wave, lane);
  __syncthreads();
  for (int row = wave; row < p.R; row += kWaves) leave_part<AM>(p, z + row * zs, end - key0, key0, ((size_t)unit * p.R + row) * p.splits + part, lane);
}
constexpr int kChecked = 64;  // parts of requests that a workgroup looks at together

// Workgroups: the requests' own parts, behind the prefix (they read most of what comes from memory); the prefix's; and those that look for parts of the prefix that a request does not have in
// common and do them, a part of every `checkers`-th item each: where the tables are what the prefix table says they have nothing to do.
template <typename T, int D, int AM, int kTiles> __global__ __launch_bounds__(64 * kWaves) void split_prefix_kernel(SplitParams p, int row_blocks, int checkers) {
  extern __shared__ __align__(16) float z[];
  const int tid = threadIdx.x, behind = p.units * (p.splits - p.prefix_parts), common = p.Hkv * row_blocks * p.prefix_parts;
  int at = blockIdx.x;
  if (at < behind) {
    const int unit = at % p.units, part = at / p.units, key0 = p.prefix + part * p.chunk, len = length_at(p.lens, p.lens_bits, unit / p.Hkv, p.N);
    if (key0 < len) own_part<T, D, AM>(p, unit, key0, key0 + p.chunk < len ? key0 + p.chunk : len, p.prefix_parts + part, z);
    return;
  }
  at -= behind;
  if (at < common) {
    const int kvh = at % p.Hkv, block = at / p.Hkv % row_blocks, part = at / p.Hkv / row_blocks;
    shared_part<T, D, AM, kTiles>(p, kvh, block * kPrefixRows, part, *reinterpret_cast<PrefixLds*>(z), reinterpret_cast<int*>(z) + sizeof(PrefixLds) / 4);
    return;
  }
  at -= common;
  __shared__ int todo[kChecked];
  const long long items = (long long)p.units * p.prefix_parts;
  const int most = (p.chunk - 1) / p.page + 2;  // pages of a part
  for (long long item0 = at; item0 < items; item0 += (long long)checkers * kChecked) {
    const int n = (int)(((items - item0 - 1) / checkers + 1) < kChecked ? (items - item0 - 1) / checkers + 1 : kChecked);
    __syncthreads();
    // item: part by part of a unit, so that one unit's parts fall to many workgroups
    auto part_of = [&](int i, int& unit, int& key0, int& end) {
      const long long item = item0 + (long long)i * checkers;
      unit = (int)(item / p.prefix_parts);
      const int part = (int)(item - (long long)unit * p.prefix_parts);
      key0 = part * p.chunk;
      end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix;
      return part;
    };
    for (int i = tid; i < n; i += 64 * kWaves) {
      int unit, key0, end;
      part_of(i, unit, key0, end);
      const int len = length_at(p.lens, p.lens_bits, unit / p.Hkv, p.N);
      todo[i] = len < end ? (len > key0 ? len : 0) : -1;  // where the request's keys end, 0: none, -1: if an entry differs
    }
    __syncthreads();
    for (int i = tid; i < n * most; i += 64 * kWaves) {
      int unit, key0, end;
      part_of(i / most, unit, key0, end);
      const int entry = page_of(p, key0) + i % most;
      if (entry <= page_of(p, end - 1) && entry_differs(p, unit / p.Hkv, entry)) atomicMax(&todo[i / most], 1);
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const int what = todo[i];
      if (what < 0) continue;
      int unit, key0, end;
      const int part = part_of(i, unit, key0, end), len = length_at(p.lens, p.lens_bits, unit / p.Hkv, p.N);
      if (len > key0) own_part<T, D, AM>(p, unit, key0, len < end ? len : end, part, z);
    }
  }
}

template <typename T, int D, int AM, int kTiles> static void launch_tiles(const SplitParams& p, hipStream_t s) {
  const int row_blocks = (p.B * p.R + kPrefixRows - 1) / kPrefixRows;
  const long long items = (long long)p.units * p.prefix_parts;
  const int checkers = (int)(items < 256 ? items : 256);
  const size_t pages = (p.chunk / p.page + 2) * 4, mine = scores_lds(p.R, p.chunk, p.page, true), common = sizeof(PrefixLds) + pages;
  const dim3 grid((unsigned)((long long)p.Hkv * row_blocks * p.prefix_parts + (long long)p.units * (p.splits - p.prefix_parts) + checkers));
  hipLaunchKernelGGL((split_prefix_kernel<T, D, AM, kTiles>), grid, dim3(64 * kWaves), mine > common ? mine : common, s, p, row_blocks, checkers);
}
template <typename T, int D, int AM> static void launch(const SplitParams& p, hipStream_t s) {
  if (p.chunk > 512) launch_tiles<T, D, AM, 16>(p, s);
  else if (p.chunk > 256) launch_tiles<T, D, AM, 8>(p, s);
  else if (p.chunk > 128) launch_tiles<T, D, AM, 4>(p, s);
  else launch_tiles<T, D, AM, 2>(p, s);
}
template <typename T, int D> static void launch_am(const SplitParams& p, int am, hipStream_t s) {
  if (am == AM_15) launch<T, D, AM_15>(p, s);
  else if (am == AM_2) launch<T, D, AM_2>(p, s);
  else launch<T, D, AM_GEN>(p, s);
}
template <> void prefix_scores_launch<ADSP_T>(const SplitParams& p, int D, int am, hipStream_t s) {
  if (D == 32) launch_am<ADSP_T, 32>(p, am, s);
  else if (D == 64) launch_am<ADSP_T, 64>(p, am, s);
  else if (D == 128) launch_am<ADSP_T, 128>(p, am, s);
  else launch_am<ADSP_T, 256>(p, am, s);
}
}  // namespace split
}  // namespace adsp
