// One translation unit per element type (-DADSP_T=...): the first kernel of paged attention where many requests' tables start with the same pages.
//
// A workgroup takes a part of the prefix and up to 64 rows (queries of whatever requests): a wave holds 64 keys in registers and goes through the rows, sixteen at a time.  Rows whose
// request does not have these pages, or ends inside the part, are left to other workgroups, which look at the tables in the same way and do a part of the prefix for one request only
// where it was left: the prefix table says what is worth sharing, and no more.
//
// What bounds it: K from memory, and with many rows the products and vector instructions.  Scores are not kept but formed twice, which the matrix units have time for: for the largest of every few, 64 of a
// row's keys in a part, whose threshold is a lower bound of the row's and close to the part's, as they hold most of its support; and for the keys above it.  Of those a lane has one here and
// there: four scores of which one lies above go to a queue in LDS, from which 64 lanes take 64 such together.  Only where the maxima say that many keys lie above (flat scores) steps are taken on all.
#include "attn_split.h"

namespace adsp {
namespace split {
constexpr int kMaxPitch = 68;  // of a row's 64 maxima: on other banks than the next row's
// Of a row's 64 maxima above the bound: from more on steps on all scores pay.  us, 32/8 heads, D = 128, bf16, normal queries times 0.5, 0.35, 0.1, from 48, 62, never: 64 requests behind 8192: 74.0, 65.4, 65.7; 82.8, 75.8, -;
// 205, 205, 213; 16 behind 65500: 138, 122, 123; 181, 171, -; 1883, 1882, 2193.  (Times 1: 52.1, 51.5, 52.3.)
constexpr int kCrowd = 62;
constexpr int kQueue = 128;    // fours of scores of a wave: fewer than 64 that wait, and 64 more

// LDS of a part: queries (pieces of 16 bytes that change places with the row's number: sixteen rows at one piece lie in different banks), the waves' queues, maxima, and a few words a row.
struct PrefixLds {
  unsigned char* q;
  f32x4* queue;                               // [W][kQueue]
  float *maxima, *top, *bound, *near, *sums;  // near: the bound in products, below by some roundings; sums: [W][rows][2]
  int* queue_at;                              // [W][kQueue]
  unsigned long long* above;                  // [W][rows]: the wave's keys above the row's bound, a bit each
  int *differs;                               // of the requests that have rows here
  int *unit_row, *item, *pages;               // a row's place among those of all heads, and its request's among those here, or -1
  uint32_t* list;                             // the number of a row's part among all, or ~0
  __device__ __forceinline__ PrefixLds(void* at, int rows, int row_bytes, int W)
      : q((unsigned char*)at),
        queue(reinterpret_cast<f32x4*>(q + rows * row_bytes)),
        maxima(reinterpret_cast<float*>(queue + W * kQueue)),
        top(maxima + rows * kMaxPitch),
        bound(top + rows),
        near(bound + rows),
        sums(near + rows),
        queue_at(reinterpret_cast<int*>(sums + 2 * W * rows)),
        above(reinterpret_cast<unsigned long long*>(queue_at + W * kQueue)),
        differs(reinterpret_cast<int*>(above + W * rows)),
        unit_row(differs + rows),
        item(unit_row + rows),
        pages(item + 2 * rows),
        list(reinterpret_cast<uint32_t*>(item + rows)) {}
  static size_t bytes(int rows, int row_bytes, int W, int pages) {
    return (size_t)rows * row_bytes + (size_t)W * kQueue * 20 + ((size_t)rows * (kMaxPitch + 7 + 4 * W) + pages) * 4;
  }
};
template <int kPieces> __device__ __forceinline__ int place_of_piece(int row, int piece) {
  constexpr int kSide = kPieces < 16 ? 16 / kPieces : 1;
  return row * kPieces + (piece ^ (row / kSide & (kPieces < 16 ? kPieces - 1 : 15)));
}
__device__ __forceinline__ bool entry_differs(const SplitParams& p, int b, int i) { return p.tables[(long long)b * p.table_stride + i] != p.prefix_table[i]; }
__device__ __forceinline__ float quad_sum(float v) {
  v += dpp_move<0xb1, 0xf>(v, v);
  return v + dpp_move<0x4e, 0xf>(v, v);
}
// A bound in products, below it by some roundings: what lies above the bound lies above this.
__device__ __forceinline__ float near_of(float bound, float inv_scale) {
  const float t = bound * inv_scale;
  return t < INFINITY ? t - 1e-6f * fabsf(t) : t;
}
// The sum over a row's four lanes of a wave: 16 apart.
__device__ __forceinline__ float row_lanes_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The products of rows_product for several tiles of keys, a step of all tiles behind the other: no product waits for the one in front of it.
template <typename T, int kTiles, int kSteps> __device__ __forceinline__ void tiles_product(const u32x4 (&k)[kTiles][kSteps], const u32x4 (&q)[kSteps], float (&z)[4 * kTiles]) {
  if constexpr (elem_traits<T>::kVec == 4) {  // (single precision: rows_product has four sums of its own)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const f32x4 acc = rows_product<T>(k[j], q);
#pragma unroll
      for (int i = 0; i < 4; ++i) z[4 * j + i] = acc[i];
    }
  } else {
    f32x4 acc[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        if constexpr (elem_traits<T>::kIsBf16) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[j][s]), __builtin_bit_cast(bf16x8, q[s]), acc[j], 0, 0, 0);
        else acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[j][s]), __builtin_bit_cast(f16x8, q[s]), acc[j], 0, 0, 0);
      }
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[4 * j + i] = acc[j][i];
  }
}

// A part of the prefix and the rows that a workgroup has there: [row0, row0 + 16 row_tiles) of head `kvh`.
template <typename T, int D, int W> struct SharedPart {
  static constexpr int kB = elem_traits<T>::kBytes, kSteps = D * kB / 64, kPieces = D * kB / 16;
  static constexpr int kKeys = wave_keys(D * kB), kTiles = kKeys / 16, kScores = kTiles * 4;  // of a wave, of a lane
  const SplitParams& p;
  const PrefixLds lds;
  const int lane, wave, r, g, rows, key0, part;
  u32x4 kf[kTiles][kSteps];  // the wave's keys; tile j has keys 16 j + r of them in its lanes
  int q_at[kSteps];          // places of a tile's first rows: those of the others lie 16 rows further
  int seen;                  // of the lane's scores, those of keys that are there: bit 4 j + i
  bool whole;

  __device__ __forceinline__ SharedPart(const SplitParams& params, int kvh, int row0, int row_tiles, int which, void* shared)
      : p(params), lds(shared, row_tiles * 16, D * kB, W), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), r(lane & 15), g(lane >> 4),
        rows(row_tiles * 16), key0(which * params.chunk), part(which) {
    const int tid = threadIdx.x, all = p.B * p.R, end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix, n = end - key0;
    const int first = page_of(p, key0), count = page_of(p, end - 1) - first + 1;
    const int b0 = row0 / p.R, b1 = (row0 + rows < all ? row0 + rows - 1 : all - 1) / p.R;
    for (int i = tid; i < count; i += 64 * W) {
      const int id = p.prefix_table[first + i];
      lds.pages[i] = (unsigned)id < (unsigned)p.pages ? id : -1;
    }
    for (int i = tid; i < W * rows; i += 64 * W) lds.above[i] = 0;
    for (int i = tid; i <= b1 - b0; i += 64 * W) lds.differs[i] = length_at(p.lens, p.lens_bits, b0 + i, p.N) < end ? 1 : 0;
    for (int i = tid; i < rows; i += 64 * W) {
      const int row = row0 + i < all ? row0 + i : all - 1, b = row / p.R;
      lds.unit_row[i] = (b * p.Hkv + kvh) * p.R + (row - b * p.R);
      lds.item[i] = row0 + i < all ? b - b0 : -1;
    }
    __syncthreads();
    int there = 0;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const int at = wave * kKeys + j * 16 + r, key = key0 + (at < n ? at : n - 1);
      const int pg = page_of(p, key), id = lds.pages[pg - first];
      there |= (id >= 0 && at < n ? 1 : 0) << j;
      const long long off = (id >= 0 ? id : 0) * p.k_s0 + (key - pg * p.page) * p.k_sn + kvh * p.k_sh;
      const u32x4* const src = reinterpret_cast<const u32x4*>((const char*)p.k + off * kB) + g;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kf[j][s] = src[s * 4];
    }
    for (int i = tid; i < rows * kPieces; i += 64 * W) {
      const int row = i / kPieces, piece = i % kPieces;
      reinterpret_cast<u32x4*>(lds.q)[place_of_piece<kPieces>(row, piece)] = reinterpret_cast<const u32x4*>((const char*)p.q + (size_t)lds.unit_row[row] * D * kB)[piece];
    }
    for (int i = tid; i < count * (b1 - b0 + 1); i += 64 * W) {
      const int item = i / count;
      if (entry_differs(p, b0 + item, first + i % count)) lds.differs[item] = 1;
    }
    whole = __builtin_amdgcn_ballot_w64(there != (1 << kTiles) - 1) == 0;
    seen = 0;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) seen |= (__shfl(there, g * 4 + i, 64) >> j & 1) << (4 * j + i);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q_at[s] = place_of_piece<kPieces>(r, s * 4 + g) * 16;
    __syncthreads();
  }
  // Whether a row is one and has this part's pages; the number of its part among all.
  __device__ __forceinline__ bool has(int row) const { return lds.item[row] >= 0 && !lds.differs[lds.item[row]]; }
  __device__ __forceinline__ uint32_t number(int row) const { return (uint32_t)lds.unit_row[row] * p.splits + part; }
  // products of rows 16 tile + r with the lane's keys 16 j + 4 g + i of the wave's; scores are `scale` times that
  __device__ __forceinline__ void form(int tile, float (&z)[kScores]) const {
    u32x4 qf[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = *reinterpret_cast<const u32x4*>(lds.q + q_at[s] + tile * (16 * D * kB));
    tiles_product<T>(kf, qf, z);
    if (!whole) {
#pragma unroll
      for (int e = 0; e < kScores; ++e) z[e] = seen >> e & 1 ? z[e] : -INFINITY;
    }
  }
  // The keys above the rows' bounds (`near` and `bound`), entry i of wave w at place i W + w of a row's list, so that no wave waits for another.
  __device__ __forceinline__ void leave_entries(int row_tiles) const {
    f32x4* const queue = lds.queue + wave * kQueue;
    int* const queue_at = lds.queue_at + wave * kQueue;
    unsigned long long* const above = lds.above + wave * rows;
    int head = 0, waiting = 0;
    auto take = [&](int n) {  // the first n of the queue, one to a lane
      asm volatile("" ::: "memory");
      if (lane < n) {
        const f32x4 x = queue[(head + lane) % kQueue];
        const int at = queue_at[(head + lane) % kQueue], row = at >> 16, key = key0 + (at & 0xffff);
        const float t = lds.bound[row];
        float z[4];
        uint32_t in = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[i] = x[i] * p.rows.scale;
          in |= z[i] > t ? 1u << i : 0u;
        }
        if (in != 0) {
          // (a row's keys come in their order: those in front of this one have their bits by now, in whatever order the lanes' bits were put there)
          const int bit = (at & 0xffff) - wave * kKeys;
          atomicOr(above + row, (unsigned long long)in << bit);
          const int place = __builtin_popcountll(above[row] & ((1ull << bit) - 1ull));
          uint32_t to = (lds.list[row] * p.chunk + (uint32_t)place * W + wave) * (uint32_t)sizeof(Entry);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (z[i] > t) {
              *reinterpret_cast<Entry*>((char*)p.entries + to) = Entry{z[i], key + i};
              to += W * sizeof(Entry);
            }
        }
      }
      head = (head + n) % kQueue;
      waiting -= n;
      asm volatile("" ::: "memory");
    };
    for (int tile = 0; tile < row_tiles; ++tile) {
      float z[kScores];
      form(tile, z);
      const float t = lds.near[tile * 16 + r];
      const int at = (tile * 16 + r) << 16 | (wave * kKeys + g * 4);
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const bool in = fmaxf(fmaxf(z[4 * j], z[4 * j + 1]), fmaxf(z[4 * j + 2], z[4 * j + 3])) > t;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
        if (in) {
          const int place = (head + waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))) % kQueue;
          queue[place] = f32x4{z[4 * j], z[4 * j + 1], z[4 * j + 2], z[4 * j + 3]};
          queue_at[place] = at + j * 16;
        }
        waiting += __builtin_popcountll(who);
        if (waiting >= 64) take(64);
      }
    }
    take(waiting);
    __syncthreads();
    // what is left of a row: the places up to the longest list's end, those of shorter lists without weight
    for (int i = threadIdx.x; i < rows * W; i += 64 * W) {
      const int row = i / W, w = i % W;
      const uint32_t at = lds.list[row];
      if (at == ~0u) continue;
      int longest = 0;
      for (int v = 0; v < W; ++v) {
        const int c = __builtin_popcountll(lds.above[v * rows + row]);
        longest = c > longest ? c : longest;
      }
      for (int e = __builtin_popcountll(lds.above[w * rows + row]); e < longest; ++e) p.entries[(size_t)at * p.chunk + e * W + w] = Entry{-INFINITY, key0};
      const float m = lds.top[row];
      if (w == 0) p.parts[at] = Part{m, m > -INFINITY ? lds.bound[row] : -INFINITY, longest * W};
    }
  }
};

template <typename T, int D, int AM, int W> __device__ __forceinline__ void shared_part(const SplitParams& p, int kvh, int row0, int row_tiles, int part, void* shared) {
  using S = SharedPart<T, D, W>;
  constexpr int kScores = S::kScores, kMax = 16 / W < kScores ? 16 / W : kScores, kRun = kScores / kMax;  // maxima that a lane leaves of a row, and the scores that each is the largest of
  static_assert(W * 4 * kMax == 64, "64 maxima to a row");
  const S s(p, kvh, row0, row_tiles, part, shared);
  const PrefixLds& lds = s.lds;
  const int tid = threadIdx.x, rows = s.rows, r = s.r, g = s.g, wave = s.wave;
  for (int tile = 0; tile < row_tiles; ++tile) {
    float z[kScores];
    s.form(tile, z);
    float* const to = lds.maxima + (tile * 16 + r) * kMaxPitch + (wave * 4 + g) * kMax;
#pragma unroll
    for (int k = 0; k < kMax; ++k) {
      float most = z[k * kRun];
#pragma unroll
      for (int e = 1; e < kRun; ++e) most = fmaxf(most, z[k * kRun + e]);
      to[k] = fmaxf(most * p.rows.scale, -INFINITY);  // (a NaN has no weight)
    }
  }
  __syncthreads();
  // ---- a lower bound of each row's threshold from these: four lanes to a row, sixteen values to a lane ----
  int crowded = 0;
  const float inv_scale = 1.f / p.rows.scale;
  for (int i = tid; i < 4 * rows; i += 64 * W) {
    const int row = i / 4;
    float x[16], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 four = *reinterpret_cast<const f32x4*>(lds.maxima + row * kMaxPitch + i % 4 * 16 + k * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, x[4 * k + e] = four[e]);
    }
    m = fmaxf(m, dpp_move<0xb1, 0xf>(m, m));
    m = fmaxf(m, dpp_move<0x4e, 0xf>(m, m));
    const bool solvable = m > -INFINITY && m < INFINITY;
    // (below the maximum less 1 by some roundings; a score of +inf: the bound lies there, above which no key of the row lies, and the row is 0)
    float t = solvable ? m - 1.f - 2e-6f * fmaxf(fabsf(m), 1.f) : m, above = 0.f;
    for (int it = 0; it < 4; ++it) {
      float a[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 16; ++e) accum_stats<AM>(x[e] - t, p.rows.c0, a);
      a[0] = quad_sum(a[0]);
      a[1] = quad_sum(a[1]);
      const float to = raised<AM>(t, a[0], a[1], p.rows);
      t = solvable ? to : t;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) above += x[e] > t ? 1.f : 0.f;
    above = quad_sum(above);
    if (i % 4 == 0) {
      // (a row that is no row, or another's, or has no key: nothing lies above its bound)
      const bool mine = s.has(row);
      const float bound = mine && m > -INFINITY ? t : INFINITY;
      lds.top[row] = m;
      lds.bound[row] = bound;
      lds.near[row] = near_of(bound, inv_scale);
      lds.list[row] = mine ? s.number(row) : ~0u;
      crowded |= mine && solvable && above > (float)kCrowd ? 1 : 0;
    }
  }
  int passes = __syncthreads_or(crowded) ? 3 : 0;
  // ---- flat scores: steps of Newton's method on all of them ----
  for (; passes > 0; --passes) {
    for (int tile = 0; tile < row_tiles; ++tile) {
      float z[kScores], a[2] = {0.f, 0.f};
      s.form(tile, z);
      const float t = lds.bound[tile * 16 + r];
#pragma unroll
      for (int e = 0; e < kScores; ++e) accum_stats<AM>(z[e] * p.rows.scale - t, p.rows.c0, a);
      a[0] = row_lanes_sum(a[0]);
      a[1] = row_lanes_sum(a[1]);
      if (g < 2) lds.sums[(wave * rows + tile * 16 + r) * 2 + g] = g ? a[1] : a[0];
    }
    __syncthreads();
    for (int row = tid; row < rows; row += 64 * W) {
      const float t = lds.bound[row];
      float a0 = 0.f, a1 = 0.f;
      for (int w = 0; w < W; ++w) {
        a0 += lds.sums[(w * rows + row) * 2];
        a1 += lds.sums[(w * rows + row) * 2 + 1];
      }
      if (t < INFINITY) {
        const float to = raised<AM>(t, a0, a1, p.rows);
        lds.bound[row] = to;
        lds.near[row] = near_of(to, inv_scale);
      }
    }
    __syncthreads();
  }
  s.leave_entries(row_tiles);
}
// ---- sixteen rows or fewer -------------------------------------------------------------------------------------------
// There the scores stay where the matrix product leaves them, 16 rows of up to 256 keys to a wave: formed once, and fewer steps that wait for one another.  It is straight code, which takes long to
// fetch; with more rows, for which K would have to be loaded again for every sixteen, it loses.  us, 32/8 heads, D = 128, bf16, in all, these -> the others: 4 requests behind 2000: 12.9, 15.9;
// 16 behind 65500: 85 -> 74; 64 behind 8192: 57 -> 50.
struct FewLds {
  float maxima[kFewRows][kMaxPitch];
  float top[kFewRows], bound[kFewRows];
  int counts[kWaves][kFewRows];
  int differs[kFewRows];
};

template <typename T, int D, int AM, int kTiles> __device__ __forceinline__ void few_rows_part(const SplitParams& p, int kvh, int part, FewLds& lds, int* pages) {
  constexpr int row0 = 0;
  constexpr int kB = elem_traits<T>::kBytes, kSteps = D * kB / 64;
  constexpr int kBatch = kSteps <= 4 ? 2 : 1;  // tiles whose rows of K are under way together
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4, all = p.B * p.R;
  const int key0 = part * p.chunk, end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix, n = end - key0;
  const int first = page_of(p, key0), count = page_of(p, end - 1) - first + 1;
  const int b0 = row0 / p.R, b1 = (row0 + kFewRows < all ? row0 + kFewRows - 1 : all - 1) / p.R;
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
  const float m = lds.top[r], t = lds.bound[r];
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
  if (g == 3) lds.counts[wave][r] = s;
  __syncthreads();
  int upto = s - c, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int in_wave = lds.counts[w][r];
    upto += w < wave ? in_wave : 0;
    total += in_wave;
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
template <typename T, int D, int AM, int W> __device__ __forceinline__ void own_part(const SplitParams& p, int unit, int key0, int end, int part, float* z) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), zs = score_stride(p.chunk), b = unit / p.Hkv;
  int* const pages = reinterpret_cast<int*>(z + p.R * zs);
  const int first = page_of(p, key0), last = page_of(p, end - 1);
  __syncthreads();  // (the part before has been read)
  for (int i = first + tid; i <= last; i += 64 * W) pages[i - first] = table_entry(p, b, i);
  __syncthreads();
  chunk_scores<T, D, true, W>(p, b, unit % p.Hkv, key0, end - key0, z, pages, wave, lane);
  __syncthreads();
  for (int row = wave; row < p.R; row += W) leave_part<AM>(p, z + row * zs, end - key0, key0, ((size_t)unit * p.R + row) * p.splits + part, lane);
}
constexpr int kChecked = 64;  // parts of requests that a workgroup looks at together

// Workgroups: the requests' own parts, behind the prefix; those that look for parts of the prefix that a request does not have in common and do them, every `checkers`-th part each: where
// the tables are what the prefix table says they have nothing to do; and the parts of the prefix.
// kFew: tiles of 16 keys of a wave where the rows are sixteen or fewer, else 0.  (Else two workgroups of eight waves to a CU: 128 registers a lane.)
template <typename T, int D, int AM, int W, int kFew>
__global__ __launch_bounds__(64 * W, kFew == 0 && D * elem_traits<T>::kBytes <= 256 ? 4 : 2) void split_prefix_kernel(SplitParams p, int row_tiles, int row_blocks, int checkers) {
  extern __shared__ __align__(16) float z[];
  const int tid = threadIdx.x, behind = p.units * (p.splits - p.prefix_parts);
  int at = blockIdx.x;
  if (at >= behind + checkers) {
    at -= behind + checkers;
    const int kvh = at % p.Hkv, block = at / p.Hkv % row_blocks, part = at / p.Hkv / row_blocks;
    if constexpr (kFew > 0) few_rows_part<T, D, AM, kFew>(p, kvh, part, *reinterpret_cast<FewLds*>(z), reinterpret_cast<int*>(z) + sizeof(FewLds) / 4);
    else shared_part<T, D, AM, W>(p, kvh, block * row_tiles * 16, row_tiles, part, z);
    return;
  }
  // items of the others: a part behind the prefix, or those of the prefix, part by part of a unit, so that one unit's fall to many workgroups
  __shared__ int todo[kChecked];
  const bool checks = at >= behind;
  const long long items = checks ? (long long)p.units * p.prefix_parts : behind;
  const int most = (p.chunk - 1) / p.page + 2, step = checks ? checkers : behind;  // pages of a part
  auto part_of = [&](long long item, int& unit, int& key0, int& end) {
    int part;
    if (checks) {
      unit = (int)(item / p.prefix_parts);
      part = (int)(item - (long long)unit * p.prefix_parts);
      key0 = part * p.chunk;
      end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix;
    } else {
      unit = (int)(item % p.units);
      part = p.prefix_parts + (int)(item / p.units);
      key0 = p.prefix + (part - p.prefix_parts) * p.chunk;
      end = key0 + p.chunk;
    }
    return part;
  };
  for (long long item0 = checks ? at - behind : at; item0 < items; item0 += (long long)step * kChecked) {
    const int n = (int)(((items - item0 - 1) / step + 1) < kChecked ? (items - item0 - 1) / step + 1 : kChecked);
    int unit, key0, end;
    __syncthreads();
    for (int i = tid; i < n; i += 64 * W) {
      part_of(item0 + (long long)i * step, unit, key0, end);
      todo[i] = checks && length_at(p.lens, p.lens_bits, unit / p.Hkv, p.N) >= end ? -1 : 1;  // (done by the workgroups of the prefix, unless an entry differs)
    }
    __syncthreads();
    for (int i = tid; i < (checks ? n * most : 0); i += 64 * W) {
      part_of(item0 + (long long)(i / most) * step, unit, key0, end);
      const int entry = page_of(p, key0) + i % most;
      if (entry <= page_of(p, end - 1) && entry_differs(p, unit / p.Hkv, entry)) atomicMax(&todo[i / most], 1);
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      if (todo[i] < 0) continue;
      const int part = part_of(item0 + (long long)i * step, unit, key0, end), len = length_at(p.lens, p.lens_bits, unit / p.Hkv, p.N);
      if (len > key0) own_part<T, D, AM, W>(p, unit, key0, len < end ? len : end, part, z);
    }
  }
}

template <typename T, int D, int AM, int W, int kFew> static void launch_waves(const SplitParams& p, hipStream_t s) {
  constexpr int kRowBytes = D * elem_traits<T>::kBytes;
  const int tiles = (p.B * p.R + 15) / 16, parts = p.Hkv * p.prefix_parts, row_tiles = prefix_row_tiles(tiles, parts, kRowBytes);
  const int row_blocks = (tiles + row_tiles - 1) / row_tiles;
  const long long items = (long long)p.units * p.prefix_parts;
  const int checkers = (int)(items < 256 ? items : 256);
  const size_t mine = scores_lds(p.R, p.chunk, p.page, true), pages = p.chunk / p.page + 2;
  const size_t common = kFew > 0 ? sizeof(FewLds) + pages * 4 : PrefixLds::bytes(row_tiles * 16, kRowBytes, W, (int)pages);
  const dim3 grid((unsigned)((long long)parts * row_blocks + (long long)p.units * (p.splits - p.prefix_parts) + checkers));
  hipLaunchKernelGGL((split_prefix_kernel<T, D, AM, W, kFew>), grid, dim3(64 * W), mine > common ? mine : common, s, p, row_tiles, row_blocks, checkers);
}
template <typename T, int D, int AM> static void launch(const SplitParams& p, hipStream_t s) {
  constexpr int kKeys = wave_keys(D * elem_traits<T>::kBytes);
  if ((long long)p.B * p.R <= kFewRows) {
    if (p.chunk > 512) launch_waves<T, D, AM, kWaves, 16>(p, s);
    else if (p.chunk > 256) launch_waves<T, D, AM, kWaves, 8>(p, s);
    else if (p.chunk > 128) launch_waves<T, D, AM, kWaves, 4>(p, s);
    else launch_waves<T, D, AM, kWaves, 2>(p, s);
  } else if (p.chunk == 8 * kKeys) {
    launch_waves<T, D, AM, 8, 0>(p, s);
  } else if (p.chunk == 4 * kKeys) {
    launch_waves<T, D, AM, 4, 0>(p, s);
  } else if constexpr (kKeys >= 32) {
    launch_waves<T, D, AM, 2, 0>(p, s);
  }
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
