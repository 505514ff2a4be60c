// One translation unit per element type (-DADSP_T=...): parts of a prefix that requests have in common.
//
// The first kernel where many requests' tables start with the same pages.  There a workgroup takes up to 32 rows, of whatever requests, and a part of the prefix: K comes from memory
// once for all of them, and once from L2 for every 32 rows.  Rows whose request does not have these pages, or ends inside the part, are left to the workgroups of the
// requests, which look at the table in the same way and do a part of the prefix only where no other does: the prefix table says what is worth sharing, and no more.
#include "attn_split.h"

namespace adsp {
namespace split {
constexpr int prefix_waves(int row_bytes) { return row_bytes <= 512 ? 8 : 4; }  // (64 rows of K in a wave's registers)

// Scores of keys [key0, key0 + n) of head `kvh`, whose pages lie in LDS, for rows [row0, row0 + 16 kTiles) of all requests: as chunk_scores.
template <typename T, int D, int kTiles, int W>
__device__ __forceinline__ void prefix_scores(const SplitParams& p, int kvh, int row0, int key0, int n, float* z, const int* pages, int wave, int lane) {
  constexpr int kB = elem_traits<T>::kBytes, kSteps = D * kB / 64;
  constexpr int kKeys = kSteps <= 4 ? 4 : (kSteps == 8 ? 2 : 1);  // tiles of 16 keys in registers
  const int r = lane & 15, g = lane >> 4, zs = score_stride(p.chunk), first_page = page_of(p, key0), all = p.B * p.R;
  const char* const kbase = (const char*)p.k + kvh * p.k_sh * kB;
  u32x4 qf[kTiles][kSteps];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int row = row0 + t * 16 + r < all ? row0 + t * 16 + r : all - 1, b = row / p.R;
    const u32x4* src = reinterpret_cast<const u32x4*>((const char*)p.q + ((size_t)(b * p.Hkv + kvh) * p.R + (row - b * p.R)) * D * kB) + g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[t][s] = src[s * 4];
  }
  const int n64 = (n + 63) & ~63;
  for (int k0 = wave * (kKeys * 16); k0 < n64; k0 += W * kKeys * 16) {
    u32x4 kf[kKeys][kSteps];
    int there = 0;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int at = k0 + j * 16 + r, key = key0 + (at < n ? at : n - 1);
      const int pg = page_of(p, key), id = pages[pg - first_page];
      there |= (id >= 0 ? 1 : 0) << j;
      const long long off = (id >= 0 ? id : 0) * p.k_s0 + (key - pg * p.page) * p.k_sn;
      const u32x4* src = reinterpret_cast<const u32x4*>(kbase + off * kB) + g;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kf[j][s] = src[s * 4];
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int j = 0; j < kKeys; ++j) {
        f32x4 acc = rows_product<T>(kf[j], qf[t]);
        const int at = k0 + j * 16 + g * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool see = at + i < n && (__shfl(there, g * 4 + i, 64) >> j & 1);
          acc[i] = see ? acc[i] * p.rows.scale : -INFINITY;
        }
        *reinterpret_cast<f32x4*>(z + (t * 16 + r) * zs + at) = acc;
      }
    }
  }
}
__device__ __forceinline__ bool entry_differs(const SplitParams& p, int b, int i) { return p.tables[(long long)b * p.table_stride + i] != p.prefix_table[i]; }

template <typename T, int D, int AM, int kTiles, int W> __global__ __launch_bounds__(64 * W) void split_prefix_kernel(SplitParams p, int row_blocks, int strides) {
  extern __shared__ __align__(16) float z[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), zs = score_stride(p.chunk);
  const int common = p.Hkv * row_blocks * p.prefix_parts;
  int at = blockIdx.x;
  if (at < common) {
    const int kvh = at % p.Hkv, block = at / p.Hkv % row_blocks, part = at / p.Hkv / row_blocks, row0 = block * kTiles * 16, all = p.B * p.R;
    const int key0 = part * p.chunk, end = key0 + p.chunk < p.prefix ? key0 + p.chunk : p.prefix, n = end - key0;
    int* const differs = reinterpret_cast<int*>(z + kTiles * 16 * zs);
    int* const pages = differs + kPrefixRows;
    const int first = page_of(p, key0), count = page_of(p, end - 1) - first + 1;
    const int b0 = row0 / p.R, b1 = (row0 + kTiles * 16 < all ? row0 + kTiles * 16 - 1 : all - 1) / p.R;
    if (tid <= b1 - b0) differs[tid] = length_at(p.lens, p.lens_bits, b0 + tid, p.N) < end ? 1 : 0;
    for (int i = tid; i < count; i += 64 * W) {
      const int id = p.prefix_table[first + i];
      pages[i] = (unsigned)id < (unsigned)p.pages ? id : -1;
    }
    __syncthreads();
    for (int i = tid; i < count * (b1 - b0 + 1); i += 64 * W) {
      const int b = i / count;
      if (entry_differs(p, b0 + b, first + i % count)) differs[b] = 1;
    }
    prefix_scores<T, D, kTiles, W>(p, kvh, row0, key0, n, z, pages, wave, lane);
    __syncthreads();
    for (int i = wave; i < kTiles * 16 && row0 + i < all; i += W) {
      const int b = (row0 + i) / p.R, r = row0 + i - b * p.R;
      if (differs[b - b0]) continue;
      leave_part<AM>(p, z + i * zs, n, key0, ((size_t)(b * p.Hkv + kvh) * p.R + r) * p.splits + part, lane);
    }
    return;
  }
  // a request's own parts: those behind the prefix, a workgroup each, then those of the prefix, `strides` workgroups for all of them
  at -= common;
  const int own = p.splits - p.prefix_parts, unit = at % p.units, group = at / p.units, b = unit / p.Hkv, kvh = unit % p.Hkv;
  const int len = length_at(p.lens, p.lens_bits, b, p.N);
  const bool behind = group < own;
  int* const pages = reinterpret_cast<int*>(z + p.R * zs);
  for (int part = behind ? p.prefix_parts + group : group - own; part < (behind ? p.splits : p.prefix_parts); part += behind ? p.splits : strides) {
    const int key0 = behind ? p.prefix + group * p.chunk : part * p.chunk;
    if (key0 >= len) return;  // (of all parts that come)
    int end = key0 + p.chunk;
    if (!behind && end > p.prefix) end = p.prefix;
    const bool whole = !behind && len >= end;
    if (end > len) end = len;
    const int first = page_of(p, key0), last = page_of(p, end - 1);
    int mine = whole ? 0 : 1;
    __syncthreads();  // (the part before has been read)
    for (int i = first + tid; i <= last; i += 64 * W) {
      pages[i - first] = table_entry(p, b, i);
      if (whole && entry_differs(p, b, i)) mine = 1;
    }
    if (!__syncthreads_or(mine)) continue;  // (computed for all)
    chunk_scores<T, D, true, W>(p, b, kvh, key0, end - key0, z, pages, wave, lane);
    __syncthreads();
    for (int row = wave; row < p.R; row += W) leave_part<AM>(p, z + row * zs, end - key0, key0, ((size_t)unit * p.R + row) * p.splits + part, lane);
  }
}

template <typename T, int D, int AM> static void launch(const SplitParams& p, hipStream_t s) {
  constexpr int W = prefix_waves(D * elem_traits<T>::kBytes);
  const int rows = p.B * p.R, strides = p.prefix_parts < 8 ? p.prefix_parts : 8, own = p.splits - p.prefix_parts;
  const int block_rows = rows <= 16 ? 16 : kPrefixRows, row_blocks = (rows + block_rows - 1) / block_rows;
  const size_t lds = prefix_lds(p.R > block_rows ? p.R : block_rows, p.chunk, p.page);
  const dim3 grid((unsigned)((long long)p.Hkv * row_blocks * p.prefix_parts + (long long)p.units * (own + strides)));
  if (rows <= 16) hipLaunchKernelGGL((split_prefix_kernel<T, D, AM, 1, W>), grid, dim3(64 * W), lds, s, p, row_blocks, strides);
  else hipLaunchKernelGGL((split_prefix_kernel<T, D, AM, 2, W>), grid, dim3(64 * W), lds, s, p, row_blocks, strides);
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
