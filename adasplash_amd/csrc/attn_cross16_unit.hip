// One translation unit per (16-bit type, head dim 64 or 128) of the attention kernels for queries and keys of two lengths, compiled with
// -DADSP_T=<bf16_t|f16_t> -DADSP_TAG=<bf16|f16> -DADSP_D=<head dim>: the forward with resident scores, the forward and the gradients on all pairs.
#include "attn_bwd16_kernel.h"
#include "attn_fwd16_kernel.h"
#include "attn_resident_kernel.h"

#define ADSP_CAT_(n, a, d) n##a##_d##d
#define ADSP_CAT(n, a, d) ADSP_CAT_(n, a, d)

namespace adsp {

static dim3 grid_of(const AttnParams& p, int rows) { return dim3(xcd_grid((long long)p.B * p.Hkv, (long long)((p.N + rows - 1) / rows) * (p.Hq / p.Hkv))); }

// The fewest waves whose registers hold the longest rows, four at least; one, where it holds them, in a launch of more than 512 row blocks: then nothing waits for another
// wave, and none is idle.  us, four waves -> one: 17 x 32/16 heads, 969 x 3, D = 128: 102 -> 53 (5.1 TB/s); 969 x 60: 125 -> 72; 969 x 120: 170 -> 128; 4 x 8, 2000 x 100, D = 64:
// 16.6 -> 12.3; 700 x 100: 8.4, 8.5; 8 x 8, 300 x 60: 6.8 -> 6.3.  (Two waves for up to 256 keys: 17 x 32/16, 969 x 250: 225, 221, flat scores 219, 227.)
template <int AM> static void launch_resident(const AttnCrossParams& p, hipStream_t s) {
  using namespace resident;
  const dim3 grid = grid_of(p, kRows);
  if (p.Nk <= kRows * kBlocks && (long long)p.B * p.Hq * ((p.N + kRows - 1) / kRows) > 512) hipLaunchKernelGGL((attn_resident_fwd_kernel<ADSP_T, ADSP_D, AM, 1, true>), grid, dim3(64), 0, s, p);
  else if (p.Nk <= kRows * kBlocks * 4) hipLaunchKernelGGL((attn_resident_fwd_kernel<ADSP_T, ADSP_D, AM, 4, true>), grid, dim3(256), 0, s, p);
  else if (p.Nk <= kRows * kBlocks * 8) hipLaunchKernelGGL((attn_resident_fwd_kernel<ADSP_T, ADSP_D, AM, 8, true>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((attn_resident_fwd_kernel<ADSP_T, ADSP_D, AM, kMaxWaves, true>), grid, dim3(64 * kMaxWaves), 0, s, p);
}
template <int AM> static void launch_all_pairs(const AttnCrossParams& p, hipStream_t s) {
  using namespace fwd16;
  const dim3 grid = grid_of(p, kMaskRows);
  if (p.taus) hipLaunchKernelGGL((attn_fwd16_kernel<ADSP_T, ADSP_D, AM, true, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((attn_fwd16_kernel<ADSP_T, ADSP_D, AM, false, true>), grid, dim3(256), 0, s, p);
}
template <int AM> static void launch_fwd(const AttnCrossParams& p, bool resident, hipStream_t s) {
  if (resident) launch_resident<AM>(p, s);
  else launch_all_pairs<AM>(p, s);
}
int ADSP_CAT(launch_attn_cross16_fwd_, ADSP_TAG, ADSP_D)(const AttnCrossParams& p, int am, bool resident, hipStream_t s) {
  if (resident && p.Nk > kResidentMaxKeys) return -1;
  if (am == ATT_15) launch_fwd<ATT_15>(p, resident, s);
  else if (am == ATT_2) launch_fwd<ATT_2>(p, resident, s);
  else launch_fwd<ATT_GEN>(p, resident, s);
  return 0;
}

template <int AM, int P, bool kSplit> static void launch_dq(const AttnBwdCrossParams& p, hipStream_t s) {
  const long long blocks = (p.N + 128 / P - 1) / (128 / P);
  hipLaunchKernelGGL((bwd16::attn_bwd16_dq_kernel<ADSP_T, ADSP_D, AM, P, kSplit, true>), dim3(xcd_grid((long long)p.B * p.Hkv, blocks * (p.Hq / p.Hkv))), dim3(256), 0, s, p);
}
template <int AM, int P> static void launch_dkdv(const AttnBwdCrossParams& p, hipStream_t s) {
  const long long blocks = (long long)((p.Nk + 128 / P - 1) / (128 / P)) * (P == 4 ? p.q_parts : 1);
  hipLaunchKernelGGL((bwd16::attn_bwd16_dkdv_kernel<ADSP_T, ADSP_D, AM, P, true>), dim3(xcd_grid((long long)p.B * p.Hkv, blocks)), dim3(256), 0, s, p);
}
// Parts that a row's walk is split in: as few as give every CU a workgroup of 128 / parts rows.
static int parts_of(long long rows) { return rows >= 256ll * 128 ? 1 : (rows >= 256ll * 64 ? 2 : 4); }
// At head dim 128, where a CU has one workgroup, two parts already where three CUs of four get one: 8 x 16/4 heads, 200 x 500, gradients: 98 us with four, 79 with two; 8 x 16/8, 160 x 200: 57, 44; D = 64:
// 39, 44.
static int parts_of_keys(long long rows) { return ADSP_D == 128 && rows >= 192ll * 64 && rows < 256ll * 64 ? 2 : parts_of(rows); }
// which: 1 = dQ, 2 = dK and dV, 3 = both.  dQ's weights are two 16-bit values each where these kernels serve the call, as in the short training steps of the attention of a sequence to itself: the
// result's own rounding is all that is left (16 x 12 heads, 130 x 500, bf16, against 64 bits: 2.4e-3 -> 1.7e-3; f16 3.0e-4 -> 2.1e-4).  A step, us: that one 53.4 -> 54.8; 2 x 8, 448 x 1000, D = 64: 41.2 -> 42.4;
// 8 x 16/4, 200 x 500, D = 128: 90.6 -> 92.8.  Behind the kernels on the supports (block_flags) one value, as there.
template <int AM> static void launch_bwd(const AttnBwdCrossParams& p, int which, hipStream_t s) {
  const int pq = parts_of((long long)p.B * p.Hq * p.N), pk = p.q_parts > 1 ? 4 : parts_of_keys((long long)p.B * p.Hkv * p.Nk);
  if (which & 1) {
    if (!p.block_flags) {
      if (pq == 1) launch_dq<AM, 1, true>(p, s);
      else if (pq == 2) launch_dq<AM, 2, true>(p, s);
      else launch_dq<AM, 4, true>(p, s);
    } else {
      if (pq == 1) launch_dq<AM, 1, false>(p, s);
      else if (pq == 2) launch_dq<AM, 2, false>(p, s);
      else launch_dq<AM, 4, false>(p, s);
    }
  }
  if (which & 2) {
    AttnBwdCrossParams pd = p;
    pd.n_mblk = (p.Nk + kMaskRows - 1) / kMaskRows;  // (the key blocks' flags)
    if (pk == 1) launch_dkdv<AM, 1>(pd, s);
    else if (pk == 2) launch_dkdv<AM, 2>(pd, s);
    else launch_dkdv<AM, 4>(pd, s);
  }
}
int ADSP_CAT(launch_attn_cross16_bwd_, ADSP_TAG, ADSP_D)(const AttnBwdCrossParams& p, int am, int which, hipStream_t s) {
  if (am == ATT_15) launch_bwd<ATT_15>(p, which, s);
  else if (am == ATT_2) launch_bwd<ATT_2>(p, which, s);
  else launch_bwd<ATT_GEN>(p, which, s);
  return 0;
}
}  // namespace adsp
