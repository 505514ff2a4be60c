// One translation unit per (16-bit type, head dim 64 or 128) of the forward on 32 rows a workgroup with lists (attn_f32_kernel.h), and of the gradients from the lists that it
// kept, for queries and keys of two lengths, compiled with -DADSP_T=<bf16_t|f16_t> -DADSP_TAG=<bf16|f16> -DADSP_D=<head dim>.
#include "attn_f32_kernel.h"

#define ADSP_CAT_(n, a, d) n##a##_d##d
#define ADSP_CAT(n, a, d) ADSP_CAT_(n, a, d)

namespace adsp {
template <int AM> static void launch_fwd(const AttnCrossParams& p, hipStream_t s) {
  const long long rows = (p.N + f32path::kRows - 1) / f32path::kRows;
  const dim3 grid(xcd_grid((long long)p.B * p.Hkv, rows * (p.Hq / p.Hkv)));
  if (f32path::eight_waves(p)) hipLaunchKernelGGL((f32path::attn_rows32_fwd_kernel<ADSP_T, ADSP_D, AM, true, 8>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((f32path::attn_rows32_fwd_kernel<ADSP_T, ADSP_D, AM, true>), grid, dim3(256), 0, s, p);
}
int ADSP_CAT(launch_attn_cross_rows32_fwd_, ADSP_TAG, ADSP_D)(const AttnCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_fwd<ATT_15>(p, s);
  else if (am == ATT_2) launch_fwd<ATT_2>(p, s);
  else launch_fwd<ATT_GEN>(p, s);
  return 0;
}
// what it leaves over: row blocks without lists, and the K/V heads of those
template <int AM> static void launch_dq(const AttnBwdCrossParams& p, hipStream_t s) {
  const long long blocks = (p.N + f32path::kRows - 1) / f32path::kRows;
  hipLaunchKernelGGL((f32path::attn_lists_dq_kernel<ADSP_T, ADSP_D, AM>), dim3(xcd_grid((long long)p.B * p.Hkv, blocks * (p.Hq / p.Hkv))), dim3(256), 0, s, p);
}
int ADSP_CAT(launch_attn_cross_lists_dq_, ADSP_TAG, ADSP_D)(const AttnBwdCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_dq<ATT_15>(p, s);
  else if (am == ATT_2) launch_dq<ATT_2>(p, s);
  else launch_dq<ATT_GEN>(p, s);
  return 0;
}
int ADSP_CAT(launch_attn_cross_lists_dkdv_, ADSP_TAG, ADSP_D)(const AttnBwdCrossParams& p, hipStream_t s) {
  const long long blocks = (p.Nk + f32path::kRows - 1) / f32path::kRows;
  hipLaunchKernelGGL((f32path::attn_lists_dkdv_kernel<ADSP_T, ADSP_D>), dim3(xcd_grid((long long)p.B * p.Hkv, blocks)), dim3(256), 0, s, p);
  return 0;
}
}  // namespace adsp
