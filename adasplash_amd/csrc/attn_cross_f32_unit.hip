// One translation unit per head dim of the single-precision kernels on 32 rows a workgroup for queries and keys of two lengths
// (attn_f32_kernel.h), compiled with -DADSP_D=<64|128>.
#include "attn_f32_kernel.h"

#define ADSP_CAT_(a, d) a##d
#define ADSP_CAT(a, d) ADSP_CAT_(a, d)

namespace adsp {
using namespace f32path;

static dim3 grid_of(int B, int Hkv, int group, int N) { return dim3(xcd_grid((long long)B * Hkv, (long long)((N + kRows - 1) / kRows) * group)); }

template <int AM> static void launch_bwd(const AttnBwdCrossParams& p, hipStream_t s) {
  const dim3 rows = grid_of(p.B, p.Hkv, p.Hq / p.Hkv, p.N);
  if (p.fwd_streams && !p.streams) hipLaunchKernelGGL((attn_lists_dq_kernel<float, ADSP_D, AM>), rows, dim3(256), 0, s, p);  // (few keys: every row block has lists)
  else hipLaunchKernelGGL((attn_rows32_dq_kernel<ADSP_D, AM, true>), rows, dim3(256), 0, s, p);
  if (p.streams) hipLaunchKernelGGL((attn_lists_dkdv_kernel<float, ADSP_D>), grid_of(p.B, p.Hkv, 1, p.Nk), dim3(256), 0, s, p);
  hipLaunchKernelGGL((attn_rows32_dkdv_kernel<ADSP_D, AM, true>), grid_of(p.B, p.Hkv, p.q_parts, p.Nk), dim3(256), 0, s, p);
}
template <int AM> static void launch_fwd(const AttnCrossParams& p, hipStream_t s) {
  const dim3 grid = grid_of(p.B, p.Hkv, p.Hq / p.Hkv, p.N);
  const int waves = few_waves(p);
  if (waves == 1) hipLaunchKernelGGL((attn_rows32_fwd_kernel<float, ADSP_D, AM, true, 1>), grid, dim3(64), 0, s, p);
  else if (waves == 2) hipLaunchKernelGGL((attn_rows32_fwd_kernel<float, ADSP_D, AM, true, 2>), grid, dim3(128), 0, s, p);
  else if (eight_waves(p)) hipLaunchKernelGGL((attn_rows32_fwd_kernel<float, ADSP_D, AM, true, 8>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((attn_rows32_fwd_kernel<float, ADSP_D, AM, true>), grid, dim3(256), 0, s, p);
}
int ADSP_CAT(launch_attn_cross_f32_fwd_d, ADSP_D)(const AttnCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_fwd<ATT_15>(p, s);
  else if (am == ATT_2) launch_fwd<ATT_2>(p, s);
  else launch_fwd<ATT_GEN>(p, s);
  return 0;
}
int ADSP_CAT(launch_attn_cross_f32_bwd_d, ADSP_D)(const AttnBwdCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_bwd<ATT_15>(p, s);
  else if (am == ATT_2) launch_bwd<ATT_2>(p, s);
  else launch_bwd<ATT_GEN>(p, s);
  return 0;
}
}  // namespace adsp
