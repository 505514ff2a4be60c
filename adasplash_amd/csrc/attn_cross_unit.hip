// One translation unit per (element type, head dim) of the tile kernels for queries and keys of two lengths (attn_kernel.h,
// attn_bwd_kernel.h): what the kernels made for head dims 64 and 128 do not take.  Compiled with -DADSP_T=<bf16_t|f16_t|float>
// -DADSP_TAG=<bf16|f16|f32> -DADSP_D=<head dim>.  (The 16-bit gradients at head dims 64 and 128 are attn_cross16_unit.hip's, whatever alpha is.)
#include "attn_bwd_kernel.h"

#define ADSP_CAT_(n, a, d) n##a##_d##d
#define ADSP_CAT(n, a, d) ADSP_CAT_(n, a, d)

namespace adsp {

template <int AM> static void launch_fwd(const AttnCrossParams& p, hipStream_t s) {
  using G = TileGeo<ADSP_T, ADSP_D>;
  AttnCrossParams q = p;
  q.fine_masks = p.mask_words <= 64 ? 1 : 0;  // (up to 128K keys: beyond, the block bits would cost occupancy)
  const size_t words = (size_t)(q.fine_masks ? 4 + 4 * G::kNW : 4) * p.mask_words + G::kPoolTail;
  const long long blocks = (p.N + G::kBM - 1) / G::kBM;
  hipLaunchKernelGGL((attn_fwd_kernel<ADSP_T, ADSP_D, AM, true, true>), dim3(xcd_grid((long long)p.B * p.Hkv, blocks * (p.Hq / p.Hkv))), dim3(G::kThreads),
                     words * sizeof(uint32_t), s, q);
}
int ADSP_CAT(launch_attn_cross_fwd_, ADSP_TAG, ADSP_D)(const AttnCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_fwd<ATT_15>(p, s);
  else if (am == ATT_2) launch_fwd<ATT_2>(p, s);
  else launch_fwd<ATT_GEN>(p, s);
  return 0;
}

#if ADSP_GRADIENTS
template <int AM> static void launch_bwd(const AttnBwdCrossParams& p, hipStream_t s) {
  const long long heads = (long long)p.B * p.Hkv, rows = (p.N + kBwdRows - 1) / kBwdRows, keys = (p.Nk + kBwdRows - 1) / kBwdRows;
  hipLaunchKernelGGL((attn_bwd_dq_kernel<ADSP_T, ADSP_D, AM, true>), dim3(xcd_grid(heads, rows * (p.Hq / p.Hkv))), dim3(256), 0, s, p);
  hipLaunchKernelGGL((attn_bwd_dkdv_kernel<ADSP_T, ADSP_D, AM, true>), dim3(xcd_grid(heads, keys)), dim3(256), 0, s, p);
}
int ADSP_CAT(launch_attn_cross_bwd_, ADSP_TAG, ADSP_D)(const AttnBwdCrossParams& p, int am, hipStream_t s) {
  if (am == ATT_15) launch_bwd<ATT_15>(p, s);
  else if (am == ATT_2) launch_bwd<ATT_2>(p, s);
  else launch_bwd<ATT_GEN>(p, s);
  return 0;
}
#endif
}  // namespace adsp
