// One translation unit per (16-bit type, head dim 64 or 128) of the kernels on the supports for queries and keys of two lengths, compiled
// with -DADSP_T=<bf16_t|f16_t> -DADSP_TAG=<bf16|f16> -DADSP_D=<head dim>.
#include "attn_bwd_sparse_kernel.h"
#include "attn_sparse_kernel.h"

#define ADSP_CAT_(n, a, d) n##a##_d##d
#define ADSP_CAT(n, a, d) ADSP_CAT_(n, a, d)

namespace adsp {
int ADSP_CAT(launch_attn_cross_sparse_fwd_, ADSP_TAG, ADSP_D)(const AttnCrossParams& p, int am, int max_slots, hipStream_t s) {
  return launch_attn_sparse<ADSP_T, ADSP_D, true>(p, am, max_slots, s);
}
// keys = 0: dQ, 2: dK and dV from its streams
template <int AM> static int launch_bwd(const AttnBwdCrossParams& p, int keys, int max_slots, hipStream_t s) {
  return keys == 2 ? launch_attn_bwd_sparse_one<ADSP_T, ADSP_D, AM, 2, true>(p, max_slots, s) : launch_attn_bwd_sparse_one<ADSP_T, ADSP_D, AM, 0, true>(p, max_slots, s);
}
int ADSP_CAT(launch_attn_cross_sparse_bwd_, ADSP_TAG, ADSP_D)(const AttnBwdCrossParams& p, int am, int keys, int max_slots, hipStream_t s) {
  if (am == ATT_15) return launch_bwd<ATT_15>(p, keys, max_slots, s);
  if (am == ATT_2) return launch_bwd<ATT_2>(p, keys, max_slots, s);
  return launch_bwd<ATT_GEN>(p, keys, max_slots, s);
}
}  // namespace adsp
