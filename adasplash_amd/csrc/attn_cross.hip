// C ABI of the attention of queries to keys of another length (an encoder's states): argument checks and dispatch.
#include <math.h>

#include "attn_two_lengths.h"
#include "../../include/adasplash_hip.h"

namespace adsp {
#define ADSP_DECL(tag, d)                                                                       \
  int launch_attn_cross_fwd_##tag##_d##d(const AttnCrossParams&, int, hipStream_t);             \
  int launch_attn_cross_bwd_##tag##_d##d(const AttnBwdCrossParams&, int, hipStream_t);          \
  int launch_attn_cross16_fwd_##tag##_d##d(const AttnCrossParams&, int, bool, hipStream_t);     \
  int launch_attn_cross16_bwd_##tag##_d##d(const AttnBwdCrossParams&, int, hipStream_t);
#define ADSP_DECL_TAG(tag) ADSP_DECL(tag, 16) ADSP_DECL(tag, 32) ADSP_DECL(tag, 64) ADSP_DECL(tag, 128) ADSP_DECL(tag, 256)
ADSP_DECL_TAG(f32)
ADSP_DECL_TAG(bf16)
ADSP_DECL_TAG(f16)
int launch_attn_cross_f32_fwd_d64(const AttnCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_fwd_d128(const AttnCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_bwd_d64(const AttnBwdCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_bwd_d128(const AttnBwdCrossParams&, int, hipStream_t);

namespace cross {
typedef int (*fwd_fn)(const AttnCrossParams&, int, hipStream_t);
typedef int (*bwd_fn)(const AttnBwdCrossParams&, int, hipStream_t);
typedef int (*fwd16_fn)(const AttnCrossParams&, int, bool, hipStream_t);
// indexed by adsp_dtype and by the head dim's place among 16, 32, 64, 128, 256
#define ADSP_ROW(name, tag) {name##_##tag##_d16, name##_##tag##_d32, name##_##tag##_d64, name##_##tag##_d128, name##_##tag##_d256}
static const fwd_fn kFwd[3][5] = {ADSP_ROW(launch_attn_cross_fwd, f32), ADSP_ROW(launch_attn_cross_fwd, bf16), ADSP_ROW(launch_attn_cross_fwd, f16)};
static const bwd_fn kBwd[3][5] = {
    ADSP_ROW(launch_attn_cross_bwd, f32),
    {launch_attn_cross_bwd_bf16_d16, launch_attn_cross_bwd_bf16_d32, launch_attn_cross16_bwd_bf16_d64, launch_attn_cross16_bwd_bf16_d128, launch_attn_cross_bwd_bf16_d256},
    {launch_attn_cross_bwd_f16_d16, launch_attn_cross_bwd_f16_d32, launch_attn_cross16_bwd_f16_d64, launch_attn_cross16_bwd_f16_d128, launch_attn_cross_bwd_f16_d256}};
static const fwd16_fn kFwd16[2][2] = {{launch_attn_cross16_fwd_bf16_d64, launch_attn_cross16_fwd_bf16_d128}, {launch_attn_cross16_fwd_f16_d64, launch_attn_cross16_fwd_f16_d128}};

static int slot_of(int D) { return D == 16 ? 0 : (D == 32 ? 1 : (D == 64 ? 2 : (D == 128 ? 3 : (D == 256 ? 4 : -1)))); }
// An alpha whose 1 / (alpha - 1) is 1 in fp32 is 2 to the kernels: the generic ones raise u = 0 to the power 1 / (alpha - 1) - 1.
static int alpha_mode(double alpha) { return alpha == 1.5 ? ATT_15 : (alpha == 2.0 || (float)(1.0 / (alpha - 1.0)) == 1.f ? ATT_2 : ATT_GEN); }
// The kernels made for head dims 64 and 128: an alpha whose powers stay inside fp32, and in single precision 16-bit key indices.
static bool special(int D, int dtype, double alpha, int Nk) {
  return (D == 64 || D == 128) && alpha >= 1.125 && (dtype != ADSP_F32 || Nk <= 65536);
}

static int check(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, const void* vq, int vq_bits, const void* vk, int vk_bits) {
  if (dtype != ADSP_F32 && dtype != ADSP_BF16 && dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Nq <= 0 || Nk <= 0 || Hq % Hkv != 0 || slot_of(D) < 0) return ADSP_ERR_SHAPE;
  constexpr int kMost = kMaskWords * 32 * kBN;
  if (Nq > kMost || Nk > kMost) return ADSP_ERR_SHAPE;
  // (workgroups of 32 rows, a launch's number of them)
  if ((long long)B * Hq * ((Nq + 31) / 32 + (Nk + 31) / 32) >= (1ll << 30)) return ADSP_ERR_SHAPE;
  if (!(alpha > 1.0) || alpha > 2.0) return ADSP_ERR_UNSUPPORTED;
  if ((vq && vq_bits != 32 && vq_bits != 64) || (vk && vk_bits != 32 && vk_bits != 64)) return ADSP_ERR_UNSUPPORTED;
  return ADSP_OK;
}
}  // namespace cross
}  // namespace adsp

extern "C" int adsp_attn_cross_fwd(const void* q, const void* k, const void* v, void* out, float* taus, const void* varlen_q, int varlen_q_bits,
                                   const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha,
                                   void* stream) {
  using namespace adsp;
  if (!q || !k || !v || !out) return ADSP_ERR_NULL;
  const int rc = cross::check(B, Hq, Hkv, Nq, Nk, D, dtype, alpha, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  if (rc != ADSP_OK) return rc;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) != 0) return ADSP_ERR_ALIGN;
  AttnCrossParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.taus = taus;
  p.varlen = varlen_q;
  p.varlen_bits = varlen_q_bits;
  p.varlen_k = varlen_k;
  p.varlen_k_bits = varlen_k_bits;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.N = Nq;
  p.Nk = Nk;
  p.n_mblk = (Nq + kMaskRows - 1) / kMaskRows;
  p.mask_words = ((Nk + kBN - 1) / kBN + 31) / 32;
  p.niter = 11;  // (of the tile kernel's steps as many as the block-mask variant takes; the others iterate to convergence)
  p.alpha = (float)alpha;
  p.c0 = (float)(1.0 / (alpha - 1.0));
  p.qscale = (float)((alpha - 1.0) / sqrt((double)D));
  const int am = cross::alpha_mode(alpha), slot = cross::slot_of(D);
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  int st;
  if (!cross::special(D, dtype, alpha, Nk)) st = cross::kFwd[dtype][slot](p, am, s);
  else if (dtype == ADSP_F32) st = D == 64 ? launch_attn_cross_f32_fwd_d64(p, am, s) : launch_attn_cross_f32_fwd_d128(p, am, s);
  else st = cross::kFwd16[dtype - ADSP_BF16][D == 128](p, am, Nk <= kResidentMaxKeys, s);
  return st == 0 && hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}

extern "C" int adsp_attn_cross_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus, const void* varlen_q,
                                   int varlen_q_bits, const void* varlen_k, int varlen_k_bits, void* dq, void* dk, void* dv, float* delta, float* zinv,
                                   int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, void* stream) {
  using namespace adsp;
  if (!q || !k || !v || !dout || !taus || !dq || !dk || !dv || !delta || !zinv) return ADSP_ERR_NULL;
  const int rc = cross::check(B, Hq, Hkv, Nq, Nk, D, dtype, alpha, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  if (rc != ADSP_OK) return rc;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) != 0) return ADSP_ERR_ALIGN;
  AttnBwdCrossParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.dout = dout;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.taus = taus;
  p.delta = delta;
  p.zinv = zinv;
  p.varlen = varlen_q;
  p.varlen_bits = varlen_q_bits;
  p.varlen_k = varlen_k;
  p.varlen_k_bits = varlen_k_bits;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.N = Nq;
  p.Nk = Nk;
  p.n_mblk = (Nq + kMaskRows - 1) / kMaskRows;
  p.mask_words = ((Nk + kBN - 1) / kBN + 31) / 32;
  p.qscale = (float)((alpha - 1.0) / sqrt((double)D));
  p.sm_scale = (float)(1.0 / sqrt((double)D));
  p.c0 = (float)(1.0 / (alpha - 1.0));
  const int am = cross::alpha_mode(alpha);
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  int st;
  if (dtype == ADSP_F32 && cross::special(D, dtype, alpha, Nk)) st = D == 64 ? launch_attn_cross_f32_bwd_d64(p, am, s) : launch_attn_cross_f32_bwd_d128(p, am, s);
  else st = cross::kBwd[dtype][cross::slot_of(D)](p, am, s);
  return st == 0 && hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
