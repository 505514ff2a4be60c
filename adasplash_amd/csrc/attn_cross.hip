// C ABI of the attention of queries to keys of another length (an encoder's states): argument checks, workspaces and dispatch.
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "attn_probe.h"

namespace adsp {
#define ADSP_DECL(tag, d)                                                              \
  int launch_attn_cross_fwd_##tag##_d##d(const AttnCrossParams&, int, hipStream_t);    \
  int launch_attn_cross_bwd_##tag##_d##d(const AttnBwdCrossParams&, int, hipStream_t);
#define ADSP_DECL_TAG(tag) ADSP_DECL(tag, 16) ADSP_DECL(tag, 32) ADSP_DECL(tag, 64) ADSP_DECL(tag, 128) ADSP_DECL(tag, 256)
ADSP_DECL_TAG(f32)
ADSP_DECL_TAG(bf16)
ADSP_DECL_TAG(f16)
int launch_attn_cross_f32_fwd_d64(const AttnCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_fwd_d128(const AttnCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_bwd_d64(const AttnBwdCrossParams&, int, hipStream_t);
int launch_attn_cross_f32_bwd_d128(const AttnBwdCrossParams&, int, hipStream_t);
#define ADSP_DECL_16(tag, d)                                                                    \
  int launch_attn_cross16_fwd_##tag##_d##d(const AttnCrossParams&, int, bool, hipStream_t);     \
  int launch_attn_cross16_bwd_##tag##_d##d(const AttnBwdCrossParams&, int, int, hipStream_t);   \
  int launch_attn_cross_rows32_fwd_##tag##_d##d(const AttnCrossParams&, int, hipStream_t);      \
  int launch_attn_cross_lists_dq_##tag##_d##d(const AttnBwdCrossParams&, int, hipStream_t);     \
  int launch_attn_cross_lists_dkdv_##tag##_d##d(const AttnBwdCrossParams&, hipStream_t);        \
  int launch_attn_cross_sparse_fwd_##tag##_d##d(const AttnCrossParams&, int, int, hipStream_t); \
  int launch_attn_cross_sparse_bwd_##tag##_d##d(const AttnBwdCrossParams&, int, int, int, hipStream_t);
ADSP_DECL_16(bf16, 64)
ADSP_DECL_16(bf16, 128)
ADSP_DECL_16(f16, 64)
ADSP_DECL_16(f16, 128)
#define ADSP_CALL_16(name, D, dtype, ...)                                                                \
  ((dtype) == ADSP_BF16 ? ((D) == 64 ? name##_bf16_d64(__VA_ARGS__) : name##_bf16_d128(__VA_ARGS__))    \
                        : ((D) == 64 ? name##_f16_d64(__VA_ARGS__) : name##_f16_d128(__VA_ARGS__)))

namespace cross {
typedef int (*fwd_fn)(const AttnCrossParams&, int, hipStream_t);
typedef int (*bwd_fn)(const AttnBwdCrossParams&, int, hipStream_t);
// indexed by adsp_dtype and by the head dim's place among 16, 32, 64, 128, 256
#define ADSP_ROW(name, tag) {name##_##tag##_d16, name##_##tag##_d32, name##_##tag##_d64, name##_##tag##_d128, name##_##tag##_d256}
static const fwd_fn kFwd[3][5] = {ADSP_ROW(launch_attn_cross_fwd, f32), ADSP_ROW(launch_attn_cross_fwd, bf16), ADSP_ROW(launch_attn_cross_fwd, f16)};
// (16 bits at head dims 64 and 128: launch_attn_cross16_bwd, whatever alpha is)
static const bwd_fn kBwd[3][5] = {ADSP_ROW(launch_attn_cross_bwd, f32),
                                  {launch_attn_cross_bwd_bf16_d16, launch_attn_cross_bwd_bf16_d32, nullptr, nullptr, launch_attn_cross_bwd_bf16_d256},
                                  {launch_attn_cross_bwd_f16_d16, launch_attn_cross_bwd_f16_d32, nullptr, nullptr, launch_attn_cross_bwd_f16_d256}};

static int slot_of(int D) { return D == 16 ? 0 : (D == 32 ? 1 : (D == 64 ? 2 : (D == 128 ? 3 : (D == 256 ? 4 : -1)))); }
// An alpha whose 1 / (alpha - 1) is 1 in fp32 is 2 to the kernels: the generic ones raise u = 0 to the power 1 / (alpha - 1) - 1.
static int alpha_mode(double alpha) { return alpha == 1.5 ? ATT_15 : (alpha == 2.0 || (float)(1.0 / (alpha - 1.0)) == 1.f ? ATT_2 : ATT_GEN); }
static size_t align256(size_t x) { return (x + 255) / 256 * 256; }

struct Call {
  int B, Hq, Hkv, Nq, Nk, D, dtype;
  double alpha;
  // blocks of 32 x 32 scores, padding included
  long long blocks() const { return (long long)B * Hq * ((Nq + 31) / 32) * ((Nk + 31) / 32); }
};

// Which kernels serve a call.
enum Route {
  TILES,      // the tile kernels: other head dims, other alphas
  F32,        // 32 rows a workgroup, single precision, head dims 64 and 128 (16-bit key indices)
  ALL_PAIRS,  // 16 bits: the forward with resident scores, or on 32 rows a workgroup, the gradients on all pairs
  SUPPORTS,   // 16 bits: probe, the kernels on the supports, and those on all pairs for what they leave over
};
static bool supports_enabled() {  // (ADSP_SPARSE=0, as for the attention of a sequence to itself)
  const char* e = getenv("ADSP_SPARSE");
  return !(e && strcmp(e, "0") == 0);
}
// The kernels on the supports do less where scores are peaked and rows are long, but take five to eight launches and items of 128 rows; those on all pairs fill the chip with
// less.  The lines lie where the two meet for q of spread 1; us, on the supports -> all pairs, q of spread 1 and 3, alpha = 1.5, bf16 (queries x keys):
//   forward alone, up to 512 keys (always all pairs): 16 x 16 heads, 500 x 500, D = 64: 104 -> 58, 73 -> 54; 32 x 16, D = 128: 256 -> 205, 182 -> 198;
//     up to 1024: 16 x 16, 448 x 1000, D = 64: 130 -> 108, 93 -> 99; 1000 x 1000: 226 -> 229, 152 -> 210; 8 x 16/4, 448 x 1000, D = 128: 99 -> 86, 77 -> 83; 16 x 16/4: 157 -> 166, 115 -> 156;
//     up to 2048: 4 x 16, 448 x 1500, D = 64: 74 -> 69, 55 -> 64; 6 x 16: 95 -> 103, 70 -> 94; 4 x 8, D = 128: 82 -> 50, 66 -> 47; 4 x 16/4: 83 -> 94, 64 -> 88;
//     beyond (32 rows a workgroup): 2 x 16/4, 256 x 4000, D = 64: 104 -> 73, 71 -> 46; 4 x 16/4, 512 x 4000: 106 -> 151, 74 -> 98; 2 x 16, 512 x 4000, D = 128: 133 -> 89, 106 -> 62;
//     4 x 16/4: 130 -> 168, 105 -> 115; 4 x 32/8, 1024 x 5000: 381 -> 720, 293 -> 517;
//   a training step (before dQ's weights had two parts on all pairs, which costs a step 1 to 3 %), up to 512 keys: 16 x 16, 500 x 500, D = 64: 245 -> 164, 163 -> 159; 32 x 16, D = 128: 729 -> 701, 470 -> 695; 64 x 16, 2000 x 500, D = 64: 3170 -> 2186, 1807 -> 2129;
//     up to 1024: 16 x 16, 448 x 1000, D = 64: 347 -> 284, 248 -> 279; 1000 x 1000: 565 -> 567, 353 -> 549; 8 x 8, 448 x 1000, D = 128: 198 -> 174, 143 -> 173; 12 x 8: 252 -> 250, 177 -> 248;
//     up to 2048: 4 x 16, 448 x 1500, D = 64: 179 -> 147, 129 -> 142; 16 x 16: 418 -> 487, 295 -> 463; D = 128 (from kept lists): 4 x 8: 190 -> 116, 136 -> 81; 2 x 16/4: 199 -> 134, 124 -> 92;
//     beyond (from kept lists): 2 x 16/4, 256 x 4000, D = 64: 176 -> 115, 118 -> 88; 4 x 16: 512 x 4000: 296 -> 330, 229 -> 241; 4 x 16/4: 203 -> 320, 134 -> 228; D = 128: 2 x 16, 64 x 8000:
//     387 -> 166, 308 -> 138; 2 x 16, 512 x 4000: 266 -> 205, 192 -> 150; 4 x 16, 512 x 2500: 307 -> 275, 238 -> 202; 512 x 4000: 382 -> 381, 292 -> 284; 4 x 16/4: 260 -> 346, 179 -> 258.
static Route route_of(const Call& c, bool train) {
  if ((c.D != 64 && c.D != 128) || c.alpha < 1.125) return TILES;
  if (c.dtype == ADSP_F32) return c.Nk <= 65536 ? F32 : TILES;
  if (c.Nq > 65536 || c.Nk > 65536 || c.Nk <= 512 || !supports_enabled()) return ALL_PAIRS;  // (16-bit indices)
  const int at = c.Nk <= 1024 ? 0 : (c.Nk <= kResidentMaxKeys ? 1 : 2);
  static const int kForward[2][3] = {{180000, 50000, 80000}, {60000, 30000, 80000}}, kTrain[2][3] = {{180000, 80000, 80000}, {40000, 30000, 100000}};
  return c.blocks() <= (train ? kTrain : kForward)[c.D == 128][at] ? ALL_PAIRS : SUPPORTS;
}

// All pairs, 16 bits, forward: whether it is the one on 32 rows a workgroup (16-bit key indices), which keeps lists for the gradients.  Beyond the keys that fit registers, against 128 rows a
// workgroup: 4 x 32/8 heads, 1024 x 5000, D = 128: 720 us against 1026; 2 x 16, 32 x 8000: 124 against 597; flat scores, q of spread 1/8: 1602 against 672 and 274 against 367.  In training at
// D = 128 already beyond 1024 keys, for the gradients' sake; a step with resident scores and gradients on all pairs -> with lists, q of spread 1 and 3: 2 x 16/4, 448 x 1500: 213 -> 134, 210 -> 92;
// 8, 1000 x 1900: 130 -> 93, 129 -> 68; 4 x 16, 100 x 1000: 79, 78, 78 -> 59; D = 64: 2 x 8, 448 x 1500: 62, 71, 60 -> 53; 4 x 16, 100 x 2000: 75, 94, 73, 74.  (Flat scores pay for the walks:
// 2 x 16/4: 227, 242; 8 x 8, 125 x 1900: 132, 171; 4 x 16, 100 x 1100: 91, 120.)
static bool rows32_16bit(const Call& c, bool train) { return c.Nk <= 65536 && (c.Nk > kResidentMaxKeys || (train && c.D == 128 && c.Nk > 1024)); }

// Workspace of the kernels on the supports, forward and backward (see attn_probe.h for the control words), and what the forward keeps for the backward.
constexpr int kMaxSlots = 1024;                       // workgroups of the persistent kernels
constexpr size_t kSlotBytes = (size_t)4 * 1616 * 8;   // four waves x 1616 candidates x (score, key)
static long long row_blocks(const Call& c) { return (long long)c.B * c.Hq * mblocks_of(c.Nq); }
static int slots_of(long long items) { return (int)(items > kMaxSlots ? kMaxSlots : (items + 7) / 8 * 8); }
struct FwdSpace {
  size_t scales_off, flags_off, events_off, k8_off, total;
  int slots;
};
static FwdSpace fwd_space(const Call& c) {
  FwdSpace w = {};
  w.slots = slots_of(row_blocks(c));
  w.scales_off = 256 + ((size_t)c.B * c.Hkv + 1) * 8;
  w.flags_off = align256(w.scales_off + (size_t)c.B * c.Hkv * 16);
  w.events_off = align256(w.flags_off + (size_t)row_blocks(c) * 4);
  w.k8_off = align256(w.events_off + (size_t)w.slots * kSlotBytes);
  w.total = w.k8_off + (size_t)c.B * c.Hkv * npad_of(c.Nk) * c.D;
  return w;
}
struct Kept {
  size_t lens_off, tshift_off, streams_off, total;
};
static Kept kept_space(const Call& c) {
  Kept k = {};
  const size_t items = (size_t)row_blocks(c);
  k.lens_off = align256(items * 4);
  k.tshift_off = align256(k.lens_off + items * 4 * 2);
  k.streams_off = align256(k.tshift_off + (size_t)c.B * c.Hq * c.Nq * 4);
  k.total = k.streams_off + items * kSlotBytes;
  return k;
}
struct BwdSpace {
  size_t flags_off, events_off, queue2_off, kvflags_off, scratch_off, streams_off, dir_off, total;
  int slots, dir_stride;
};
static BwdSpace bwd_space(const Call& c) {
  BwdSpace w = {};
  const long long items = row_blocks(c), keys = (long long)c.B * c.Hkv * mblocks_of(c.Nk);
  w.slots = slots_of(items > keys ? items : keys);
  w.flags_off = align256(256 + ((size_t)c.B * c.Hkv + 1) * 8);
  w.events_off = align256(w.flags_off + (size_t)items * 4);
  w.queue2_off = align256(w.events_off + (size_t)w.slots * kSlotBytes);
  w.kvflags_off = align256(w.queue2_off + 256);
  w.scratch_off = align256(w.kvflags_off + (size_t)keys * 4);
  w.streams_off = align256(w.scratch_off + (size_t)w.slots * 4 * 32 * 2 * c.D * 4);
  w.dir_stride = (mblocks_of(c.Nk) * 4 + 2) / 2 * 2;
  w.dir_off = align256(w.streams_off + (size_t)items * kSlotBytes);
  w.total = w.dir_off + align256((size_t)items * 4 * w.dir_stride * 2);
  return w;
}

// The lists that a forward on 32 rows a workgroup keeps; not of up to 128 keys, of which most may be members (fp32, 1 x 8 heads, 40 x 57, D = 64, gradients with and without: 18.9 and 17.2 us,
// flat scores 35.6 and 17.4).  Beside them, two weights a member from the dQ kernel for that of dK and dV.  Of up to 32 keys, where the walk's kernel has one wave of four at work, dQ is
// formed from them where there are more row blocks than run at once, and dK and dV by their walk; a step without -> with, q of spread 1 and 1/8: 17 x 32/16, 969 x 3, D = 128: 1181 -> 646,
// 1165 -> 646; 969 x 32: 1251 -> 855, 1374 -> 1260; 4 x 8, 2100 x 10, D = 64: 87 -> 68, 90 -> 79; 2100 x 32: 94 -> 84, 108 -> 120.
static bool for_dq_only(const Call& c) { return c.Nk <= 128; }
static size_t lists_bytes(const Call& c, Route route) {
  if (route != F32 && !(route == ALL_PAIRS && rows32_16bit(c, true))) return 0;
  if (for_dq_only(c) && (c.Nk > 32 || (long long)c.B * c.Hq * ((c.Nq + 31) / 32) <= 512)) return 0;
  // (32-bit offsets inside a K/V head's rows)
  return (long long)(c.Hq / c.Hkv) * c.Nq < (1 << 21) ? kept_lists_bytes((size_t)c.B * c.Hq * c.Nq) : 0;
}
// Parts of the queries over which dK and dV are summed, where a launch has fewer than two blocks of 32 keys to a CU (16 bits, D = 128: than one, two waves to 64 keys do better from there on): as many as
// make twice that, of eight blocks of queries at least.  Gradients, us, one part -> this, fp32 and bf16: 4 heads, 2000 queries, 5 keys, D = 64: 77 -> 29, 32 -> 19; 4 x 8, 2000 x 10: 103 -> 55,
// 36 -> 23; 2000 x 100: 112 -> 91, 39 -> 37; 2 x 64/16, 2000 x 10, D = 128: 881 -> 515, 256 -> 123; beyond a block to a CU 17 x 32/16, 969 x 3: fp32 524 -> 456; bf16, 7 x 16/4, 250 x 500: 79, with parts 123.
static int q_parts_of(const Call& c, Route route) {
  if (route != F32 && !(route == ALL_PAIRS && c.dtype != ADSP_F32 && (c.D == 64 || c.D == 128))) return 1;
  const long long groups = (long long)c.B * c.Hkv * ((c.Nk + 31) / 32), steps = (long long)(c.Hq / c.Hkv) * ((c.Nq + 31) / 32);
  const int few = c.dtype == ADSP_F32 || c.D == 64 ? 512 : 256;
  if (groups >= few) return 1;
  const long long most = steps / 8, want = (2 * few - 1 + groups) / groups;
  return (int)(want < most ? want : (most < 1 ? 1 : most));
}
static size_t q_parts_bytes(const Call& c, Route route) {
  const int parts = q_parts_of(c, route);
  return parts > 1 ? (size_t)parts * 2 * c.B * c.Hkv * c.Nk * c.D * 4 : 0;
}
// their sums, in the order of the parts: a thread has four values of dK or dV
template <typename T> __global__ __launch_bounds__(256) void sum_parts_kernel(AttnBwdCrossParams p, int D) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  const size_t rows = (size_t)p.B * p.Hkv * p.Nk, pieces = rows * D / 4, id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= 2 * pieces) return;
  const f32x4* const from = reinterpret_cast<const f32x4*>(p.q_part_rows) + id;
  f32x4 s = from[0];
  for (int i = 1; i < p.q_parts; ++i) s += from[(size_t)i * 2 * pieces];
  void* const to = id < pieces ? p.dk : p.dv;
  const size_t at = id < pieces ? id : id - pieces;
  if constexpr (elem_traits<T>::kBytes == 4) reinterpret_cast<f32x4*>(to)[at] = s;
  else reinterpret_cast<uint2*>(to)[at] = uint2{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])};
}
static void sum_parts(const AttnBwdCrossParams& p, int D, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)(((size_t)p.B * p.Hkv * p.Nk * D / 2 + 255) / 256));
  if (dtype == ADSP_F32) hipLaunchKernelGGL((sum_parts_kernel<float>), grid, dim3(256), 0, s, p, D);
  else if (dtype == ADSP_BF16) hipLaunchKernelGGL((sum_parts_kernel<bf16_t>), grid, dim3(256), 0, s, p, D);
  else hipLaunchKernelGGL((sum_parts_kernel<f16_t>), grid, dim3(256), 0, s, p, D);
}
static size_t pairs_bytes(const Call& c) { return (size_t)c.B * c.Hq * c.Nq * kKeptMembers * 8; }

static int check(const Call& c, const void* vq, int vq_bits, const void* vk, int vk_bits) {
  if (c.dtype != ADSP_F32 && c.dtype != ADSP_BF16 && c.dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  if (c.B <= 0 || c.Hq <= 0 || c.Hkv <= 0 || c.Nq <= 0 || c.Nk <= 0 || c.Hq % c.Hkv != 0 || slot_of(c.D) < 0) return ADSP_ERR_SHAPE;
  constexpr int kMost = kMaskWords * 32 * kBN;
  if (c.Nq > kMost || c.Nk > kMost) return ADSP_ERR_SHAPE;
  // (workgroups of 32 rows, a launch's number of them)
  if ((long long)c.B * c.Hq * ((c.Nq + 31) / 32 + (c.Nk + 31) / 32) >= (1ll << 30)) return ADSP_ERR_SHAPE;
  if (!(c.alpha > 1.0) || c.alpha > 2.0) return ADSP_ERR_UNSUPPORTED;
  if ((vq && vq_bits != 32 && vq_bits != 64) || (vk && vk_bits != 32 && vk_bits != 64)) return ADSP_ERR_UNSUPPORTED;
  return ADSP_OK;
}
static bool valid(const Call& c) { return check(c, nullptr, 0, nullptr, 0) == ADSP_OK; }
// What forward, backward and probe share.
template <typename P> static void fill(P& p, const Call& c, const void* varlen_q, int varlen_q_bits, const void* varlen_k, int varlen_k_bits) {
  p.varlen = varlen_q;
  p.varlen_bits = varlen_q_bits;
  p.varlen_k = varlen_k;
  p.varlen_k_bits = varlen_k_bits;
  p.B = c.B;
  p.Hq = c.Hq;
  p.Hkv = c.Hkv;
  p.N = c.Nq;
  p.Nk = c.Nk;
  p.Npad = npad_of(c.Nk);
  p.n_mblk = mblocks_of(c.Nq);
  p.mask_words = mask_words_of(c.Nk);
  p.c0 = (float)(1.0 / (c.alpha - 1.0));
  p.qscale = (float)((c.alpha - 1.0) / sqrt((double)c.D));
}
static bool space_ok(const void* p, size_t have, size_t need) { return need == 0 || (p && have >= need && ((uintptr_t)p & 15) == 0); }
constexpr float kProbeMaxSupport = 28.f;  // as for the attention of a sequence to itself
}  // namespace cross
}  // namespace adsp

extern "C" size_t adsp_attn_cross_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, int train) {
  using namespace adsp::cross;
  const Call c{B, Hq, Hkv, Nq, Nk, D, dtype, alpha};
  return valid(c) && route_of(c, train != 0) == SUPPORTS ? fwd_space(c).total : 0;
}
extern "C" size_t adsp_attn_cross_supports_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha) {
  using namespace adsp::cross;
  const Call c{B, Hq, Hkv, Nq, Nk, D, dtype, alpha};
  if (!valid(c)) return 0;
  const Route route = route_of(c, true);
  return route == SUPPORTS ? kept_space(c).total : lists_bytes(c, route);
}
extern "C" size_t adsp_attn_cross_bwd_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, int kept) {
  using namespace adsp::cross;
  const Call c{B, Hq, Hkv, Nq, Nk, D, dtype, alpha};
  if (!valid(c)) return 0;
  const Route route = route_of(c, true);
  return route == SUPPORTS ? bwd_space(c).total : (kept && lists_bytes(c, route) && !for_dq_only(c) ? pairs_bytes(c) : q_parts_bytes(c, route));
}

extern "C" int adsp_attn_cross_fwd(const void* q, const void* k, const void* v, void* out, float* taus, const void* varlen_q, int varlen_q_bits,
                                   const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha,
                                   void* workspace, size_t workspace_bytes, void* supports, size_t supports_bytes, void* stream) {
  using namespace adsp;
  if (!q || !k || !v || !out) return ADSP_ERR_NULL;
  const cross::Call c{B, Hq, Hkv, Nq, Nk, D, dtype, alpha};
  const int rc = cross::check(c, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  if (rc != ADSP_OK) return rc;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) != 0) return ADSP_ERR_ALIGN;
  const cross::Route route = cross::route_of(c, taus != nullptr);
  AttnCrossParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.taus = taus;
  cross::fill(p, c, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  p.niter = 11;  // (of the tile kernel's steps as many as the block-mask variant takes; the others iterate to convergence)
  p.alpha = (float)alpha;
  const int am = cross::alpha_mode(alpha), slot = cross::slot_of(D);
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  if (const size_t need = taus && supports ? cross::lists_bytes(c, route) : 0) {
    if (!cross::space_ok(supports, supports_bytes, need)) return ADSP_ERR_WORKSPACE;
    p.save_streams = (unsigned char*)supports;
  }
  int st;
  if (route == cross::TILES) {
    st = cross::kFwd[dtype][slot](p, am, s);
  } else if (route == cross::F32) {
    st = D == 64 ? launch_attn_cross_f32_fwd_d64(p, am, s) : launch_attn_cross_f32_fwd_d128(p, am, s);
  } else if (route == cross::ALL_PAIRS) {
    if (cross::rows32_16bit(c, taus != nullptr)) st = ADSP_CALL_16(launch_attn_cross_rows32_fwd, D, dtype, p, am, s);
    else if (Nk <= kResidentMaxKeys) st = ADSP_CALL_16(launch_attn_cross16_fwd, D, dtype, p, am, true, s);
    else st = ADSP_CALL_16(launch_attn_cross16_fwd, D, dtype, p, am, false, s);
  } else {
    const cross::FwdSpace w = cross::fwd_space(c);
    if (!cross::space_ok(workspace, workspace_bytes, w.total)) return ADSP_ERR_WORKSPACE;
    if (supports && !cross::space_ok(supports, supports_bytes, cross::kept_space(c).total)) return ADSP_ERR_WORKSPACE;
    unsigned char* const ws = (unsigned char*)workspace;
    p.queue = (uint32_t*)ws;
    p.hints = p.queue + 64;
    p.w1_scales = (float*)(ws + w.scales_off);
    p.block_flags = (int32_t*)(ws + w.flags_off);
    p.events = ws + w.events_off;
    p.k8 = ws + w.k8_off;
    p.probe_max_support = cross::kProbeMaxSupport;
    if (supports) {
      const cross::Kept kept = cross::kept_space(c);
      unsigned char* const sp = (unsigned char*)supports;
      p.save_flags = (int32_t*)sp;
      p.save_lens = (uint16_t*)(sp + kept.lens_off);
      p.save_tshift = (float*)(sp + kept.tshift_off);
      p.save_streams = sp + kept.streams_off;
    }
    launch_probe<true, true>(p, D, dtype, am, nullptr, nullptr, s);
    st = ADSP_CALL_16(launch_attn_cross_sparse_fwd, D, dtype, p, am, w.slots, s);
    if (st == 0) st = ADSP_CALL_16(launch_attn_cross16_fwd, D, dtype, p, am, false, s);  // (what it left over)
  }
  return st == 0 && hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}

extern "C" int adsp_attn_cross_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus, const void* varlen_q,
                                   int varlen_q_bits, const void* varlen_k, int varlen_k_bits, void* dq, void* dk, void* dv, float* delta, float* zinv,
                                   int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, void* workspace, size_t workspace_bytes,
                                   const void* supports, size_t supports_bytes, void* stream) {
  using namespace adsp;
  if (!q || !k || !v || !dout || !taus || !dq || !dk || !dv || !delta || !zinv) return ADSP_ERR_NULL;
  const cross::Call c{B, Hq, Hkv, Nq, Nk, D, dtype, alpha};
  const int rc = cross::check(c, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  if (rc != ADSP_OK) return rc;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) != 0) return ADSP_ERR_ALIGN;
  const cross::Route route = cross::route_of(c, true);
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
  cross::fill(p, c, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
  p.sm_scale = (float)(1.0 / sqrt((double)D));
  const int am = cross::alpha_mode(alpha);
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  const size_t lists = supports ? cross::lists_bytes(c, route) : 0;
  const bool pairs = lists && !cross::for_dq_only(c);
  // What a forward kept lies as its route has it, which ADSP_SPARSE may have changed since: a buffer of another size than this route's is of another layout.
  if (supports && supports_bytes != (route == cross::SUPPORTS ? cross::kept_space(c).total : lists)) return ADSP_ERR_WORKSPACE;
  if (lists) {
    if (!cross::space_ok(supports, supports_bytes, lists) || (pairs && !cross::space_ok(workspace, workspace_bytes, cross::pairs_bytes(c)))) return ADSP_ERR_WORKSPACE;
    p.fwd_streams = (const unsigned char*)supports;
    if (pairs) p.streams = (unsigned char*)workspace;
  }
  p.q_parts = 1;
  if (const size_t need = pairs ? 0 : cross::q_parts_bytes(c, route)) {
    if (!cross::space_ok(workspace, workspace_bytes, need)) return ADSP_ERR_WORKSPACE;
    p.q_parts = cross::q_parts_of(c, route);
    p.q_part_rows = (float*)workspace;
  }
  int st;
  if (route == cross::SUPPORTS) {
    const cross::BwdSpace w = cross::bwd_space(c);
    if (!cross::space_ok(workspace, workspace_bytes, w.total)) return ADSP_ERR_WORKSPACE;
    if (supports && !cross::space_ok(supports, supports_bytes, cross::kept_space(c).total)) return ADSP_ERR_WORKSPACE;
    unsigned char* const ws = (unsigned char*)workspace;
    p.queue = (uint32_t*)ws;
    p.hints = p.queue + 64;
    p.block_flags = (int32_t*)(ws + w.flags_off);
    p.events = ws + w.events_off;
    p.streams = ws + w.streams_off;
    p.stream_dir = (uint16_t*)(ws + w.dir_off);
    p.dir_stride = w.dir_stride;
    if (supports) {
      const cross::Kept kept = cross::kept_space(c);
      const unsigned char* const sp = (const unsigned char*)supports;
      p.fwd_flags = (const int32_t*)sp;
      p.fwd_lens = (const uint16_t*)(sp + kept.lens_off);
      p.fwd_tshift = (const float*)(sp + kept.tshift_off);
      p.fwd_streams = sp + kept.streams_off;
    }
    AttnCrossParams pp = {};  // what the probe reads, and the control words that it clears
    pp.q = q;
    pp.k = k;
    cross::fill(pp, c, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits);
    pp.queue = p.queue;
    pp.hints = p.hints;
    pp.probe_max_support = cross::kProbeMaxSupport;
    uint32_t* const queue2 = (uint32_t*)(ws + w.queue2_off);
    int32_t* const kv_flags = (int32_t*)(ws + w.kvflags_off);
    launch_probe<false, true>(pp, D, dtype, am, queue2, kv_flags, s);
    st = ADSP_CALL_16(launch_attn_cross_sparse_bwd, D, dtype, p, am, 0, w.slots, s);
    if (st == 0) st = ADSP_CALL_16(launch_attn_cross16_bwd, D, dtype, p, am, 1, s);
    p.queue2 = queue2;
    p.kv_flags = kv_flags;
    p.part_scratch = (float*)(ws + w.scratch_off);
    if (st == 0) st = ADSP_CALL_16(launch_attn_cross_sparse_bwd, D, dtype, p, am, 2, w.slots, s);
    if (st == 0) st = ADSP_CALL_16(launch_attn_cross16_bwd, D, dtype, p, am, 2, s);
  } else if (route == cross::F32) {
    st = D == 64 ? launch_attn_cross_f32_bwd_d64(p, am, s) : launch_attn_cross_f32_bwd_d128(p, am, s);
  } else if (dtype != ADSP_F32 && (D == 64 || D == 128)) {
    st = lists ? ADSP_CALL_16(launch_attn_cross_lists_dq, D, dtype, p, am, s) : 0;
    if (st == 0) st = ADSP_CALL_16(launch_attn_cross16_bwd, D, dtype, p, am, lists ? 1 : 3, s);
    if (st == 0 && lists) st = ADSP_CALL_16(launch_attn_cross_lists_dkdv, D, dtype, p, s);
    if (st == 0 && lists) st = ADSP_CALL_16(launch_attn_cross16_bwd, D, dtype, p, am, 2, s);
  } else {
    st = cross::kBwd[dtype][cross::slot_of(D)](p, am, s);
  }
  if (st == 0 && p.q_parts > 1) cross::sum_parts(p, D, dtype, s);
  return st == 0 && hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
