// Positions of queries and keys: the C entry points, how a call is shared out, and the sums behind the weights' gradients.
#include <algorithm>

#include "../../include/adasplash_hip.h"
#include "rotary.h"

namespace adsp {
namespace rotary {
constexpr int kLimit = 0x7fff0000;  // tokens of a call: with a workgroup's more they stay below 2^31
constexpr int64_t kElements = (int64_t)(0xffffffffu / kThreads) * kThreads * 8;  // and of one head: a launch has fewer than 2^32 threads along an axis, eight elements to each

struct SumParams {
  const float* partial[2];
  void* out[2];
  int rows[2], f32[2], D;
};
// The partial rows of a weight's gradient added up, always in the same order: a workgroup has 16 columns and 64 sums of each, four rows under way at a time.  us for 1368
// and 342 rows of 128 (4 x 8192 tokens, 32/8 heads): 7.0; sixteen sums, a row at a time, 36.
constexpr int kSums = 64;
template <typename T> __global__ __launch_bounds__(16 * kSums) void rotary_weights_kernel(SumParams p) {
  __shared__ float sums[kSums][17];
  const int which = blockIdx.y, col = threadIdx.x % 16, row0 = threadIdx.x / 16, d = blockIdx.x * 16 + col, rows = p.rows[which];
  if (!p.out[which]) return;
  const float* const from = p.partial[which] + d;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r = row0; r < rows; r += 4 * kSums) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = r + u * kSums < rows ? from[(size_t)(r + u * kSums) * p.D] : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) sum[u] += x[u];
  }
  sums[row0][col] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (row0 > 0) return;
  float all = 0.f;
  for (int i = 0; i < kSums; ++i) all += sums[i][col];
  if (p.f32[which]) {
    ((float*)p.out[which])[d] = all;
  } else {
    const uint32_t bits = pack2<T>(all, all);
    ((uint16_t*)p.out[which])[d] = (uint16_t)bits;
  }
}

// Workgroups: `per` heads each, as many as still leave the chip four workgroups a CU; with gradients some eight a CU in all, each with several steps of tokens (and one partial row of
// the weights' gradients).
static void share_out(Params& p, int D, bool gradients) {
  const int in_block = kThreads * 8 / D, all = (int)((p.tokens + in_block - 1) / in_block);
  p.per = 8;
  auto blocks = [&](int heads) { return (heads + p.per - 1) / p.per; };
  while (p.per > 1 && (long long)all * (blocks(p.of[0].heads) + blocks(p.of[1].heads)) < 1024) p.per /= 2;
  for (Rows& r : p.of) r.blocks = blocks(r.heads);
  const int most = gradients ? std::max(1, 2048 / (p.of[0].blocks + p.of[1].blocks)) : all;
  p.token_steps = (all + most - 1) / most;
  p.token_blocks = (all + p.token_steps - 1) / p.token_steps;
}
static int describe(Params& p, const void* positions, int positions_bits, int64_t pos_b, int64_t pos_n, const double* frequencies, int64_t B, int Hq, int Hkv, int64_t N, int D,
                    int rot, float eps, float factor, int dtype) {
  if (!positions || (rot > 0 && !frequencies)) return ADSP_ERR_NULL;
  if (dtype != ADSP_F32 && dtype != ADSP_BF16 && dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256) return ADSP_ERR_SHAPE;
  if (B <= 0 || N <= 0 || B > kLimit || N > kLimit || B * N > kLimit || Hq < 0 || Hkv < 0 || Hq + Hkv <= 0 || Hq > 65535 - Hkv) return ADSP_ERR_SHAPE;
  if (B * N > kElements / D || rot < 0 || rot > D || rot % 8 != 0) return ADSP_ERR_SHAPE;
  if (positions_bits != 32 && positions_bits != 64) return ADSP_ERR_UNSUPPORTED;
  p.positions = positions;
  p.pos_bits = positions_bits;
  p.pos_b = pos_b;
  p.pos_n = pos_n;
  p.frequencies = frequencies;
  p.tokens = (uint32_t)(B * N);
  p.N = (uint32_t)N;
  p.of[0].heads = Hq;
  p.of[1].heads = Hkv;
  p.rot = rot;
  p.eps = eps;
  p.factor = factor;
  p.inv_d = 1.f / (float)D;
  return ADSP_OK;
}
static bool aligned(std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* x : pointers) all |= (uintptr_t)x;
  return (all & 15) == 0;
}
static bool aligned_strides(const int64_t* strides, int n, int dtype) {
  int64_t all = 0;
  for (int i = 0; i < n; ++i) all |= strides[i] * (dtype == ADSP_F32 ? 4 : 2);
  return (all & 15) == 0;
}
static void run(const Params& p, int D, int layout, int mode, int dtype, hipStream_t s) {
  if (dtype == ADSP_F32) launch<float>(p, D, layout == ADSP_ROTARY_HALF, mode, s);
  else if (dtype == ADSP_BF16) launch<bf16_t>(p, D, layout == ADSP_ROTARY_HALF, mode, s);
  else launch<f16_t>(p, D, layout == ADSP_ROTARY_HALF, mode, s);
}
static bool known(int layout) { return layout == ADSP_ROTARY_HALF || layout == ADSP_ROTARY_INTERLEAVED; }
static int set_weight(Params& p, int which, const void* weight, int weight_dtype, int dtype) {
  if (weight && weight_dtype != dtype && weight_dtype != ADSP_F32) return ADSP_ERR_DTYPE;
  p.of[which].weight = weight;
  p.weight_f32[which] = weight_dtype == ADSP_F32;
  return ADSP_OK;
}
}  // namespace rotary
}  // namespace adsp

extern "C" int adsp_rotary_fwd(const void* q, const void* k, void* q_out, void* k_out, const void* positions, int positions_bits, int64_t positions_stride_b,
                               int64_t positions_stride_n, const double* frequencies, const void* q_weight, int q_weight_dtype, const void* k_weight, int k_weight_dtype, int B,
                               int Hq, int Hkv, int N, int D, int rotary_dim, int layout, const int64_t* strides, float eps, float factor, int dtype, void* stream) {
  using namespace adsp::rotary;
  Params p = {};
  int rc = describe(p, positions, positions_bits, positions_stride_b, positions_stride_n, frequencies, B, Hq, Hkv, N, D, rotary_dim, eps, factor, dtype);
  if (rc != ADSP_OK) return rc;
  if (!known(layout)) return ADSP_ERR_UNSUPPORTED;
  if ((Hq > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !k_out)) || !strides) return ADSP_ERR_NULL;
  if (!aligned({q, k, q_out, k_out, q_weight, k_weight}) || !aligned_strides(strides, 12, dtype)) return ADSP_ERR_ALIGN;
  for (int i = 0; i < 2; ++i) {
    rc = set_weight(p, i, i ? k_weight : q_weight, i ? k_weight_dtype : q_weight_dtype, dtype);
    if (rc != ADSP_OK) return rc;
    Rows& r = p.of[i];
    r.x = i ? k : q;
    r.y = i ? k_out : q_out;
    r.x_b = strides[3 * i], r.x_h = strides[3 * i + 1], r.x_n = strides[3 * i + 2];
    r.y_b = strides[6 + 3 * i], r.y_h = strides[7 + 3 * i], r.y_n = strides[8 + 3 * i];
  }
  share_out(p, D, false);
  (void)hipGetLastError();
  run(p, D, layout, 0, dtype, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}

extern "C" size_t adsp_rotary_bwd_workspace_bytes(int B, int Hq, int Hkv, int N, int D) {
  using namespace adsp::rotary;
  if (B <= 0 || N <= 0 || (int64_t)B * N > kLimit || Hq < 0 || Hkv < 0 || Hq + Hkv <= 0 || D < 16 || D > 256) return 0;
  Params p = {};
  p.tokens = (uint32_t)((int64_t)B * N);
  p.of[0].heads = Hq;
  p.of[1].heads = Hkv;
  share_out(p, D, true);
  return (size_t)p.token_blocks * (p.of[0].blocks + p.of[1].blocks) * D * sizeof(float);
}

extern "C" int adsp_rotary_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq, void* dk, const void* positions, int positions_bits,
                               int64_t positions_stride_b, int64_t positions_stride_n, const double* frequencies, const void* q_weight, int q_weight_dtype,
                               const void* k_weight, int k_weight_dtype, void* dq_weight, void* dk_weight, int B, int Hq, int Hkv, int N, int D, int rotary_dim, int layout,
                               const int64_t* strides, float eps, float factor, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace adsp::rotary;
  Params p = {};
  int rc = describe(p, positions, positions_bits, positions_stride_b, positions_stride_n, frequencies, B, Hq, Hkv, N, D, rotary_dim, eps, factor, dtype);
  if (rc != ADSP_OK) return rc;
  if (!known(layout)) return ADSP_ERR_UNSUPPORTED;
  if ((Hq > 0 && (!dq_out || !dq)) || (Hkv > 0 && (!dk_out || !dk)) || !strides) return ADSP_ERR_NULL;
  if ((q_weight && Hq > 0 && (!q || !dq_weight)) || (k_weight && Hkv > 0 && (!k || !dk_weight))) return ADSP_ERR_NULL;
  if (!aligned({q, k, dq_out, dk_out, dq, dk, q_weight, k_weight, workspace}) || !aligned_strides(strides, 18, dtype)) return ADSP_ERR_ALIGN;
  const bool weights = (q_weight && Hq > 0) || (k_weight && Hkv > 0);
  if (weights && (!workspace || workspace_bytes < adsp_rotary_bwd_workspace_bytes(B, Hq, Hkv, N, D))) return ADSP_ERR_WORKSPACE;
  for (int i = 0; i < 2; ++i) {
    rc = set_weight(p, i, i ? k_weight : q_weight, i ? k_weight_dtype : q_weight_dtype, dtype);
    if (rc != ADSP_OK) return rc;
    Rows& r = p.of[i];
    r.x = i ? k : q;
    r.dy = i ? dk_out : dq_out;
    r.y = i ? dk : dq;
    r.x_b = strides[3 * i], r.x_h = strides[3 * i + 1], r.x_n = strides[3 * i + 2];
    r.dy_b = strides[6 + 3 * i], r.dy_h = strides[7 + 3 * i], r.dy_n = strides[8 + 3 * i];
    r.y_b = strides[12 + 3 * i], r.y_h = strides[13 + 3 * i], r.y_n = strides[14 + 3 * i];
  }
  share_out(p, D, true);
  p.of[0].partial = (float*)workspace;
  p.of[1].partial = (float*)workspace + (size_t)p.token_blocks * p.of[0].blocks * D;
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  run(p, D, layout, 2, dtype, s);
  if (weights) {
    SumParams sp = {};
    for (int i = 0; i < 2; ++i) {
      sp.partial[i] = p.of[i].partial;
      sp.out[i] = p.of[i].weight && p.of[i].heads > 0 ? (i ? dk_weight : dq_weight) : nullptr;
      sp.rows[i] = p.token_blocks * p.of[i].blocks;
      sp.f32[i] = p.weight_f32[i];
    }
    sp.D = D;
    const dim3 grid((unsigned)(D / 16), 2), block(16 * kSums);
    if (dtype == ADSP_F16) hipLaunchKernelGGL(rotary_weights_kernel<adsp::f16_t>, grid, block, 0, s, sp);
    else hipLaunchKernelGGL(rotary_weights_kernel<adsp::bf16_t>, grid, block, 0, s, sp);
  }
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}

extern "C" int adsp_paged_write_rotary(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots, const void* positions, int positions_bits,
                                       int64_t positions_stride, const double* frequencies, const void* k_weight, int k_weight_dtype, int64_t tokens, int heads, int D,
                                       int rotary_dim, int layout, int64_t pages, int page_size, const int64_t* strides, float eps, float factor, int dtype, void* stream) {
  using namespace adsp::rotary;
  Params p = {};
  int rc = describe(p, positions, positions_bits, 0, positions_stride, frequencies, 1, 0, heads, tokens, D, rotary_dim, eps, factor, dtype);
  if (rc != ADSP_OK) return rc;
  if (!known(layout)) return ADSP_ERR_UNSUPPORTED;
  if (!k || !v || !k_pages || !v_pages || !slots || !strides) return ADSP_ERR_NULL;
  if (heads <= 0 || pages <= 0 || page_size <= 0) return ADSP_ERR_SHAPE;
  if (!aligned({k, v, k_pages, v_pages, k_weight}) || !aligned_strides(strides, 10, dtype)) return ADSP_ERR_ALIGN;
  rc = set_weight(p, 1, k_weight, k_weight_dtype, dtype);
  if (rc != ADSP_OK) return rc;
  const int64_t es = dtype == ADSP_F32 ? 4 : 2;
  Rows& r = p.of[1];
  r.x = k;
  r.y = k_pages;
  r.x_n = strides[0], r.x_h = strides[1];
  p.pages.slots = (const long long*)slots;
  p.pages.v = (const char*)v;
  p.pages.v_pages = (char*)v_pages;
  p.pages.v_st = strides[2] * es, p.pages.v_sh = strides[3] * es;
  p.pages.k_sp = strides[4] * es, p.pages.k_sph = strides[5] * es, p.pages.k_sps = strides[6] * es;
  p.pages.v_sp = strides[7] * es, p.pages.v_sph = strides[8] * es, p.pages.v_sps = strides[9] * es;
  p.pages.n_slots = (long long)pages * page_size;
  p.pages.page = page_size;
  share_out(p, D, false);
  (void)hipGetLastError();
  run(p, D, layout, 1, dtype, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
