// What runs in front of the kernels on the supports (16-bit types, head dims 64 and 128): the probe of a K/V head's scores, and
// the e4m3 copy of K that the forward's first walk reads.
#pragma once
#include "attn_two_lengths.h"
#include "../../include/adasplash_hip.h"

namespace adsp {

// e4m3 copy of K for the first walk of the sparse-support forward: [B * Hkv][Npad][D] bytes in the order of K, values
// beyond the format's range saturated, rows from N on zero.  The values are multiplied by the head's power of two first
// (`ak`, from the probe) and lie on the first walk's grid of 1/16 (see attn_sparse_kernel.h).
// A thread converts 16 values at a time: element `id` of the head's rows.
template <typename T, int D>
struct K8Copy {
  const u32x4* src;  // the head's rows, 8 values a piece
  u32x4* dst;
  long long rows, n;  // of K; of the copy: whole tiles of the sequence's length
  u32x4 lo, hi;
  __device__ K8Copy(const uint16_t* k, unsigned char* k8, size_t head, int N, int Npad, int L)
      : src(reinterpret_cast<const u32x4*>(k + head * (size_t)N * D)), dst(reinterpret_cast<u32x4*>(k8 + head * (size_t)Npad * D)),
        rows((long long)N * (D / 16)), n((long long)((L + kBN - 1) / kBN * kBN) * (D / 16)) {}
  __device__ void load(long long id) {
    lo = hi = u32x4{0u, 0u, 0u, 0u};
    if (id < n && id < rows) {
      lo = src[2 * id];
      hi = src[2 * id + 1];
    }
  }
  __device__ void store(long long id, float ak) const {
    if (id >= n) return;
    auto on_grid = [ak](float x) { return (x * ak + 786432.f) - 786432.f; };
    u32x4 out;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      out[e >> 1] = cvt_e4m3_pair(on_grid(unpack_lo<T>(lo[e + 1])), on_grid(unpack_hi<T>(lo[e + 1])), cvt_e4m3_pair(on_grid(unpack_lo<T>(lo[e])), on_grid(unpack_hi<T>(lo[e])), 0u, false), true);
      out[2 + (e >> 1)] = cvt_e4m3_pair(on_grid(unpack_lo<T>(hi[e + 1])), on_grid(unpack_hi<T>(hi[e + 1])), cvt_e4m3_pair(on_grid(unpack_lo<T>(hi[e])), on_grid(unpack_hi<T>(hi[e])), 0u, false), true);
    }
    dst[id] = out;
  }
};

// The copy by itself, behind the probe: a thread to 16 values.  Heads the probe has marked as dense are skipped.
template <typename T, int D, bool kCross = false>
__global__ __launch_bounds__(256) void k8_layout_kernel(FwdParams<kCross> p) {
  const int u = blockIdx.y;
  const int NK = key_rows<kCross>(p), L = key_length<kCross>(p, u / p.Hkv, NK);
  if (p.hints[2 * u] >= (1u << 20)) return;
  K8Copy<T, D> copy(reinterpret_cast<const uint16_t*>(p.k), const_cast<unsigned char*>(p.k8), (size_t)u, NK, p.Npad, L);
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  copy.load(id);
  copy.store(id, p.w1_scales[4 * u + 1]);
}

static int npad_of(int N) { return (N + kBN - 1) / kBN * kBN; }
static int mblocks_of(int N) { return (N + kMaskRows - 1) / kMaskRows; }
static int mask_words_of(int N) { return ((N + kBN - 1) / kBN + 31) / 32; }

// Control words of the sparse-support forward (the `queue` pointer of AttnParams): eight work counters, the number
// of row blocks it left to the dense kernel, a word saying that the probe below leaves every K/V head to the dense
// kernel; from word 64 on two words per K/V head and two more (the first of a head's pair is 1 << 20 when the probe
// leaves the whole head to the dense kernel; the backward's kernels keep row-block counters in the others), then four
// floats per K/V head (AttnParams::w1_scales).
//
// attn_probe_kernel clears them and looks at a sample of each K/V head's scores (one workgroup per head: four long
// query rows of the group's first head against 256 evenly spaced keys): from the sample's variance the support a
// Gaussian score distribution would have for a row that sees n keys follows in closed form (n s^2 g(a) = 1 with
// g(a) = (1 + a^2) Q(a) - a phi(a) for alpha = 1.5, n s h(a) = 1 with h(a) = phi(a) - a Q(a) for alpha = 2; support
// n Q(a)).  It grows with n: the probe stores the largest n whose predicted support the candidate lists hold, and the
// sparse-support kernels leave the row blocks that see more keys to the dense kernels without spending a walk on
// them.  The prediction only decides which kernel does the work (a row block it gets wrong is caught by the kernel's
// own checks), and it depends on the inputs alone: the same call takes the same way every time.
//
// What bounds it is latency, one workgroup per K/V head in front of the real work: the sampled keys' rows and the query rows are
// all under way at once, and the length whose predicted support just fits comes from the support point instead
// of the other way round -- a lane takes an a, n(a) = 1 / (mass above a per key) and support n(a) Q(a) are closed forms that
// grow with a, and a second look between the two neighbouring lanes refines it (bisecting a for 64 lengths
// took 14 rounds, each an integral of 32 terms at a generic alpha).  192 heads, D = 64: 10.7 -> 6.7 us a launch.
//
// (all 256 threads; `first`: writes what it finds; `share` as in the kernel below, written by thread 0)
template <typename T, int D, bool kCross>
__device__ __forceinline__ void probe_head(const FwdParams<kCross>& p, int am, int u, int L, int LQ, bool first, float* share) {
  __shared__ float red[4][2][4];
  __shared__ float ksum[4];
  const int tid = threadIdx.x;
  const int b = u / p.Hkv, kvh = u % p.Hkv, group = p.Hq / p.Hkv;
  if (L < 256 || (kCross && LQ == 0)) return;  // short sequences: finding out in the kernel costs little
  // Lanes side by side read a row's pieces of 16 bytes, so a load is whole lines; the sums over a row's lanes leave each lane with one
  // key's scores.  (A row to a lane made each load 64 lines, which several workgroups on a CU pay for one after another: 64 heads, D = 128, 11.7 -> 9.4 us a launch; with the copy of 32 workgroups a head 6 us less.)
  constexpr int P = D / 8;  // pieces of a row, and loads of 64 / P rows a wave
  const int lane = tid & 63, piece = lane % P;
  const int last_row = L - 1 - 3 * (L / 16);
  const int span = (is_causal<kCross>(p) ? last_row + 1 : L);
  const u32x4* kg = reinterpret_cast<const u32x4*>(p.k) + (size_t)(b * p.Hkv + kvh) * key_rows<kCross>(p) * P + piece;
  u32x4 kw[P], qw[4];
#pragma unroll
  for (int i = 0; i < P; ++i) kw[i] = kg[(size_t)(((long long)((tid & ~63) + i * (64 / P) + lane / P) * span) / 256) * P];
  const u32x4* qg = reinterpret_cast<const u32x4*>(p.q) + (size_t)(b * p.Hq + kvh * group) * p.N * P + piece;
#pragma unroll
  for (int j = 0; j < 4; ++j) qw[j] = qg[(size_t)(LQ - 1 - j * (LQ / 16)) * P];
  float dot[P][4];
  float ksq = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) dot[i][j] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = unpack_lo<T>(kw[i][e]), hi = unpack_hi<T>(kw[i][e]);
      ksq = fmaf(lo, lo, fmaf(hi, hi, ksq));
#pragma unroll
      for (int j = 0; j < 4; ++j) dot[i][j] = fmaf(lo, unpack_lo<T>(qw[j][e]), fmaf(hi, unpack_hi<T>(qw[j][e]), dot[i][j]));
    }
  }
#pragma unroll
  for (int h = P / 2; h > 0; h >>= 1) {
    const bool upper = (lane & h) != 0;
#pragma unroll
    for (int i = 0; i < h; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float keep = upper ? dot[i + h][j] : dot[i][j], give = upper ? dot[i][j] : dot[i + h][j];
        dot[i][j] = keep + __shfl_xor(give, h, 64);
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float z = dot[0][j] * p.qscale;
    const float s1 = wave_sum(z), s2 = wave_sum(z * z);
    if (lane == 0) {
      red[tid >> 6][0][j] = s1;
      red[tid >> 6][1][j] = s2;
    }
  }
  {
    const float ks = wave_sum(ksq);
    if (lane == 0) ksum[tid >> 6] = ks;
  }
  __syncthreads();
  if (tid == 0 && p.w1_scales) {
    // Scales of the first walk's operands: the sampled raw scores' root mean square goes to about 8 (the walk's
    // tags hold scores up to 512), shared between q and k so that k's own root mean square comes near 8 / sqrt(D).
    float raw2 = 0.f;
    for (int j = 0; j < 4; ++j) raw2 += red[0][1][j] + red[1][1][j] + red[2][1][j] + red[3][1][j];
    const float s_rms = sqrtf(raw2 / 1024.f) / p.qscale;
    const float k_rms = sqrtf((ksum[0] + ksum[1] + ksum[2] + ksum[3]) / (256.f * (float)D));
    if (s_rms > 0.f && k_rms > 0.f && s_rms < INFINITY && k_rms < INFINITY) {
      const float a = exp2f(rintf(log2f(8.f / s_rms)));
      float ak = exp2f(rintf(log2f(8.f / (sqrtf((float)D) * k_rms))));
      ak = fminf(fmaxf(ak, 0x1p-40f), 0x1p40f);
      float aq = fminf(fmaxf(a / ak, 0x1p-40f), 0x1p40f);
      if (first) {
        p.w1_scales[4 * u] = aq;
        p.w1_scales[4 * u + 1] = ak;
      }
      share[0] = ak;
    }
  }
  if (tid >= 64) return;
  // The first wave: the score spread pooled over the four sampled rows, and the largest n whose support, were the scores
  // Gaussian with that spread, still fits: what the sparse-support kernels compare a row block's keys with.
  float var = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float s1 = red[0][0][j] + red[1][0][j] + red[2][0][j] + red[3][0][j];
    const float s2 = red[0][1][j] + red[1][1][j] + red[2][1][j] + red[3][1][j];
    const float mean = s1 / 256.f;
    var += 0.25f * fmaxf(s2 / 256.f - mean * mean, 0.f);
  }
  const float sd = sqrtf(var);
  // keys whose rows have their threshold `a` spreads above the mean, and the support of such a row
  auto keys_at = [&](float a, float& support) -> float {
    const float Q = 0.5f * erfcf(a * 0.70710678f), phi = 0.39894228f * __expf(-0.5f * a * a);
    float f;  // mass of one key
    if (am == ATT_2) f = sd * (phi - a * Q);
    else if (am == ATT_15) f = var * ((1.f + a * a) * Q - a * phi);
    else {  // any alpha: E[(sd (Z - a))_+^c0] by the midpoint rule over [a, a + 8]
      float acc = 0.f;
#pragma unroll 4
      for (int i = 0; i < 32; ++i) {
        const float x = 0.25f * ((float)i + 0.5f);
        acc += __expf(p.c0 * __logf(sd * x)) * 0.39894228f * __expf(-0.5f * (a + x) * (a + x));
      }
      f = acc * 0.25f;
    }
    const float n = f > 0.f ? 1.f / f : INFINITY;
    support = n * Q;
    return n;
  };
  float lo = -2.f, width = 9.f, n_true = 0.f;
  for (int round = 0; round < 2; ++round) {
    const float step = width * (1.f / 63.f);
    float support;
    const float n = keys_at(lo + (float)tid * step, support);
    const unsigned long long fits = __builtin_amdgcn_ballot_w64(support <= p.probe_max_support);
    // (support grows with a: the lanes that fit are the first ones.  None: the threshold lies below every key of any length
    // considered, the support is the whole row; a spread of zero or a NaN ends here too)
    const int last = fits == ~0ull ? 63 : __builtin_ctzll(~fits) - 1;
    if (last < 0) {
      if (round == 0) n_true = p.probe_max_support * (1.f / 0.97725f);
      break;
    }
    // (all of them: even the shortest lengths have their threshold above the range, and so few keys there that any fits)
    n_true = round == 0 && last == 63 ? INFINITY : __shfl(n, last, 64);
    lo += (float)last * step;
    width = step;
    if (last == 63) break;
  }
  // on a geometric grid of lengths from 64 to a million keys, rounded down
  const float top = floorf(log2f(n_true * (1.f / 64.f)) * (63.f / 14.f) + 1e-4f);
  const float n_fit = n_true < 64.f ? 0.f : (top >= 63.f ? INFINITY : 64.f * exp2f(top * (14.f / 63.f)));
  if (tid != 0) return;
  // A head goes one way as a whole: by its longest rows, which see all L keys and hold most of the work.  (Serving only
  // its shorter row blocks from their supports was measured and loses: for a row block of few tiles the fixed cost of the
  // lists outweighs the walks saved, and a launch split between the two kernels took 15 % longer than the dense kernel
  // alone.)  A marked head: the copy of K skips it and the sparse-support kernels leave its row blocks to the dense ones.
  const bool fits_all = n_fit >= (float)L;
  if (p.w1_scales && first) p.w1_scales[4 * u + 2] = fits_all ? INFINITY : 0.f;
  if (!fits_all) {
    if (first) p.queue[64 + 2 * u] = 1u << 20;
    share[1] = 1.f;
  }
}

// In front of a backward it clears the control words and flags of the dK/dV kernels as well (`ctrl2`, `kv_flags`).
//
// COPY, in front of a forward: gridDim.y workgroups look at a head, each to the same result, the first of them writes it, and
// all of them go on with the e4m3 copy of the head's K (none where the head is marked; tiles that lie wholly behind a
// sequence's length, which no walk reads, are left out).  A launch and the
// wait for the probe's end are saved by that; where and how it is worth it: launch_probe_as.
template <typename T, int D, bool COPY, bool kCross = false>
__global__ __launch_bounds__(256) void attn_probe_kernel(FwdParams<kCross> p, int am, uint32_t* ctrl2, int32_t* kv_flags) {
  __shared__ float share[2];  // COPY: k's scale; nonzero where the head is marked
  const int u = blockIdx.x, tid = threadIdx.x;
  const int units = p.B * p.Hkv;
  uint32_t* const ctrl = p.queue;
  const int b = u / p.Hkv, kvh = u % p.Hkv, group = p.Hq / p.Hkv;
  const bool first = !COPY || blockIdx.y == 0;
  int L = p.N;
  if (p.varlen) {
    long long l = p.varlen_bits == 64 ? ((const long long*)p.varlen)[b] : (long long)((const int*)p.varlen)[b];
    L = (int)(l < 0 ? 0 : (l > p.N ? p.N : l));
  }
  const int NK = key_rows<kCross>(p), LQ = L;
  if constexpr (kCross) L = key_length<kCross>(p, b, NK);
  if (first) {
    if (u == 0 && tid < 11) ctrl[tid] = 0u;
    if (u == 0 && tid < 2) ctrl[64 + 2 * units + tid] = 0u;
    if (tid < 2) ctrl[64 + 2 * u + tid] = 0u;
    if (ctrl2 && u == 0 && tid < 11) ctrl2[tid] = 0u;
    if (kv_flags) {
      const int n_kblk = (NK + kMaskRows - 1) / kMaskRows;
      for (int i = tid; i < n_kblk; i += 256) kv_flags[(size_t)u * n_kblk + i] = 0;
    }
    if (p.save_flags)  // supports kept for the backward: no row block of this K/V head has a valid stream yet
      for (int i = tid; i < group * p.n_mblk; i += 256) p.save_flags[(size_t)(b * p.Hq + kvh * group) * p.n_mblk + i] = 0;
    if (p.w1_scales && tid < 4) p.w1_scales[4 * u + tid] = tid < 2 ? 1.f : (tid == 2 ? INFINITY : 0.f);
  }
  if constexpr (COPY) {
    K8Copy<T, D> copy(reinterpret_cast<const uint16_t*>(p.k), const_cast<unsigned char*>(p.k8), (size_t)u, NK, p.Npad, L);
    long long id = (long long)blockIdx.y * 256 + tid;
    copy.load(id);  // (under way while the probe works)
    if (tid == 0) {
      share[0] = 1.f;
      share[1] = 0.f;
    }
    probe_head<T, D, kCross>(p, am, u, L, LQ, first, share);
    __syncthreads();
    const float ak = share[0];
    if (share[1] != 0.f) return;
    const long long step = (long long)gridDim.y * 256;
    for (; id - tid < copy.n; id += step) {
      K8Copy<T, D> now = copy;
      copy.load(id + step);
      now.store(id, ak);
    }
  } else {
    probe_head<T, D, kCross>(p, am, u, L, LQ, true, share);
  }
}

// The probe, and in front of a forward (COPY) the e4m3 copy of K, for the head dims the sparse-support kernels serve.
constexpr long long kCopyPieces = 4096;  // pieces of 256 threads x 16 values that the probe's own workgroups copy
template <typename T, int D, bool COPY, bool kCross = false>
static void launch_probe_as(const FwdParams<kCross>& p, int am, uint32_t* ctrl2, int32_t* kv_flags, hipStream_t s) {
  const long long units = (long long)p.B * p.Hkv;
  if constexpr (COPY) {
    const long long pieces = ((long long)p.Npad * (D / 16) + 255) / 256;
    // Up to 32 MiB of K the probe's workgroups copy it.  About one to a CU: looking at a head again costs each of them the sample's loads (2 x 32/8
    // heads, N = 2048, D = 128: forward 150 us with the copy behind the probe, 146.5 with 256 workgroups, 147.2 with 512, 152 with 1024), and more, to
    // what a CU holds, once eight pieces and more are left to each.  The forward, copy behind the probe against this: 32/8 heads, N = 2048, D = 128
    // 98.4 -> 93.6; 8 heads, N = 4096, D = 64 116.4 -> 113.0; 4 x 16 heads 329 -> 326 (16 MiB).  For larger K the copy
    // wants more bytes in flight than these workgroups have: 4 x 16 heads, N = 4096, D = 128 (64 MiB) 304 -> 309; 8 x 8 heads, N <= 8192 2223 -> 2250.
    if (units * pieces <= kCopyPieces) {
      long long parts = (255 + units) / units;
      const long long more = pieces / 8 < 768 / units ? pieces / 8 : 768 / units;
      parts = parts > more ? parts : more;
      parts = parts < pieces ? parts : pieces;
      hipLaunchKernelGGL((attn_probe_kernel<T, D, true, kCross>), dim3((unsigned)units, (unsigned)parts), dim3(256), 0, s, p, am, ctrl2, kv_flags);
      return;
    }
    hipLaunchKernelGGL((attn_probe_kernel<T, D, false, kCross>), dim3((unsigned)units), dim3(256), 0, s, p, am, ctrl2, kv_flags);
    hipLaunchKernelGGL((k8_layout_kernel<T, D, kCross>), dim3((unsigned)pieces, (unsigned)units), dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((attn_probe_kernel<T, D, false, kCross>), dim3((unsigned)units), dim3(256), 0, s, p, am, ctrl2, kv_flags);
  }
}
template <bool COPY, bool kCross = false>
static void launch_probe(const FwdParams<kCross>& p, int D, int dtype, int am, uint32_t* ctrl2, int32_t* kv_flags, hipStream_t s) {
  if (dtype == ADSP_BF16) {
    if (D == 64) launch_probe_as<bf16_t, 64, COPY, kCross>(p, am, ctrl2, kv_flags, s);
    else launch_probe_as<bf16_t, 128, COPY, kCross>(p, am, ctrl2, kv_flags, s);
  } else {
    if (D == 64) launch_probe_as<f16_t, 64, COPY, kCross>(p, am, ctrl2, kv_flags, s);
    else launch_probe_as<f16_t, 128, COPY, kCross>(p, am, ctrl2, kv_flags, s);
  }
}

}  // namespace adsp
