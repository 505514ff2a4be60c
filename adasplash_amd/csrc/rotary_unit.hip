// One translation unit per element type (-DADSP_T=...): heads of queries and keys normed and turned by their tokens' positions.
//
//   n = x w / sqrt(mean x^2 + eps)   (with a weight; else n = x),   theta = position * frequency,
//   (a, b) of n -> factor (a cos theta - b sin theta, b cos theta + a sin theta),   the rest of the head as it is;
// pairs (a, b) are elements i and i + rot / 2 ("half") or 2 i and 2 i + 1 ("interleaved") of the first `rot`.  Backward, with g the gradient turned the other way, r = 1 / sqrt(mean x^2 + eps):
//   dw = sum over rows of g x r,   dx = r (w g - x r^2 mean(x w g)).
//
// What bounds it: HBM, every row once in and once out; a decoding step's call: latency.  us in the kernel, 32/8 heads, D = 128, bf16: one token 3.4; 8190 tokens 27.2 (168 MB, 6.2 TB/s); 4 x 8192 with norms, rows as a
// projection leaves them, 128 (671 MB, 5.2 TB/s), their gradients 222 (1007 MB, 4.5 TB/s); 8 heads of K and V of 16000 tokens into pages 21.0 (131 MB, 6.2 TB/s).
// A group of D / 8 lanes has a token, and goes through the workgroup's heads with the same angles: eight elements of a row to a lane, of which four and four belong to
// four pairs.  Cosines and sines are formed where they are used, four to a lane and token: a table of them would be read as often as a head's rows, and would end at some position.
#include "rotary.h"

namespace adsp {
namespace rotary {

// cos and sin of position * frequency.  The product has 53 bits and so has its part of a turn (fp32 would have none left at a position of some millions): off by 2^-52 of the product, below
// fp32's own roundings up to positions of 2^28.  Quarter turns are taken off in 64 bits, what is left is at most pi / 4, and there the two series end where the next term is below 2e-9.
__device__ __forceinline__ void cos_sin(double position, double frequency, float& c, float& s) {
  const double quarters = position * frequency * 0.63661977236758134308, k = __builtin_rint(quarters);
  const float y = (float)((quarters - k) * 1.57079632679489661923), y2 = y * y;
  const int quadrant = (int)(k - 4.0 * __builtin_floor(k * 0.25));
  const float sn = fmaf(y * y2, fmaf(y2, fmaf(y2, fmaf(y2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), y);
  const float cs = fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const float a = quadrant & 1 ? sn : cs, b = quadrant & 1 ? cs : sn;
  c = quadrant == 1 || quadrant == 2 ? -a : a;
  s = quadrant >= 2 ? -b : b;
}

template <int kLanes> __device__ __forceinline__ float group_sum(float v) {
  if constexpr (kLanes >= 2) v += dpp_move<0xb1, 0xf>(v, v);
  if constexpr (kLanes >= 4) v += dpp_move<0x4e, 0xf>(v, v);
  if constexpr (kLanes >= 8) v += dpp_move<0x141, 0xf>(v, v);
  if constexpr (kLanes >= 16) v += dpp_move<0x140, 0xf>(v, v);
  if constexpr (kLanes >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// Eight elements of a row as two runs of four, 8 or 16 bytes each.
template <typename T> struct Eight {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  using Raw = std::conditional_t<elem_traits<T>::kVec == 4, u32x4, u32x2>;
  Raw a, b;
  __device__ __forceinline__ void load(const void* row, int ea, int eb) {
    a = *reinterpret_cast<const Raw*>((const char*)row + ea * elem_traits<T>::kBytes);
    b = *reinterpret_cast<const Raw*>((const char*)row + eb * elem_traits<T>::kBytes);
  }
  __device__ __forceinline__ void store(void* row, int ea, int eb) const {
    *reinterpret_cast<Raw*>((char*)row + ea * elem_traits<T>::kBytes) = a;
    *reinterpret_cast<Raw*>((char*)row + eb * elem_traits<T>::kBytes) = b;
  }
  static __device__ __forceinline__ void unpack(Raw r, float* x) {
    if constexpr (elem_traits<T>::kVec == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bits = r[i];
        x[i] = __builtin_bit_cast(float, bits);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[2 * i] = unpack_lo<T>(r[i]);
        x[2 * i + 1] = unpack_hi<T>(r[i]);
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float* x) {
    Raw r;
    if constexpr (elem_traits<T>::kVec == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) r[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    }
    return r;
  }
  __device__ __forceinline__ void get(float* x) const {
    unpack(a, x);
    unpack(b, x + 4);
  }
  __device__ __forceinline__ void set(const float* x) {
    a = pack(x);
    b = pack(x + 4);
  }
};

// Where a lane's eight elements lie in a row, and the angles of its four pairs.
template <bool kHalf> struct Lane {
  int ea, eb;
  bool turned;  // (the others stay as they are: not even an angle of 0 would do, where 0 times an infinity beside an element makes a NaN of it)
  __device__ __forceinline__ Lane(int c, int rot) {
    turned = c < rot / 8;
    if (kHalf && turned) {
      ea = 4 * c;
      eb = ea + rot / 2;
    } else {
      ea = 8 * c;
      eb = ea + 4;
    }
  }
  // elements i and j of the lane's eight that form pair e
  static __device__ __forceinline__ int first(int e) { return kHalf ? e : 2 * e; }
  static __device__ __forceinline__ int second(int e) { return kHalf ? e + 4 : 2 * e + 1; }
};
struct Angles {
  float c[4], s[4];
  __device__ __forceinline__ void set(const Params& p, bool turned, int lane, double position) {
    if (!turned) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cos_sin(position, p.frequencies[lane * 4 + e], c[e], s[e]);
      c[e] *= p.factor;
      s[e] *= p.factor;
    }
  }
  template <bool kHalf> __device__ __forceinline__ void turn(float* x) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float &a = x[Lane<kHalf>::first(e)], &b = x[Lane<kHalf>::second(e)];
      const float t = a * c[e] - b * s[e];
      b = b * c[e] + a * s[e];
      a = t;
    }
  }
  template <bool kHalf> __device__ __forceinline__ void turn_back(float* x) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float &a = x[Lane<kHalf>::first(e)], &b = x[Lane<kHalf>::second(e)];
      const float t = a * c[e] + b * s[e];
      b = b * c[e] - a * s[e];
      a = t;
    }
  }
};
__device__ __forceinline__ double position_of(const Params& p, long long b, long long n) {
  const long long at = b * p.pos_b + n * p.pos_n;
  return p.pos_bits == 64 ? (double)((const long long*)p.positions)[at] : (double)((const int*)p.positions)[at];
}
template <typename T> __device__ __forceinline__ void load_weight(const void* weight, bool f32, int ea, int eb, float* w) {
  if (f32) {
    Eight<float> e;
    e.load(weight, ea, eb);
    e.get(w);
  } else {
    Eight<T> e;
    e.load(weight, ea, eb);
    e.get(w);
  }
}
__device__ __forceinline__ float inv_rms(float sum, const Params& p) { return __builtin_amdgcn_rsqf(fmaf(sum, p.inv_d, p.eps)); }

// Workgroup: 4 * 64 / kLanes tokens, `per` heads of q or of k, one after another.  us in a graph, loads of one, two, four, eight heads ahead: one token with norms 3.2, 3.7, 4.0, 4.5; 8190 tokens 26.8, 27.1, 27.0, 26.6; 32768 with norms,
// contiguous, 119, 121, 132, 145.  (The rows of 4 x 8192 as a projection leaves them, with gradients: 354, 351.)
template <typename T, int D, bool kHalf, bool kPages> __global__ __launch_bounds__(kThreads) void rotary_kernel(Params p) {
  constexpr int kLanes = D / 8, kTokens = kThreads / kLanes, kB = elem_traits<T>::kBytes;
  const int tid = threadIdx.x, c = tid % kLanes;
  const int which = (int)blockIdx.y < p.of[0].blocks ? 0 : 1;
  const Rows& rows = p.of[which];
  const int h0 = ((int)blockIdx.y - (which ? p.of[0].blocks : 0)) * p.per, h1 = h0 + p.per < rows.heads ? h0 + p.per : rows.heads;
  const uint32_t token = blockIdx.x * kTokens + tid / kLanes;
  const bool valid = token < p.tokens;
  const uint32_t t = valid ? token : p.tokens - 1;
  const long long b = t / p.N, n = t % p.N;
  const Lane<kHalf> lane(c, p.rot);
  const char* const x = (const char*)rows.x + (b * rows.x_b + n * rows.x_n) * kB;
  char* y;
  long long y_h;
  bool writes = valid;
  if constexpr (kPages) {
    const long long slot = p.pages.slots[t];
    writes = writes && slot >= 0 && slot < p.pages.n_slots;
    const long long pg = writes ? slot / p.pages.page : 0, in = writes ? slot - pg * p.pages.page : 0;
    y = (char*)rows.y + pg * p.pages.k_sp + in * p.pages.k_sps;
    y_h = p.pages.k_sph;
    // V's rows go as they are, in pieces of 16 bytes
    const char* const v = p.pages.v + t * p.pages.v_st;
    char* const to = p.pages.v_pages + pg * p.pages.v_sp + in * p.pages.v_sps;
    if (writes) {
      for (int h = h0; h < h1; ++h)
        for (int i = c; i < D * kB / 16; i += kLanes)
          *reinterpret_cast<u32x4*>(to + h * p.pages.v_sph + i * 16) = *reinterpret_cast<const u32x4*>(v + h * p.pages.v_sh + i * 16);
    }
  } else {
    y = (char*)rows.y + (b * rows.y_b + n * rows.y_n) * kB;
    y_h = rows.y_h * kB;
  }
  Angles angles;
  angles.set(p, lane.turned, c, position_of(p, b, n));
  float w[8];
  const bool norm = rows.weight != nullptr;
  if (norm) load_weight<T>(rows.weight, p.weight_f32[which], lane.ea, lane.eb, w);
  for (int h = h0; h < h1; ++h) {
    Eight<T> raw;
    raw.load(x + h * rows.x_h * kB, lane.ea, lane.eb);
    float v[8];
    raw.get(v);
    if (norm) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
      const float r = inv_rms(group_sum<kLanes>(sum), p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * r * w[e];
    }
    if (lane.turned) angles.turn<kHalf>(v);
    raw.set(v);
    if (writes) raw.store(y + h * y_h, lane.ea, lane.eb);
  }
}

// Gradients: as above, along the tokens in steps of the grid; the weights' sums stay in registers until the workgroup's last row.  us, 32768 tokens, loads of one, two, four heads ahead: 240, 226, 229.
template <typename T, int D, bool kHalf> __global__ __launch_bounds__(kThreads) void rotary_bwd_kernel(Params p) {
  constexpr int kLanes = D / 8, kTokens = kThreads / kLanes, kB = elem_traits<T>::kBytes, kAhead = 2;
  __shared__ float sums[kTokens][D];
  const int tid = threadIdx.x, c = tid % kLanes;
  const int which = (int)blockIdx.y < p.of[0].blocks ? 0 : 1;
  const Rows& rows = p.of[which];
  const int block = (int)blockIdx.y - (which ? p.of[0].blocks : 0), h0 = block * p.per, h1 = h0 + p.per < rows.heads ? h0 + p.per : rows.heads;
  const Lane<kHalf> lane(c, p.rot);
  const bool norm = rows.weight != nullptr;
  float w[8], dw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = dw[e] = 0.f;
  if (norm) load_weight<T>(rows.weight, p.weight_f32[which], lane.ea, lane.eb, w);
  for (int step = 0; step < p.token_steps; ++step) {
    const uint32_t token = ((uint32_t)step * p.token_blocks + blockIdx.x) * kTokens + tid / kLanes;
    const bool valid = token < p.tokens;
    const uint32_t t = valid ? token : p.tokens - 1;
    const long long b = t / p.N, n = t % p.N;
    const char* const dy = (const char*)rows.dy + (b * rows.dy_b + n * rows.dy_n) * kB;
    const char* const x = (const char*)rows.x + (b * rows.x_b + n * rows.x_n) * kB;
    char* const y = (char*)rows.y + (b * rows.y_b + n * rows.y_n) * kB;
    Angles angles;
    angles.set(p, lane.turned, c, position_of(p, b, n));
    for (int h = h0; h < h1; h += kAhead) {
      Eight<T> raw[kAhead], raw_x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int hh = h + u < h1 ? h + u : h;
        raw[u].load(dy + hh * rows.dy_h * kB, lane.ea, lane.eb);
        if (norm) raw_x[u].load(x + hh * rows.x_h * kB, lane.ea, lane.eb);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float g[8];
        raw[u].get(g);
        if (lane.turned) angles.turn_back<kHalf>(g);
        const bool counts = valid && h + u < h1;
        if (norm) {
          float v[8], sum = 0.f, dot = 0.f;
          raw_x[u].get(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
          const float r = inv_rms(group_sum<kLanes>(sum), p);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] *= r;  // the normed element
            if (counts) dw[e] = fmaf(g[e], v[e], dw[e]);
            g[e] *= w[e];
            dot = fmaf(g[e], v[e], dot);
          }
          const float mean = group_sum<kLanes>(dot) * p.inv_d;
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = r * fmaf(-mean, v[e], g[e]);
        }
        raw[u].set(g);
        if (counts) raw[u].store(y + (h + u) * rows.y_h * kB, lane.ea, lane.eb);
      }
    }
  }
  if (!norm) return;
  float* const mine = sums[tid / kLanes];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    mine[lane.ea + e] = dw[e];
    mine[lane.eb + e] = dw[4 + e];
  }
  __syncthreads();
  for (int d = tid; d < D; d += kThreads) {
    float sum = 0.f;
    for (int i = 0; i < kTokens; ++i) sum += sums[i][d];
    rows.partial[((size_t)blockIdx.x * rows.blocks + block) * D + d] = sum;
  }
}

template <typename T, int D> static void launch_d(const Params& p, bool half, int mode, hipStream_t s) {
  const dim3 grid((unsigned)p.token_blocks, (unsigned)(p.of[0].blocks + p.of[1].blocks)), block(kThreads);
  if (mode == 0) {
    if (half) hipLaunchKernelGGL((rotary_kernel<T, D, true, false>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, D, false, false>), grid, block, 0, s, p);
  } else if (mode == 1) {
    if (half) hipLaunchKernelGGL((rotary_kernel<T, D, true, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, D, false, true>), grid, block, 0, s, p);
  } else {
    if (half) hipLaunchKernelGGL((rotary_bwd_kernel<T, D, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((rotary_bwd_kernel<T, D, false>), grid, block, 0, s, p);
  }
}
template <> void launch<ADSP_T>(const Params& p, int D, bool half, int mode, hipStream_t s) {
  if (D == 16) launch_d<ADSP_T, 16>(p, half, mode, s);
  else if (D == 32) launch_d<ADSP_T, 32>(p, half, mode, s);
  else if (D == 64) launch_d<ADSP_T, 64>(p, half, mode, s);
  else if (D == 128) launch_d<ADSP_T, 128>(p, half, mode, s);
  else launch_d<ADSP_T, 256>(p, half, mode, s);
}
}  // namespace rotary
}  // namespace adsp
