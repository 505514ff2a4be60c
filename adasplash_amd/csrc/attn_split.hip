// Entmax attention of a few queries of each sequence against many keys, split over the keys and joined: one new token of every
// request over a cache of pages (block tables, grouped heads), and a few queries against an encoder's states.
//
//   z_j = (alpha - 1) q k_j / sqrt(D),  sum_j [z_j - tau]_+^c0 = 1,  out = sum_j [z_j - tau]_+^c0 v_j,  c0 = 1 / (alpha - 1) >= 1
//
// What bounds it: K from HBM, once; of V only the supports' rows are read, some tens of a sequence's thousands.
//
// Split: the rows of a K/V head (its group's heads times the queries, up to 64) share every load of K.  A workgroup takes up to 2048 keys
// of a head: its waves form the scores of 64 keys at a time on 16 x 16 matrix tiles, whose other side is the rows, and leave them in LDS;
// then a wave takes a row, holds its scores in registers, and takes Newton's steps towards the threshold that these keys alone would
// have.  A part's threshold is a lower bound of the whole row's (each further key raises it), and so is each step from below: what lies under it
// is in no support.  The part leaves the bound and the keys above it, a few dozen of 2048, where the maximum less 1 would leave hundreds.
// The second kernel, a workgroup per row, takes the largest of the bounds, gathers the keys above it, solves the threshold on them
// and reads their rows of V.  Where a workgroup can take all keys of a head, one kernel does both.  Lists are in an order that the keys' places
// give (within a part by lane), sums in the order of the lists: a call returns the same bits every time.
//
// Measured, bf16, 32/8 heads, D = 128, both kernels: 48 requests of 2048 to 8192 tokens (503 MB of K) 118 us = 4.3 TB/s, of which the second kernel's 11 (a large copy: 5.0 TB/s, a
// read of consecutive addresses 6.0); the first without its solves 101.  2 of 32767 and 131071 (336 MB): 88.  1 of 600: 11.9, latency: K after length and table 2.5 us,
// its scores 1, entries 1.6, solve 1, V 1, and two launches.  Lists to the maximum less 1 and a second kernel that walked them part by part: 130, 126, 14.4; scores of spread 1/8,
// 4 x 64/8 heads, 20000: 463 -> 92.
#include "attn_split.h"
#include "../../include/adasplash_hip.h"

namespace adsp {
namespace split {
// First kernel: workgroup (head, part).  It leaves, for each row, a lower bound of the row's threshold and the keys above it.
template <typename T, int D, int AM, bool kPaged> __global__ __launch_bounds__(64 * kWaves) void split_scores_kernel(SplitParams p) {
  extern __shared__ __align__(16) float z[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (Parts behind parts: the hardware deals workgroups out to its eight XCDs in turn, and a head's later parts, which shorter sequences do not have, must not all
  // fall to the same ones.  us, head behind head -> this: 48 requests x 8 heads of up to 8192 keys, D = 128: 123 -> 118; 128 x 8 of 3000, D = 64: 80 -> 61.)
  const int unit = blockIdx.x % p.units, part = blockIdx.x / p.units, b = unit / p.Hkv, kvh = unit % p.Hkv;
  const int key0 = part * p.chunk, zs = score_stride(p.chunk);
  int* const pages = reinterpret_cast<int*>(z + p.R * zs);
  if constexpr (kPaged) {
    const int first = page_of(p, key0), last = page_of(p, (key0 + p.chunk < p.N ? key0 + p.chunk : p.N) - 1);
    for (int i = first + tid; i <= last; i += 64 * kWaves) pages[i - first] = table_entry(p, b, i);
  }
  const int len = length_at(p.lens, p.lens_bits, b, p.N);
  if (key0 >= len) return;  // (the second kernel knows the length too)
  const int n = len - key0 < p.chunk ? len - key0 : p.chunk;
  if constexpr (kPaged) __syncthreads();
  chunk_scores<T, D, kPaged, kWaves>(p, b, kvh, key0, n, z, pages, wave, lane);
  __syncthreads();
  for (int row = wave; row < p.R; row += kWaves)
    leave_part<AM>(p, z + row * zs, n, key0, ((size_t)unit * p.R + row) * p.splits + part, lane);
}

// Rows of V added up by groups of kLanes lanes, one row to a group at a time.
template <typename T, int D> struct Gather {
  static constexpr int kVec = elem_traits<T>::kVec, kB = elem_traits<T>::kBytes, kLanes = D / kVec;
  const char* base;
  float acc[kVec], weights;  // and the sum of the weights
  __device__ __forceinline__ Gather(const SplitParams& p, bool paged, int b, int kvh, int col)
      : base((const char*)p.v + ((paged ? 0 : b * p.v_s0) + kvh * p.v_sh + col * kVec) * kB) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[e] = 0.f;
    weights = 0.f;
  }
  __device__ __forceinline__ u32x4 load(long long off) const { return *reinterpret_cast<const u32x4*>(base + off * kB); }
  __device__ __forceinline__ void add(float w, u32x4 raw) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[e] = fmaf(w, chunk_elem<T>(raw, e), acc[e]);
    weights += w;
  }
  // the groups of a wave together: every lane of a column ends with the wave's sum
  __device__ __forceinline__ void join() {
#pragma unroll
    for (int o = kLanes; o < 64; o <<= 1) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
      weights += __shfl_xor(weights, o, 64);
    }
  }
};
__device__ __forceinline__ float over_sum(float x, float sum) { return sum > 0.f ? x / sum : 0.f; }
// Entries first, first + step, ... below n of a list of weights and keys: kAhead rows of V under way together.
template <typename T, int D, bool kPaged, int kAhead, typename Weight, typename Key>
__device__ __forceinline__ void gather_list(const SplitParams& p, int b, Gather<T, D>& g, int first, int step, int n, Weight&& weight, Key&& key) {
  for (int i = first; i < n; i += kAhead * step) {
    float w[kAhead];
    int at[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = i + u * step;
      w[u] = j < n ? weight(j) : 0.f;
      at[u] = key(j < n ? j : i);  // (a slot past the end takes the first one's row with weight zero)
    }
    long long off[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if constexpr (kPaged) {
        // (the lists of a common prefix are filled up with entries without weight, whose key may lie in a page that is none: any page serves them)
        const int pg = page_of(p, at[u]), id = table_entry(p, b, pg);
        off[u] = (id >= 0 ? id : 0) * p.v_s0 + (at[u] - pg * p.page) * p.v_sn;
      } else {
        off[u] = at[u] * p.v_sn;
      }
    }
    u32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = g.load(off[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (w[u] > 0.f) g.add(w[u], raw[u]);
  }
}

// What the parts of a row left, in memory, as the 256 threads of a workgroup see it.
struct PartsRow {
  const Part* parts;
  const Entry* entries;
  int splits, chunk, tid;
  float m;  // the row's maximum
  template <typename F> __device__ __forceinline__ void for_each(F f) const {
    for (int s = 0; s < splits; ++s) {
      const int count = parts[s].count;
      for (int i = tid; i < count; i += 256) f(entries[(size_t)s * chunk + i].z - m);
    }
  }
};

// Second kernel: workgroup = row.  What bounds it is latency: parts, entries, table and values, one behind the other.  Each wave looks at a quarter of the parts,
// eight at a time whose first 64 entries are asked for before their number is known, and keeps those above the bound in its quarter of the list.
template <typename T, int D, int AM, bool kPaged> __global__ __launch_bounds__(256) void split_join_kernel(SplitParams p) {
  constexpr int kLanes = Gather<T, D>::kLanes, kVec = Gather<T, D>::kVec;
  constexpr int kGroups = 256 / kLanes;  // V rows read side by side
  constexpr int kPer = kListCap / 256, kCap = kListCap / 4, kBatch = 8;
  constexpr int kPasses = 4;
  __shared__ float sm[32];
  __shared__ float list_z[4][kCap];
  __shared__ int list_key[4][kCap];
  __shared__ int totals[4], members[4];
  __shared__ float red[4][D], red_weights[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x, unit = row / p.R, b = unit / p.Hkv, kvh = unit % p.Hkv, r = row % p.R;
  const int len = r % p.Nq < length_at(p.lens_q, p.lens_q_bits, b, p.Nq) ? length_at(p.lens, p.lens_bits, b, p.N) : 0;
  const int splits = parts_of(p, len);
  Part* const parts = p.parts + (size_t)row * p.splits;
  const Entry* const entries = p.entries + (size_t)row * p.splits * p.chunk;
  const int grp = tid / kLanes, col = tid % kLanes;
  Gather<T, D> g(p, kPaged, b, kvh, col);

  const int per = (splits + 3) / 4, s0 = wave * per, s1 = s0 + per < splits ? s0 + per : splits;
  Entry e[kBatch];
  int count[kBatch];
  auto load_batch = [&](int s) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = s + u < s1 ? s + u : s;
      count[u] = s + u < s1 ? parts[at].count : 0;
      e[u] = entries[(size_t)at * p.chunk + lane];
    }
  };
  if (s0 < s1) load_batch(s0);  // (on its way while the bound is formed)
  float m = -INFINITY, bound = -INFINITY;
  for (int s = lane; s < splits; s += 64) {
    m = fmaxf(m, parts[s].max);
    bound = fmaxf(bound, parts[s].bound);
  }
  m = wave_max(m);
  if (m > -INFINITY) {
    // from here on relative to the maximum (one of +inf leaves no key above the bound)
    bound = fmaxf(wave_max(bound) - m, -1.f);
    int mine, n0, n1, n2, n3, n;
    float sums[2];
    bool fits;
    auto take = [&](const Entry& x, bool in) {
      const float z = x.z - m;
      in = in && z > bound;
      const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
      const int place = mine + __builtin_popcountll(who & ((1ull << lane) - 1ull));
      if (in && place < kCap) {
        list_z[wave][place] = z;
        list_key[wave][place] = x.key;
      }
      mine += __builtin_popcountll(who);
      accum_stats<AM>(in ? z - bound : -1.f, p.rows.c0, sums);
    };
    // Where more keys lie above the bound than the lists hold (flat scores: a part's own threshold is far below the row's), a step of Newton's method from it
    // on all of them gives a nearer one, and they are gone through again.
    for (int pass = 0;; ++pass) {
    mine = 0;
    sums[0] = sums[1] = 0.f;
    for (int s = s0; s < s1; s += kBatch) {
      if (s > s0 || pass > 0) load_batch(s);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (count[u] == 0) continue;
        take(e[u], lane < count[u]);
        for (int i = 64; i < count[u]; i += 256) {
          Entry more[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int at = i + v * 64 + lane;
            more[v] = entries[(size_t)(s + u) * p.chunk + (at < count[u] ? at : 0)];
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) take(more[v], i + v * 64 + lane < count[u]);
        }
      }
    }
    if (lane == 0) totals[wave] = mine;
    __syncthreads();
    n0 = totals[0], n1 = totals[1], n2 = totals[2], n3 = totals[3], n = n0 + n1 + n2 + n3;
    fits = n0 <= kCap && n1 <= kCap && n2 <= kCap && n3 <= kCap;
    if (fits || pass == kPasses) break;
    row_sum<256, 2>(sums, sm);  // (its barriers: the totals have been read)
    bound = raised<AM>(bound, sums[0], sums[1], p.rows);
    }
    if (p.taus && tid == 0) parts[0].max = m;  // (behind a barrier: every wave has read the parts' maxima)
    if (fits) {
      auto place_of = [&](int j) {  // entry j of the row in the four waves' lists
        int w = 0;
        if (j >= n0) j -= n0, w = kCap;
        if (w == kCap && j >= n1) j -= n1, w = 2 * kCap;
        if (w == 2 * kCap && j >= n2) j -= n2, w = 3 * kCap;
        return w + j;
      };
      const float* const zs = &list_z[0][0];
      const int* const keys = &list_key[0][0];
      // thread t has entries t, t + 256, ...
      float ez[kPer], tau;
      int ek[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = i * 256 + tid;
        ez[i] = -INFINITY;
        ek[i] = 0;
        if (i * 256 < n && at < n) {
          ez[i] = zs[place_of(at)];
          ek[i] = keys[place_of(at)];
        }
      }
      if (n <= 256) {  // (every wave for itself: no barriers)
        ListRow<4> lr;
#pragma unroll
        for (int i = 0; i < 4; ++i) lr.z[i] = i * 64 + lane < n ? zs[place_of(i * 64 + lane)] : -INFINITY;
        tau = solve_from<AM, false>(lr, bound, p.rows, sm);
      } else {
        ListRow<kPer> lr;
#pragma unroll
        for (int i = 0; i < kPer; ++i) lr.z[i] = ez[i];
        tau = solve_from<AM, true>(lr, bound, p.rows, sm);
      }
      // the support, in the lists' place
      int count = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) count += ez[i] > tau ? 1 : 0;
      const int upto = wave_prefix_sum(count);
      if (lane == 63) members[wave] = upto;
      __syncthreads();  // (every thread has its entries)
      int at = upto - count + (wave > 0 ? members[0] : 0) + (wave > 1 ? members[1] : 0) + (wave > 2 ? members[2] : 0);
      const int n_members = members[0] + members[1] + members[2] + members[3];
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (ez[i] > tau) {
          (&list_z[0][0])[at] = prob<AM>(ez[i] - tau, p.rows.c0);
          (&list_key[0][0])[at] = ek[i];
          ++at;
        }
      __syncthreads();
      if (p.taus && tid == 0) p.taus[row] = tau;
      gather_list<T, D, kPaged, 4>(p, b, g, grp, kGroups, n_members, [&](int j) { return zs[j]; }, [&](int j) { return keys[j]; });
    } else {
      // a flat row: more keys above the bound than the lists hold; solved on the parts' entries in memory
      const PartsRow pr{parts, entries, splits, p.chunk, tid, m};
      const float tau = solve_from<AM, true>(pr, bound, p.rows, sm);
      if (p.taus && tid == 0) p.taus[row] = tau;
      for (int s = 0; s < splits; ++s) {
        const Entry* const list = entries + (size_t)s * p.chunk;
        gather_list<T, D, kPaged, 8>(p, b, g, grp, kGroups, parts[s].count, [&](int j) { return prob<AM>(list[j].z - m - tau, p.rows.c0); },
                                     [&](int j) { return list[j].key; });
      }
    }
  } else if (p.taus && tid == 0) {
    p.taus[row] = INFINITY;  // (no key, no member)
  }
  g.join();
  if (lane < kLanes) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) red[wave][lane * kVec + e] = g.acc[e];
    red_weights[wave] = g.weights;
  }
  __syncthreads();
  const float sum = red_weights[0] + red_weights[1] + red_weights[2] + red_weights[3];
  for (int d = tid; d < D; d += 256) store_elem<T>(p.out, (size_t)row * D + d, over_sum(red[0][d] + red[1][d] + red[2][d] + red[3][d], sum));
}

// Both at once where a workgroup holds all keys of a head: one launch.  A wave solves a row; the waves, W / R of them to a row, gather.
static size_t whole_lds(int R, int chunk, int page, bool paged, int W, int D) {
  return (size_t)W * (D + 1) * 4 + ((size_t)R + 3) / 4 * 16 + scores_lds(R, chunk, page, paged) + (size_t)R * chunk * 2;
}
template <typename T, int D, int AM, bool kPaged, int W> __global__ __launch_bounds__(64 * W) void split_whole_kernel(SplitParams p) {
  constexpr int kLanes = Gather<T, D>::kLanes, kVec = Gather<T, D>::kVec;
  extern __shared__ __align__(16) float lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int unit = blockIdx.x, b = unit / p.Hkv, kvh = unit % p.Hkv, zs = score_stride(p.chunk);
  static_assert(W % 4 == 0, "rows of 16 bytes behind the sums");
  float* const red = lds;                                                    // [W][D]
  float* const red_weights = red + W * D;                                    // [W]
  int* const members = reinterpret_cast<int*>(red_weights + W);              // [R], of each row
  float* const z = reinterpret_cast<float*>(members + (p.R + 3) / 4 * 4);    // [R][zs]: scores, then the members' weights
  int* const pages = reinterpret_cast<int*>(z + p.R * zs);
  uint16_t* const keys = reinterpret_cast<uint16_t*>(pages + (kPaged ? p.chunk / p.page + 2 : 0));  // [R][chunk]
  if constexpr (kPaged) {
    const int last = page_of(p, p.N - 1);
    for (int i = tid; i <= last; i += 64 * W) pages[i] = table_entry(p, b, i);
  }
  const int n = length_at(p.lens, p.lens_bits, b, p.N), nq = length_at(p.lens_q, p.lens_q_bits, b, p.Nq);
  if constexpr (kPaged) __syncthreads();
  if (n > 0) chunk_scores<T, D, kPaged, W>(p, b, kvh, 0, n, z, pages, wave, lane);
  __syncthreads();
  for (int row = wave; row < p.R; row += W) {
    float* const zr = z + row * zs;
    uint16_t* const kr = keys + row * p.chunk;
    HeldRow held;
    const float m = hold_row(held, zr, n, lane);
    int upto = 0;
    if (m > -INFINITY && row % p.Nq < nq) {
      held.less(m);  // (a maximum of +inf leaves no number above any threshold: the row is 0)
      const float tau = solve_from<AM, false>(held, -1.f, p.rows, nullptr);
      int count = 0;
      held.for_each([&](float x) { count += x > tau ? 1 : 0; });
      upto = wave_prefix_sum(count);
      int w = upto - count;
#pragma unroll
      for (int i = 0; i < kMaxChunk / 256; ++i)
        if (i * 256 < n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = held.z[i][e];
            if (x > tau) {
              zr[w] = prob<AM>(x - tau, p.rows.c0);
              kr[w] = (uint16_t)(i * 256 + lane * 4 + e);
              ++w;
            }
          }
        }
    }
    if (lane == 63) members[row] = upto;
  }
  __syncthreads();
  // per: waves to a row, a power of two
  int per = 1;
  while (per * 2 * p.R <= W) per *= 2;
  const int sub = wave % per, grp = sub * (64 / kLanes) + lane / kLanes, col = lane % kLanes;
  for (int row0 = 0; row0 < p.R; row0 += W / per) {
    const int row = row0 + wave / per;
    Gather<T, D> g(p, kPaged, b, kvh, col);
    if (row < p.R) {
      const float* const wr = z + row * zs;
      const uint16_t* const kr = keys + row * p.chunk;
      const int n_row = members[row];
      for (int i = grp; i < n_row; i += 4 * per * (64 / kLanes)) {
        u32x4 raw[4];
        float w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = i + u * per * (64 / kLanes), key = kr[j < n_row ? j : i];
          w[u] = j < n_row ? wr[j] : 0.f;
          long long off;
          if constexpr (kPaged) {
            const int pg = page_of(p, key);
            off = pages[pg] * p.v_s0 + (key - pg * p.page) * p.v_sn;
          } else {
            off = key * p.v_sn;
          }
          raw[u] = g.load(off);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (w[u] > 0.f) g.add(w[u], raw[u]);
      }
      g.join();
      if (lane < kLanes) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) red[wave * D + lane * kVec + e] = g.acc[e];
        red_weights[wave] = g.weights;
      }
    }
    if (per > 1) __syncthreads();
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (row < p.R && sub == 0) {
      const size_t at = ((size_t)unit * p.R + row) * D;
      float sum = red_weights[wave];
      for (int w = 1; w < per; ++w) sum += red_weights[wave + w];
      for (int d = lane; d < D; d += 64) {
        float x = red[wave * D + d];
        for (int w = 1; w < per; ++w) x += red[(wave + w) * D + d];
        store_elem<T>(p.out, at + d, over_sum(x, sum));
      }
    }
    if (per > 1) __syncthreads();
  }
}

// ---- gradients of a few queries --------------------------------------------------------------------------------------
// What the forward left of a row, its keys above the parts' bounds, holds its support.  The first kernel, a workgroup per row, takes the members from there:
//   dP_j = dO v_j, u_j = p_j^(2 - alpha), delta = sum u dP / sum u, dX_j = u_j (dP_j - delta), dq = sum dX_j k_j / sqrt(D),
// reads their rows of V and K only, and leaves dX and 1 / sum p.  The second, a workgroup per 64 keys of a head, adds up dv = sum p dO and dk = sum dX q / sqrt(D) over the rows
// that have a key as a member, in the order of the rows, and writes zeros elsewhere: it is bound by those writes.  No product is formed for any other pair.
struct FewParams {
  SplitParams f;  // (of the forward; out: unused)
  const void* dout;
  void *dq, *dk, *dv;
  float* dx;    // [B * Hkv * R][splits][chunk], in the places of the entries
  float* zinv;  // [B * Hkv * R]
  float sm_scale;
};
// p and u = p^(2 - alpha) of a member
template <int AM> __device__ __forceinline__ void member_weights(float x, const RowsParams& rows, float& pr, float& u) {
  if constexpr (AM == AM_15) {
    u = x;
    pr = x * x;
  } else if constexpr (AM == AM_2) {
    u = 1.f;
    pr = x;
  } else {
    const float lg = fast_log2(x);
    u = fast_exp2(lg * (rows.c0 - 1.f));
    pr = u * x;
  }
}

// Lengths that are changed between a forward and its backward name places that the forward has not written: what is read there stays inside the tensors.
__device__ __forceinline__ int kept_count(const SplitParams& p, const Part& part) { return (unsigned)part.count < (unsigned)p.chunk ? part.count : p.chunk; }
__device__ __forceinline__ int kept_key(const SplitParams& p, int key) { return (unsigned)key < (unsigned)p.N ? key : 0; }

template <typename T, int D, int AM> __global__ __launch_bounds__(256) void few_rows_dq_kernel(FewParams fp) {
  using G = Gather<T, D>;
  const SplitParams& p = fp.f;
  constexpr int kLanes = G::kLanes, kVec = G::kVec, kB = G::kB, kGroups = 256 / kLanes, kAhead = 4;
  constexpr int kCap = 512;  // members to a wave's list
  __shared__ float sm[32];
  __shared__ float list_x[4][kCap], list_dp[4 * kCap];  // z - tau, dP
  __shared__ int list_key[4][kCap], list_at[4][kCap];
  __shared__ int totals[4];
  __shared__ float red[4][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x, unit = row / p.R, b = unit / p.Hkv, kvh = unit % p.Hkv, r = row % p.R;
  const int len = r % p.Nq < length_at(p.lens_q, p.lens_q_bits, b, p.Nq) ? length_at(p.lens, p.lens_bits, b, p.N) : 0;
  const int splits = (len + p.chunk - 1) / p.chunk;
  const Part* const parts = p.parts + (size_t)row * p.splits;
  const Entry* const entries = p.entries + (size_t)row * p.splits * p.chunk;
  float* const dx = fp.dx + (size_t)row * p.splits * p.chunk;
  const float tau = splits > 0 ? p.taus[row] : INFINITY, m = splits > 0 ? parts[0].max : 0.f;
  const int grp = tid / kLanes, col = tid % kLanes;
  G g(p, false, b, kvh, col);
  const char* const kbase = (const char*)p.k + (b * p.k_s0 + kvh * p.k_sh + col * kVec) * kB;
  auto row_k = [&](int key) { return *reinterpret_cast<const u32x4*>(kbase + key * p.k_sn * kB); };
  float dout[kVec];
  {
    const u32x4 raw = reinterpret_cast<const u32x4*>((const char*)fp.dout + (size_t)row * D * kB)[col];
#pragma unroll
    for (int e = 0; e < kVec; ++e) dout[e] = chunk_elem<T>(raw, e);
  }
  auto dot = [&](u32x4 raw) {  // dO v, in every lane of the group
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < kVec; ++e) x = fmaf(dout[e], chunk_elem<T>(raw, e), x);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
  };
  // ---- the members, a quarter of the parts to a wave ----
  const int per = (splits + 3) / 4, s0 = wave * per, s1 = s0 + per < splits ? s0 + per : splits;
  int mine = 0;
  for (int s = s0; s < s1; ++s) {
    const int count = kept_count(p, parts[s]);
    for (int i = 0; i < count; i += 256) {
      Entry e[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = i + v * 64 + lane;
        e[v] = entries[(size_t)s * p.chunk + (at < count ? at : 0)];
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = i + v * 64 + lane;
        const float x = e[v].z - m - tau;
        const bool in = at < count && x > 0.f;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
        const int place = mine + __builtin_popcountll(who & ((1ull << lane) - 1ull));
        if (in && place < kCap) {
          list_x[wave][place] = x;
          list_key[wave][place] = kept_key(p, e[v].key);
          list_at[wave][place] = s * p.chunk + at;
        }
        mine += __builtin_popcountll(who);
      }
    }
  }
  if (lane == 0) totals[wave] = mine;
  __syncthreads();
  const int n0 = totals[0], n1 = totals[1], n2 = totals[2], n3 = totals[3], n = n0 + n1 + n2 + n3;
  float sums[3] = {0.f, 0.f, 0.f}, delta;  // of u, u dP and p
  if (n0 <= kCap && n1 <= kCap && n2 <= kCap && n3 <= kCap) {
    auto place_of = [&](int j) {  // member j of the row in the four waves' lists
      int w = 0;
      if (j >= n0) j -= n0, w = kCap;
      if (w == kCap && j >= n1) j -= n1, w = 2 * kCap;
      if (w == 2 * kCap && j >= n2) j -= n2, w = 3 * kCap;
      return w + j;
    };
    const float* const xs = &list_x[0][0];
    const int* const keys = &list_key[0][0];
    for (int i = grp; i < n; i += kAhead * kGroups) {
      u32x4 raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u] = g.load(keys[place_of(i + u * kGroups < n ? i + u * kGroups : i)] * p.v_sn);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float x = dot(raw[u]);
        if (col == 0 && i + u * kGroups < n) list_dp[i + u * kGroups] = x;
      }
    }
    __syncthreads();
    for (int j = tid; j < n; j += 256) {
      float pr, u;
      member_weights<AM>(xs[place_of(j)], p.rows, pr, u);
      sums[0] += u;
      sums[1] = fmaf(u, list_dp[j], sums[1]);
      sums[2] += pr;
    }
    row_sum<256, 3>(sums, sm);
    delta = sums[0] > 0.f ? sums[1] / sums[0] : 0.f;
    for (int j = tid; j < n; j += 256) {
      float pr, u;
      const int at = place_of(j);
      member_weights<AM>(xs[at], p.rows, pr, u);
      const float x = u * (list_dp[j] - delta);
      list_dp[j] = x;
      dx[(&list_at[0][0])[at]] = x;
    }
    __syncthreads();
    for (int i = grp; i < n; i += kAhead * kGroups) {
      u32x4 raw[kAhead];
      float w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = i + u * kGroups;
        w[u] = j < n ? list_dp[j] : 0.f;
        raw[u] = row_k(keys[place_of(j < n ? j : i)]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * kGroups < n) g.add(w[u], raw[u]);
    }
  } else {
    // a flat row: the entries in memory are gone through three times; dP lies in dX's places until delta is known
    auto visit = [&](auto&& f) {  // f(place, z - tau, key) for the group's members
      for (int s = 0; s < splits; ++s) {
        const int count = kept_count(p, parts[s]);
        for (int i = grp; i < count; i += kGroups) {
          const Entry e = entries[(size_t)s * p.chunk + i];
          const float x = e.z - m - tau;
          if (x > 0.f) f((size_t)s * p.chunk + i, x, kept_key(p, e.key));
        }
      }
    };
    visit([&](size_t at, float x, int key) {
      const float dp = dot(g.load(key * p.v_sn));
      float pr, u;
      member_weights<AM>(x, p.rows, pr, u);
      if (col == 0) {
        sums[0] += u;
        sums[1] = fmaf(u, dp, sums[1]);
        sums[2] += pr;
        dx[at] = dp;
      }
    });
    row_sum<256, 3>(sums, sm);
    delta = sums[0] > 0.f ? sums[1] / sums[0] : 0.f;
    visit([&](size_t at, float x, int key) {  // (a group reads what a lane of its own wave wrote)
      float pr, u;
      member_weights<AM>(x, p.rows, pr, u);
      const float w = u * (dx[at] - delta);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (col == 0) dx[at] = w;
      g.add(w, row_k(key));
    });
  }
  if (tid == 0) fp.zinv[row] = sums[2] > 0.f ? 1.f / sums[2] : 0.f;
  g.join();
  if (lane < kLanes) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) red[wave][lane * kVec + e] = g.acc[e];
  }
  __syncthreads();
  for (int d = tid; d < D; d += 256) store_elem<T>(fp.dq, (size_t)row * D + d, (red[0][d] + red[1][d] + red[2][d] + red[3][d]) * fp.sm_scale);
}

constexpr int kFewKeys = 64;  // keys of a workgroup of the second kernel: a part's chunk is a multiple of it
template <typename T, int D, int AM> __global__ __launch_bounds__(256) void few_rows_dkdv_kernel(FewParams fp) {
  const SplitParams& p = fp.f;
  constexpr int kVec = elem_traits<T>::kVec, kB = elem_traits<T>::kBytes, kPieces = D / kVec;
  __shared__ float pr[kMaxRows][kFewKeys + 1], dx[kMaxRows][kFewKeys + 1];  // read where `rows` says so
  __shared__ unsigned long long rows[kFewKeys];                            // of each key, the rows that have it as a member
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int unit = blockIdx.x % p.units, key0 = (int)(blockIdx.x / p.units) * kFewKeys, b = unit / p.Hkv;
  const int len = length_at(p.lens, p.lens_bits, b, p.N), nq = length_at(p.lens_q, p.lens_q_bits, b, p.Nq);
  if (tid < kFewKeys) rows[tid] = 0ull;
  __syncthreads();
  if (key0 < len) {
    const int s = key0 / p.chunk;
    for (int r = wave; r < p.R; r += 4) {
      if (r % p.Nq >= nq) continue;
      const size_t row = (size_t)unit * p.R + r, at0 = (row * p.splits + s) * p.chunk;
      const float tau = p.taus[row], m = p.parts[row * p.splits].max, zinv = fp.zinv[row];
      const int count = kept_count(p, p.parts[row * p.splits + s]);
      for (int i = lane; i < count; i += 64) {
        const Entry e = p.entries[at0 + i];
        const int k = e.key - key0;
        const float x = e.z - m - tau;
        if (x > 0.f && k >= 0 && k < kFewKeys) {
          float w, u;
          member_weights<AM>(x, p.rows, w, u);
          pr[r][k] = w * zinv;
          dx[r][k] = fp.dx[at0 + i] * fp.sm_scale;
          atomicOr(&rows[k], 1ull << r);
        }
      }
    }
    __syncthreads();
  }
  const int n = p.N - key0 < kFewKeys ? p.N - key0 : kFewKeys;
  const size_t out0 = ((size_t)unit * p.N + key0) * kPieces;
  const u32x4* const q = reinterpret_cast<const u32x4*>((const char*)p.q + (size_t)unit * p.R * D * kB);
  const u32x4* const dout = reinterpret_cast<const u32x4*>((const char*)fp.dout + (size_t)unit * p.R * D * kB);
  for (int id = tid; id < n * kPieces; id += 256) {
    const int k = id / kPieces, c = id % kPieces;
    float ak[kVec], av[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) ak[e] = av[e] = 0.f;
    for (unsigned long long m = rows[k]; m; m &= m - 1) {
      const int r = __builtin_ctzll(m);
      const u32x4 qv = q[r * kPieces + c], dv = dout[r * kPieces + c];
      const float w = pr[r][k], x = dx[r][k];
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        ak[e] = fmaf(x, chunk_elem<T>(qv, e), ak[e]);
        av[e] = fmaf(w, chunk_elem<T>(dv, e), av[e]);
      }
    }
    u32x4 wk, wv;
    if constexpr (kVec == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wk[e] = __builtin_bit_cast(uint32_t, ak[e]);
        wv[e] = __builtin_bit_cast(uint32_t, av[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wk[e] = pack2<T>(ak[2 * e], ak[2 * e + 1]);
        wv[e] = pack2<T>(av[2 * e], av[2 * e + 1]);
      }
    }
    reinterpret_cast<u32x4*>(fp.dk)[out0 + id] = wk;
    reinterpret_cast<u32x4*>(fp.dv)[out0 + id] = wv;
  }
}

// Keys of a part: a power of two from 64 to kMaxChunk, as large as leaves two workgroups to a CU their LDS, and no larger than gives the
// chip some four workgroups a CU.
static int chunk_of(long long units, int R, int N) {
  int chunk = kMaxChunk;
  while (chunk > 64 && (size_t)R * score_stride(chunk) * 4 > 64 * 1024) chunk /= 2;
  while (chunk > 64 && units * ((N + chunk - 1) / chunk) < 1024) chunk /= 2;
  return chunk;
}
// (64 rows of K lie in a wave's registers)
constexpr int most_waves(int row_bytes) { return row_bytes <= 256 ? 16 : (row_bytes <= 512 ? 8 : 4); }
// Whether one workgroup takes all keys of a head (split_whole_kernel), and with how many waves.  A workgroup alone on its CU reads some 28 GB/s of K, whatever
// its waves: it saves a launch and the way through memory (some 4 us and what the second kernel takes), where the heads are enough to share out the CUs or K
// is short.  us, 32/8 heads, D = 128, bf16, split -> whole: 1 request of 600: 11.9, 13.5; 4 x 500: 11.6, 12.1; 4 x 2000: 15.2, 25.5; 16 x 500: 14.5 -> 12.3; 16 x 2000: 20.4, 25.8;
// 32 x 2000: 31.3 -> 27.8; 96 x 500: 33.0 -> 20.7; 256 x 1000: 104 -> 78; 16 heads, D = 64, f16: 8 x 1500: 15.6 -> 14.3, 32 x 1500: 22.0 -> 19.2.
// Waves: 16, 8, 4 at 8 x 600 keys 13.9, 12.8, 13.9; 512 heads of 1500, D = 64: 26.9, 19.4, 19.2; 2048 of 1000: 123, 82, 78.
static int whole_waves(long long units, int R, int N, int D, int row_bytes, int page, bool paged) {
  if (N > kMaxChunk || (long long)N * row_bytes > 2048 * (units > 64 ? units : 64)) return 0;
  int W = units <= 256 ? 16 : (units <= 512 ? 8 : 4);
  W = W < most_waves(row_bytes) ? W : most_waves(row_bytes);
  return whole_lds(R, (N + 63) / 64 * 64, page, paged, W, D) <= 150 * 1024 ? W : 0;
}
struct Workspace {
  int chunk, splits;
  size_t entries_off, total;
};
static Workspace workspace_of(long long B, long long Hkv, int R, int N) {
  Workspace w;
  w.chunk = chunk_of(B * Hkv, R, N);
  w.splits = (N + w.chunk - 1) / w.chunk;
  const size_t parts = (size_t)(B * Hkv) * R * w.splits;
  w.entries_off = (parts * sizeof(Part) + 255) / 256 * 256;
  w.total = w.entries_off + parts * w.chunk * sizeof(Entry);
  return w;
}

// Keys of a part where a prefix is shared: as many as leave two workgroups of a request to a CU their LDS, and give the chip two workgroups a CU where the rows do; but no more than 64 parts for that,
// which the second kernel goes through.  us, any number of parts -> 64: 7 requests x 2 heads behind 43623, D = 64: 30.0 -> 19.4; 2 x 16/4 behind 24168: 24.5 -> 19.1; 16 x 4/1 behind 16000: 22.8 -> 19.8.
static Workspace prefix_workspace_of(long long B, long long Hkv, int R, int N, int row_bytes, int prefix, int& parts) {
  const long long row_tiles = (B * R + 15) / 16;
  const bool few = B * R <= kFewRows;  // (the parts of few rows have up to 1024 keys, and 128 at least)
  const int least = few ? 128 : (2 * wave_keys(row_bytes) < 64 ? 64 : 2 * wave_keys(row_bytes));
  Workspace w;
  w.chunk = few ? 1024 : 8 * wave_keys(row_bytes);
  while (w.chunk > least && scores_lds(R, w.chunk, 1, true) > 64 * 1024) w.chunk /= 2;
  while (w.chunk > least && Hkv * row_tiles * ((prefix + w.chunk - 1) / w.chunk) < 512 && 2 * prefix <= 64 * w.chunk) w.chunk /= 2;
  parts = (prefix + w.chunk - 1) / w.chunk;
  w.splits = parts + (N - prefix + w.chunk - 1) / w.chunk;
  const size_t all = (size_t)(B * Hkv) * R * w.splits;
  w.entries_off = (all * sizeof(Part) + 255) / 256 * 256;
  w.total = w.entries_off + all * w.chunk * sizeof(Entry);
  return w;
}
template <typename T, int D, int AM, bool kPaged> static void launch(const SplitParams& p, long long units, hipStream_t s) {
  if constexpr (kPaged) {
    if (p.prefix_parts > 0) {
      prefix_scores_launch<T>(p, D, AM, s);
      hipLaunchKernelGGL((split_join_kernel<T, D, AM, true>), dim3((unsigned)(units * p.R)), dim3(256), 0, s, p);
      return;
    }
  }
  constexpr int kRowBytes = D * elem_traits<T>::kBytes, kMost = most_waves(kRowBytes);
  if (const int W = p.taus ? 0 : whole_waves(units, p.R, p.N, D, kRowBytes, p.page, kPaged)) {
    SplitParams q = p;
    q.chunk = (p.N + 63) / 64 * 64;
    const size_t lds = whole_lds(p.R, q.chunk, p.page, kPaged, W, D);
    if (W == 16) hipLaunchKernelGGL((split_whole_kernel<T, D, AM, kPaged, (kMost < 16 ? kMost : 16)>), dim3((unsigned)units), dim3(1024), lds, s, q);
    else if (W == 8) hipLaunchKernelGGL((split_whole_kernel<T, D, AM, kPaged, (kMost < 8 ? kMost : 8)>), dim3((unsigned)units), dim3(512), lds, s, q);
    else hipLaunchKernelGGL((split_whole_kernel<T, D, AM, kPaged, 4>), dim3((unsigned)units), dim3(256), lds, s, q);
    return;
  }
  const size_t lds = scores_lds(p.R, p.chunk, p.page, kPaged);
  hipLaunchKernelGGL((split_scores_kernel<T, D, AM, kPaged>), dim3((unsigned)(units * p.splits)), dim3(64 * kWaves), lds, s, p);
  hipLaunchKernelGGL((split_join_kernel<T, D, AM, kPaged>), dim3((unsigned)(units * p.R)), dim3(256), 0, s, p);
}
template <typename T, int D, bool kPaged> static void launch_am(const SplitParams& p, long long units, double alpha, hipStream_t s) {
  if (alpha == 1.5) launch<T, D, AM_15, kPaged>(p, units, s);
  else if (alpha == 2.0) launch<T, D, AM_2, kPaged>(p, units, s);
  else launch<T, D, AM_GEN, kPaged>(p, units, s);
}
template <typename T, bool kPaged> static void launch_d(const SplitParams& p, long long units, int D, double alpha, hipStream_t s) {
  if (D == 32) launch_am<T, 32, kPaged>(p, units, alpha, s);
  else if (D == 64) launch_am<T, 64, kPaged>(p, units, alpha, s);
  else if (D == 128) launch_am<T, 128, kPaged>(p, units, alpha, s);
  else launch_am<T, 256, kPaged>(p, units, alpha, s);
}
template <typename T, int D> static void launch_few(const FewParams& p, double alpha, hipStream_t s) {
  const dim3 rows((unsigned)(p.f.units * p.f.R)), keys((unsigned)((long long)p.f.units * ((p.f.N + kFewKeys - 1) / kFewKeys))), block(256);
  if (alpha == 1.5) {
    hipLaunchKernelGGL((few_rows_dq_kernel<T, D, AM_15>), rows, block, 0, s, p);
    hipLaunchKernelGGL((few_rows_dkdv_kernel<T, D, AM_15>), keys, block, 0, s, p);
  } else if (alpha == 2.0) {
    hipLaunchKernelGGL((few_rows_dq_kernel<T, D, AM_2>), rows, block, 0, s, p);
    hipLaunchKernelGGL((few_rows_dkdv_kernel<T, D, AM_2>), keys, block, 0, s, p);
  } else {
    hipLaunchKernelGGL((few_rows_dq_kernel<T, D, AM_GEN>), rows, block, 0, s, p);
    hipLaunchKernelGGL((few_rows_dkdv_kernel<T, D, AM_GEN>), keys, block, 0, s, p);
  }
}
template <typename T> static void launch_few_d(const FewParams& p, int D, double alpha, hipStream_t s) {
  if (D == 32) launch_few<T, 32>(p, alpha, s);
  else if (D == 64) launch_few<T, 64>(p, alpha, s);
  else if (D == 128) launch_few<T, 128>(p, alpha, s);
  else launch_few<T, 256>(p, alpha, s);
}
// What a call and its backward share.
static int place(SplitParams& p, long long B, int D, int row_bytes, double alpha, const void* workspace, size_t workspace_bytes) {
  const Workspace w = p.prefix > 0 ? prefix_workspace_of(B, p.Hkv, p.R, p.N, row_bytes, p.prefix, p.prefix_parts) : workspace_of(B, p.Hkv, p.R, p.N);
  if (!workspace || workspace_bytes < w.total || ((uintptr_t)workspace & 15) != 0) return ADSP_ERR_WORKSPACE;
  const long long units = B * p.Hkv;
  if (units * (p.N / kFewKeys + 1) >= (1ll << 31) || units * p.R >= (1ll << 31)) return ADSP_ERR_SHAPE;
  p.parts = (Part*)workspace;
  p.entries = (Entry*)((char*)workspace + w.entries_off);
  p.units = (int)units;
  p.chunk = w.chunk;
  p.splits = w.splits;
  if (p.prefix > 0 && (long long)p.Hkv * ((B * p.R + 15) / 16) * p.prefix_parts + units * p.splits + 256 >= (1ll << 31)) return ADSP_ERR_SHAPE;
  p.rows = RowsParams{};
  p.rows.scale = (float)((alpha - 1.0) / sqrt((double)D));
  p.rows.c0 = (float)(1.0 / (alpha - 1.0));
  p.rows.inv_c0 = (float)(alpha - 1.0);
  return ADSP_OK;
}
template <bool kPaged> static int run(SplitParams& p, long long B, int D, int dtype, double alpha, void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (const int rc = place(p, B, D, D * (dtype == ADSP_F32 ? 4 : 2), alpha, workspace, workspace_bytes)) return rc;
  const long long units = p.units;
  (void)hipGetLastError();
  if (dtype == ADSP_F32) launch_d<float, kPaged>(p, units, D, alpha, s);
  else if (dtype == ADSP_BF16) launch_d<bf16_t, kPaged>(p, units, D, alpha, s);
  else launch_d<f16_t, kPaged>(p, units, D, alpha, s);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
static bool rows_fit(int Hq, int Hkv, int q_len) { return Hkv > 0 && q_len > 0 && Hq > 0 && Hq % Hkv == 0 && (long long)(Hq / Hkv) * q_len <= kMaxRows; }
static int check(const void* q, const void* k, const void* v, const void* out, int B, int D, int dtype, double alpha, const int64_t (&strides)[6]) {
  if (!q || !k || !v || !out) return ADSP_ERR_NULL;
  if (dtype != ADSP_F32 && dtype != ADSP_BF16 && dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  if (B <= 0 || (D != 32 && D != 64 && D != 128 && D != 256)) return ADSP_ERR_SHAPE;
  if (!(alpha > 1.0) || alpha > 2.0) return ADSP_ERR_UNSUPPORTED;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) != 0) return ADSP_ERR_ALIGN;
  for (int64_t x : strides)
    if ((x * (dtype == ADSP_F32 ? 4 : 2) & 15) != 0) return ADSP_ERR_ALIGN;
  return ADSP_OK;
}
static bool bits_ok(const void* lens, int bits) { return !lens || bits == 32 || bits == 64; }
}  // namespace split
}  // namespace adsp

extern "C" size_t adsp_attn_split_workspace_bytes(int B, int Hq, int Hkv, int q_len, int k_len) {
  if (B <= 0 || k_len <= 0 || !adsp::split::rows_fit(Hq, Hkv, q_len)) return 0;
  return adsp::split::workspace_of(B, Hkv, Hq / Hkv * q_len, k_len).total;
}

// The keys of a prefix that are computed for all requests together, or 0: there are several requests, keys enough that it pays, and places in the workspace below 2^32 bytes.  us, 32/8 heads, D = 128, bf16, 50
// tokens behind the prefix, without -> with: 2 requests behind 200: 10.5, 12.2; 2000: 14.3 -> 12.9; 65500: 47.1 -> 46.1; 4 behind 500: 11.8, 12.5; 1000: 13.7 -> 12.6; 16 behind 500: 14.5, 15.4; 1000: 19.5 -> 15.7;
// 64 behind 1000: 25.5, 28.5; 2000: 47.8 -> 36.8; 8192: 140 -> 52; 200 x 16/4 heads, D = 64, behind 1000: 27.4, 34.6.
static int shared_keys(int B, int Hq, int Hkv, int row_bytes, int prefix_blocks, int page_size, int max_length) {
  const long long keys = (long long)prefix_blocks * page_size;
  const int prefix = (int)(keys < max_length ? keys : max_length);
  if (B <= 1 || prefix < 768 || prefix < 3 * (long long)B * Hkv) return 0;
  int parts;
  return adsp::split::prefix_workspace_of(B, Hkv, Hq / Hkv, max_length, row_bytes, prefix, parts).total < (1ull << 32) ? prefix : 0;
}

extern "C" size_t adsp_attn_paged_workspace_bytes(int B, int Hq, int Hkv, int D, int dtype, int max_length, int page_size, int prefix_blocks) {
  using namespace adsp::split;
  if (B <= 0 || D <= 0 || max_length <= 0 || page_size <= 0 || prefix_blocks < 0 || !rows_fit(Hq, Hkv, 1)) return 0;
  const int row_bytes = D * (dtype == ADSP_F32 ? 4 : 2), prefix = shared_keys(B, Hq, Hkv, row_bytes, prefix_blocks, page_size, max_length);
  int parts;
  return prefix > 0 ? prefix_workspace_of(B, Hkv, Hq / Hkv, max_length, row_bytes, prefix, parts).total : workspace_of(B, Hkv, Hq / Hkv, max_length).total;
}

extern "C" int adsp_attn_paged_shared_keys(int B, int Hq, int Hkv, int D, int dtype, int max_length, int page_size, int prefix_blocks) {
  using namespace adsp::split;
  if (B <= 0 || D <= 0 || max_length <= 0 || page_size <= 0 || prefix_blocks < 0 || !rows_fit(Hq, Hkv, 1)) return 0;
  return shared_keys(B, Hq, Hkv, D * (dtype == ADSP_F32 ? 4 : 2), prefix_blocks, page_size, max_length);
}

extern "C" int adsp_attn_paged_shared_parts(int B, int Hq, int Hkv, int D, int dtype, int max_length, int page_size, int prefix_blocks, int* part_keys, int* row_tiles) {
  using namespace adsp::split;
  const int prefix = adsp_attn_paged_shared_keys(B, Hq, Hkv, D, dtype, max_length, page_size, prefix_blocks);
  if (prefix == 0) return 0;
  const int row_bytes = D * (dtype == ADSP_F32 ? 4 : 2), R = Hq / Hkv;
  int parts;
  const Workspace w = prefix_workspace_of(B, Hkv, R, max_length, row_bytes, prefix, parts);
  if (part_keys) *part_keys = w.chunk;
  if (row_tiles) *row_tiles = (long long)B * R <= kFewRows ? 0 : prefix_row_tiles(((long long)B * R + 15) / 16, (long long)Hkv * parts, row_bytes);
  return parts;
}

static int paged_fwd(const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* block_tables, int64_t table_stride, const void* lengths,
                     int lengths_bits, const int32_t* prefix_table, int prefix_blocks, int B, int Hq, int Hkv, int D, int pages, int page_size, int max_length,
                     int64_t k_stride_page, int64_t k_stride_h, int64_t k_stride_n, int64_t v_stride_page, int64_t v_stride_h, int64_t v_stride_n, int dtype, double alpha,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace adsp::split;
  if (!block_tables || !lengths || (prefix_blocks > 0 && !prefix_table)) return ADSP_ERR_NULL;
  const int rc = check(q, k_pages, v_pages, out, B, D, dtype, alpha, {k_stride_page, k_stride_h, k_stride_n, v_stride_page, v_stride_h, v_stride_n});
  if (rc != ADSP_OK) return rc;
  if (!rows_fit(Hq, Hkv, 1) || pages <= 0 || page_size <= 0 || max_length <= 0 || max_length > (1 << 30) || prefix_blocks < 0) return ADSP_ERR_SHAPE;
  if (table_stride < (max_length - 1) / page_size + 1) return ADSP_ERR_SHAPE;
  if (!bits_ok(lengths, lengths_bits) || lengths_bits == 0) return ADSP_ERR_UNSUPPORTED;
  SplitParams p = {};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.out = out;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.lens = lengths;
  p.lens_bits = lengths_bits;
  p.prefix_table = prefix_table;
  p.prefix = shared_keys(B, Hq, Hkv, D * (dtype == ADSP_F32 ? 4 : 2), prefix_blocks, page_size, max_length);
  p.B = B;
  p.k_s0 = k_stride_page;
  p.k_sh = k_stride_h;
  p.k_sn = k_stride_n;
  p.v_s0 = v_stride_page;
  p.v_sh = v_stride_h;
  p.v_sn = v_stride_n;
  p.Hkv = Hkv;
  p.R = Hq / Hkv;
  p.Nq = 1;
  p.N = max_length;
  p.pages = pages;
  p.page = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  return run<true>(p, B, D, dtype, alpha, workspace, workspace_bytes, (hipStream_t)stream);
}
extern "C" int adsp_attn_paged_fwd(const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* block_tables,
                                   int64_t table_stride, const void* lengths, int lengths_bits, int B, int Hq, int Hkv, int D, int pages,
                                   int page_size, int max_length, int64_t k_stride_page, int64_t k_stride_h, int64_t k_stride_n,
                                   int64_t v_stride_page, int64_t v_stride_h, int64_t v_stride_n, int dtype, double alpha, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return paged_fwd(q, k_pages, v_pages, out, block_tables, table_stride, lengths, lengths_bits, nullptr, 0, B, Hq, Hkv, D, pages, page_size, max_length, k_stride_page,
                   k_stride_h, k_stride_n, v_stride_page, v_stride_h, v_stride_n, dtype, alpha, workspace, workspace_bytes, stream);
}
extern "C" int adsp_attn_paged_prefix_fwd(const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* block_tables,
                                          int64_t table_stride, const void* lengths, int lengths_bits, const int32_t* prefix_table, int prefix_blocks, int B, int Hq,
                                          int Hkv, int D, int pages, int page_size, int max_length, int64_t k_stride_page, int64_t k_stride_h,
                                          int64_t k_stride_n, int64_t v_stride_page, int64_t v_stride_h, int64_t v_stride_n, int dtype, double alpha,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  return paged_fwd(q, k_pages, v_pages, out, block_tables, table_stride, lengths, lengths_bits, prefix_table, prefix_blocks, B, Hq, Hkv, D, pages, page_size, max_length,
                   k_stride_page, k_stride_h, k_stride_n, v_stride_page, v_stride_h, v_stride_n, dtype, alpha, workspace, workspace_bytes, stream);
}

// Whether a workgroup per row and the split over the keys serve a call in less time than the kernels on blocks of 32 and 128 rows, which walk all keys with each of them: an
// estimate of both in us, the forward's and with `train` the gradients' with it.  Here a row costs its solves and its gathers, in single precision on slower products; there
// a block's walk is latency, and together they are matrix and vector work.  us, forward and gradients, theirs -> these: 1 x 8 heads, 16 queries, 2000 keys, D = 64, bf16: 20 + 35 -> 15 + 15;
// 64: 20 + 36, 32 + 23; 16 x 16, 16, 2000: 31 + 101, 41 + 62; 32: 31 + 102, 79 + 145; 16 x 32/8, 4, 1000, D = 128: 31 + 129 -> 19 + 34; 16: 31 + 129, 73 + 95; 2 x 16, 32, 8000: 72 + 94 -> 44 + 54;
// 64: 71 + 95, 91 + 104; 1 x 8, 64, 30000, D = 64: 151 + 83, 119 + 106; 8 x 16, 16, 300: 8 + 20, 10 + 22; fp32: 4 x 8, 16, 500: 18 + 21 -> 13 + 14; 64: 21 + 23, 40 + 32;
// 2 x 8, 32, 5000: 66 + 47 -> 43 + 40; 64: 67 + 49, 69 + 54; 16 x 16, 8, 1000: 27 + 88, 32 + 38; 28 x 24/12, 2, 442, D = 128: 42 + 69 -> 29 + 33.
extern "C" int adsp_attn_cross_few_rows(int B, int Hq, int Hkv, int q_len, int k_len, int D, int dtype, int train) {
  if (!adsp::split::rows_fit(Hq, Hkv, q_len) || (D != 32 && D != 64 && D != 128 && D != 256)) return 0;
  const bool wide = D > 64, f32 = dtype == ADSP_F32;
  const double N = k_len, R = Hq / Hkv * q_len, rows = (double)B * Hq * q_len, units = (double)B * Hkv, kv_us = units * N * D * (f32 ? 4 : 2) / 5e6;
  const double walk = (k_len + 31) / 32, row_blocks = (double)B * Hq * ((q_len + 31) / 32), blocks = row_blocks * walk;
  double few = 8 + 0.35 * R + rows * (1.5e-3 + (f32 ? 3e-6 + 6e-8 * D : 3e-6) * N) + kv_us, theirs;
  if (train) few += 9 + 0.2 * R + rows * (7e-3 + 1.6e-6 * N) + 2 * kv_us;
  if (f32) theirs = row_blocks <= 256 ? 10 + (wide ? 0.55 : 0.36) * walk : 10 + 0.6 * walk + (wide ? 2.3e-3 : 1.2e-3) * blocks;
  else if (k_len <= 2048) theirs = 6 + 0.2 * walk + 1e-3 * blocks;
  else theirs = row_blocks <= 256 ? 10 + 0.24 * walk : 10 + 0.3 * walk + 0.8e-3 * blocks;
  if (train) {
    if (f32) theirs += 16 + (wide ? 11e-3 : 9e-3) * units * walk + 1e-3 * rows;
    else if (k_len > 2048) theirs += 35 + 8e-3 * units * walk + 2e-3 * rows;
    else theirs += 15 + (wide ? 0.64 : 0.32) * walk + (wide ? 6e-3 : 4.5e-3) * blocks;
  }
  return few < theirs;
}

static int cross_step_params(adsp::split::SplitParams& p, const void* q, const void* k, const void* v, const void* out, const void* varlen_q, int varlen_q_bits,
                             const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int q_len, int k_len, int D, int dtype, double alpha) {
  using namespace adsp::split;
  const int rc = check(q, k, v, out, B, D, dtype, alpha, {0, 0, 0, 0, 0, 0});
  if (rc != ADSP_OK) return rc;
  if (!rows_fit(Hq, Hkv, q_len) || k_len <= 0 || k_len > (1 << 30)) return ADSP_ERR_SHAPE;
  if (!bits_ok(varlen_q, varlen_q_bits) || !bits_ok(varlen_k, varlen_k_bits)) return ADSP_ERR_UNSUPPORTED;
  p = SplitParams{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.lens = varlen_k;
  p.lens_bits = varlen_k_bits;
  p.lens_q = varlen_q;
  p.lens_q_bits = varlen_q_bits;
  p.k_s0 = p.v_s0 = (long long)Hkv * k_len * D;
  p.k_sh = p.v_sh = (long long)k_len * D;
  p.k_sn = p.v_sn = D;
  p.Hkv = Hkv;
  p.R = Hq / Hkv * q_len;
  p.Nq = q_len;
  p.N = k_len;
  p.page = 1;
  return ADSP_OK;
}

extern "C" int adsp_attn_cross_step_fwd(const void* q, const void* k, const void* v, void* out, float* taus, const void* varlen_q, int varlen_q_bits,
                                        const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int q_len, int k_len, int D, int dtype,
                                        double alpha, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace adsp::split;
  SplitParams p;
  const int rc = cross_step_params(p, q, k, v, out, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits, B, Hq, Hkv, q_len, k_len, D, dtype, alpha);
  if (rc != ADSP_OK) return rc;
  p.out = out;
  p.taus = taus;
  return run<false>(p, B, D, dtype, alpha, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t adsp_attn_cross_step_bwd_scratch_bytes(int B, int Hq, int Hkv, int q_len, int k_len) {
  if (B <= 0 || k_len <= 0 || !adsp::split::rows_fit(Hq, Hkv, q_len)) return 0;
  const adsp::split::Workspace w = adsp::split::workspace_of(B, Hkv, Hq / Hkv * q_len, k_len);
  return (size_t)B * Hq * q_len * ((size_t)w.splits * w.chunk + 1) * sizeof(float);
}

extern "C" int adsp_attn_cross_step_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus, const void* varlen_q, int varlen_q_bits,
                                        const void* varlen_k, int varlen_k_bits, void* dq, void* dk, void* dv, int B, int Hq, int Hkv, int q_len, int k_len, int D,
                                        int dtype, double alpha, const void* workspace, size_t workspace_bytes, void* scratch, size_t scratch_bytes, void* stream) {
  using namespace adsp::split;
  if (!dout || !taus || !dk || !dv) return ADSP_ERR_NULL;
  FewParams fp = {};
  int rc = cross_step_params(fp.f, q, k, v, dq, varlen_q, varlen_q_bits, varlen_k, varlen_k_bits, B, Hq, Hkv, q_len, k_len, D, dtype, alpha);
  if (rc != ADSP_OK) return rc;
  if ((((uintptr_t)dout | (uintptr_t)dk | (uintptr_t)dv) & 15) != 0) return ADSP_ERR_ALIGN;
  rc = place(fp.f, B, D, D * (dtype == ADSP_F32 ? 4 : 2), alpha, workspace, workspace_bytes);
  if (rc != ADSP_OK) return rc;
  if (!scratch || scratch_bytes < adsp_attn_cross_step_bwd_scratch_bytes(B, Hq, Hkv, q_len, k_len) || ((uintptr_t)scratch & 15) != 0) return ADSP_ERR_WORKSPACE;
  fp.f.taus = const_cast<float*>(taus);
  fp.dout = dout;
  fp.dq = dq;
  fp.dk = dk;
  fp.dv = dv;
  fp.dx = (float*)scratch;
  fp.zinv = fp.dx + (size_t)B * Hq * q_len * fp.f.splits * fp.f.chunk;
  fp.sm_scale = (float)(1.0 / sqrt((double)D));
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  if (dtype == ADSP_F32) launch_few_d<float>(fp, D, alpha, s);
  else if (dtype == ADSP_BF16) launch_few_d<adsp::bf16_t>(fp, D, alpha, s);
  else launch_few_d<adsp::f16_t>(fp, D, alpha, s);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
