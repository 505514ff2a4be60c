// Pages of a cache that change hands, without a trip to the host: requests that go on from others or end (fork), and the pages that requests hold moved into another
// pool (compact).
//
// fork: request b goes on from parent(b), or ends where that names no request.  With len(s) tokens of s before the step, P slots a page, full(s) = len / P, rest(s) = len % P,
// C(s) the requests that go on from s, and shares[page] the requests that hold a page less one:
//   full pages of s: shares += |C(s)| - 1;  its last, partly filled page goes to s where s goes on from itself, else to the first of C(s) (the heir); the others of C(s) get a page of their
//   own with its rest(s) tokens copied, in the order of their numbers; where C(s) is empty, shares of all its pages -= 1.
//   A page whose shares fall to -1 is free: behind the free list's end, in the order of the requests that held it (the first of them) and of their tables; where the ring has no entry left for it
//   (one of fewer entries than pages) it keeps the -1 and is in no list.
//   Pages for copies come from the list's front, those just freed among them.  Where none is left a request has its full(s) pages only.
// What bounds it is latency: the launches hand sums over requests to one another (holders -> first holder of what is free -> how many -> where they go -> tables and copies), each a
// microsecond or two; and the copied rows, where they are many.
//
// compact: pages numbered by the first request, and place in its table, that holds them; a table cut off in front of the first page that the other pool has no room for.
// Bound by the copy of the pages.
#include "common.h"
#include "../../include/adasplash_hip.h"

namespace adsp {
namespace paged {
namespace {
constexpr int kThreads = 256;
constexpr int kMaxRequests = 8192;

__device__ __forceinline__ long long number_at(const void* x, int bits, long long i) { return bits == 64 ? ((const long long*)x)[i] : (long long)((const int*)x)[i]; }
__device__ __forceinline__ int held_at(const void* lengths, int bits, int b, long long limit) {
  const long long l = number_at(lengths, bits, b);
  return (int)(l < 0 ? 0 : (l < limit ? l : limit));
}

// Sums over a workgroup of 256, the same in every thread.
template <int N> __device__ __forceinline__ void block_sums(int (&v)[N]) {
  __shared__ int part[N][kThreads / 64];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = wave_sum_i(v[i]);
    if ((threadIdx.x & 63) == 0) part[i][threadIdx.x >> 6] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = part[i][0] + part[i][1] + part[i][2] + part[i][3];
}
// f(i, whether item i counts, its place among those that count): items 0 .. n - 1 in their order, in steps of the workgroup; returns how many count.
template <typename Counts, typename F> __device__ __forceinline__ int in_order(int n, Counts&& counts, F&& f) {
  __shared__ int totals[2][kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int before = 0, turn = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += kThreads, turn ^= 1) {
    const int i = i0 + tid;
    const bool in = i < n && counts(i);
    const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
    if (lane == 0) totals[turn][wave] = __builtin_popcountll(who);
    __syncthreads();
    int at = before + __builtin_popcountll(who & ((1ull << lane) - 1ull));
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < wave) at += totals[turn][w];
      before += totals[turn][w];
    }
    if (i < n) f(i, in, at);
  }
  return before;
}

// Rows of pages copied: what both operations do with K and V.
struct PageRows {
  const char *k, *v;
  char *k_to, *v_to;
  long long k_p, k_h, k_s, v_p, v_h, v_s;              // bytes: page, head, slot
  long long kt_p, kt_h, kt_s, vt_p, vt_h, vt_s;
  int heads, pieces;  // pieces of 16 bytes in a row
};
// The first `rows` slots of page `from` to page `to`; the pieces first, first + step, ... of the page.
__device__ __forceinline__ void copy_page(const PageRows& p, long long from, long long to, int rows, int first, int step) {
  constexpr int kAhead = 4;
  const int all = p.heads * rows * p.pieces;
  const char *const k = p.k + from * p.k_p, *const v = p.v + from * p.v_p;
  char *const kt = p.k_to + to * p.kt_p, *const vt = p.v_to + to * p.vt_p;
  for (int i = first; i < all; i += kAhead * step) {
    u32x4 a[kAhead], b[kAhead];
    int h[kAhead], s[kAhead], c[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = i + u * step < all ? i + u * step : i, row = j / p.pieces;
      c[u] = (j - row * p.pieces) * 16;
      h[u] = row / rows;
      s[u] = row - h[u] * rows;
      a[u] = *reinterpret_cast<const u32x4*>(k + h[u] * p.k_h + s[u] * p.k_s + c[u]);
      b[u] = *reinterpret_cast<const u32x4*>(v + h[u] * p.v_h + s[u] * p.v_s + c[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i + u * step < all) {
        *reinterpret_cast<u32x4*>(kt + h[u] * p.kt_h + s[u] * p.kt_s + c[u]) = a[u];
        *reinterpret_cast<u32x4*>(vt + h[u] * p.vt_h + s[u] * p.vt_s + c[u]) = b[u];
      }
  }
}

// ---- fork -------------------------------------------------------------------------------------------------------------
struct ForkParams {
  const void* parents;
  void* lengths;
  int parents_bits, lengths_bits;
  int* tables;
  long long table_stride;
  int* free_pages;
  long long* free_range;
  int* shares;
  PageRows rows;
  int B, width, page, free_entries, pages;
  // scratch
  int* old;       // [B][width]: tables before the step, the entries that are held
  int* len;       // [B]: tokens before the step
  int* children;  // [B]: requests that go on from one
  int* heir;      // [B]
  int* freed;     // [B]: pages that are free behind the step, of which the request is the first holder
  int* copies;    // [B]: 1 where a request needs a page for a copy
  int* place;     // [B]: the place of that page in the free list, or -1
  long long* range;  // first free, end behind what is freed, pages for copies
};
__device__ __forceinline__ int parent_of(const ForkParams& p, int b) {
  const long long s = number_at(p.parents, p.parents_bits, b);
  return s >= 0 && s < p.B ? (int)s : -1;
}
__device__ __forceinline__ bool in_cache(const ForkParams& p, int id) { return (unsigned)id < (unsigned)p.pages; }
// Entries of the ring that hold no free page.
__device__ __forceinline__ long long ring_room(const ForkParams& p, long long first, long long end) {
  const long long room = p.free_entries - (end - first);
  return room > 0 ? room : 0;
}
// What marks a free page with its first holder: the lowest number wins, and a mark is below -1.
__device__ __forceinline__ int mark_of(const ForkParams& p, int b) { return -2 - (p.B - 1 - b); }

// Workgroup (g, slice): who goes on from requests kGroup g and behind, and the holders of a slice of their pages.  Requests side by side often hold the same page at the same place, and atomics on one word
// wait for each other: a run of them is added up first.  us, 256 requests with the same 128 pages, a request to a workgroup and eight: 12.1, 5.1.
constexpr int kGroup = 8;
__global__ __launch_bounds__(kThreads) void fork_holders_kernel(ForkParams p) {
  const int s0 = blockIdx.x * kGroup, tid = threadIdx.x;
  __shared__ int children[kGroup], heir[kGroup], len[kGroup], full[kGroup], held[kGroup];
  if (tid < kGroup) {
    children[tid] = 0;
    heir[tid] = p.B;
    len[tid] = s0 + tid < p.B ? held_at(p.lengths, p.lengths_bits, s0 + tid, (long long)p.width * p.page) : 0;
    full[tid] = len[tid] / p.page;
    held[tid] = (len[tid] + p.page - 1) / p.page;
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += kThreads) {
    const int s = parent_of(p, b), at = s - s0;
    if (s >= 0 && (unsigned)at < (unsigned)kGroup) {
      atomicAdd(&children[at], 1);
      atomicMin(&heir[at], b == s ? -1 : b);
    }
  }
  __syncthreads();
  if (blockIdx.y == 0 && tid < kGroup && s0 + tid < p.B) {
    p.len[s0 + tid] = len[tid];
    p.children[s0 + tid] = children[tid];
    p.heir[s0 + tid] = heir[tid] < 0 ? s0 + tid : heir[tid];
  }
  for (int i = blockIdx.y * kThreads + tid; i < p.width; i += gridDim.y * kThreads) {
    int id[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) id[u] = i < held[u] ? p.tables[(s0 + u) * p.table_stride + i] : -1;
    int page = -1, sum = 0;
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      if (i < held[u]) p.old[(long long)(s0 + u) * p.width + i] = id[u];
      if (!in_cache(p, id[u])) continue;
      const int more = i < full[u] ? children[u] - 1 : (children[u] > 0 ? 0 : -1);
      if (id[u] != page) {
        if (sum != 0) atomicAdd(p.shares + page, sum);
        page = id[u];
        sum = 0;
      }
      sum += more;
    }
    if (sum != 0) atomicAdd(p.shares + page, sum);
  }
}
// Workgroup s, of a request that no one goes on from: a mark on those of its pages that no one holds.
__global__ __launch_bounds__(kThreads) void fork_mark_kernel(ForkParams p) {
  const int s = blockIdx.x;
  if (p.children[s] > 0) return;
  const int n = (p.len[s] + p.page - 1) / p.page, mark = mark_of(p, s);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int id = p.old[(long long)s * p.width + i];
    if (in_cache(p, id) && __hip_atomic_load(p.shares + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < 0) atomicMin(p.shares + id, mark);
  }
}
// Workgroup b: how many pages carry its mark, and whether it needs one.
__global__ __launch_bounds__(kThreads) void fork_count_kernel(ForkParams p) {
  const int b = blockIdx.x, tid = threadIdx.x;
  int sums[1] = {0};
  if (p.children[b] == 0) {
    const int n = (p.len[b] + p.page - 1) / p.page, mark = mark_of(p, b);
    for (int i = tid; i < n; i += kThreads) {
      const int id = p.old[(long long)b * p.width + i];
      sums[0] += in_cache(p, id) && p.shares[id] == mark ? 1 : 0;
    }
  }
  block_sums(sums);
  if (tid == 0) {
    p.freed[b] = sums[0];
    const int s = parent_of(p, b);
    bool copy = s >= 0 && p.heir[s] != b && p.len[s] % p.page > 0;
    if (copy) copy = in_cache(p, p.old[(long long)s * p.width + p.len[s] / p.page]);
    p.copies[b] = copy ? 1 : 0;
  }
}
// Workgroup b: its marked pages to the free list, and the place of the page that it copies to.
__global__ __launch_bounds__(kThreads) void fork_free_kernel(ForkParams p) {
  const int b = blockIdx.x, tid = threadIdx.x;
  int sums[4] = {0, 0, 0, 0};
  for (int i = tid; i < p.B; i += kThreads) {
    const int n = p.freed[i], c = p.copies[i];
    sums[0] += i < b ? n : 0;
    sums[1] += n;
    sums[2] += i < b ? c : 0;
    sums[3] += c;
  }
  block_sums(sums);
  const long long first = p.free_range[0] > 0 ? p.free_range[0] : 0, end = p.free_range[1] > first ? p.free_range[1] : first;
  const long long room = ring_room(p, first, end);
  if (b == 0 && tid == 0) {
    p.range[0] = first;
    p.range[1] = end + (sums[1] < room ? sums[1] : room);
    p.range[2] = sums[3];
  }
  if (tid == 0) p.place[b] = p.copies[b] ? sums[2] : -1;
  if (p.freed[b] == 0) return;
  const int n = (p.len[b] + p.page - 1) / p.page, mark = mark_of(p, b);
  const int* const row = p.old + (long long)b * p.width;
  in_order(
      n, [&](int i) { return in_cache(p, row[i]) && p.shares[row[i]] == mark; },
      [&](int i, bool in, int at) {
        if (!in) return;
        if (sums[0] + at < room) p.free_pages[(end + sums[0] + at) % p.free_entries] = row[i];
        else p.shares[row[i]] = -1;
      });
  __syncthreads();
  for (int i = tid; i < n; i += kThreads)
    if (in_cache(p, row[i]) && p.shares[row[i]] == mark) p.shares[row[i]] = 0;
}
// Workgroup (b, slice): its table and length, and a slice of the rows it copies.
__global__ __launch_bounds__(kThreads) void fork_tables_kernel(ForkParams p) {
  const int b = blockIdx.x, tid = threadIdx.x;
  const long long first = p.range[0], end = p.range[1];
  const int s = parent_of(p, b), place = p.place[b];
  const long long avail = end - first < p.free_entries ? end - first : p.free_entries;
  if (b == 0 && blockIdx.y == 0 && tid == 0) {
    p.free_range[0] = first + (p.range[2] < avail ? p.range[2] : avail);
    p.free_range[1] = end;
  }
  if (place >= 0) {
    const int held = p.len[s], full = held / p.page, rest = held % p.page;
    int id = place < avail ? p.free_pages[(first + place) % p.free_entries] : -1;
    if (!in_cache(p, id)) id = -1;
    if (blockIdx.y == 0) {
      int* const row = p.tables + b * p.table_stride;
      for (int i = tid; i < p.width; i += kThreads) row[i] = i < full ? p.old[(long long)s * p.width + i] : (i == full ? id : -1);
      if (tid == 0) {
        const long long after = id >= 0 ? held : (long long)full * p.page;
        if (p.lengths_bits == 64) ((long long*)p.lengths)[b] = after;
        else ((int*)p.lengths)[b] = (int)after;
      }
    }
    if (id >= 0) copy_page(p.rows, p.old[(long long)s * p.width + full], id, rest, blockIdx.y * kThreads + tid, gridDim.y * kThreads);
    return;
  }
  if (blockIdx.y > 0 || s == b) return;
  const int held = s >= 0 ? p.len[s] : 0, n = (held + p.page - 1) / p.page;
  int* const row = p.tables + b * p.table_stride;
  for (int i = tid; i < p.width; i += kThreads) row[i] = i < n ? p.old[(long long)s * p.width + i] : -1;
  if (tid == 0) {
    if (p.lengths_bits == 64) ((long long*)p.lengths)[b] = held;
    else ((int*)p.lengths)[b] = held;
  }
}

// A barrier behind which the workgroup's stores and atomics in memory have been done: __syncthreads waits for LDS only, and leaves the order of what is under way in memory to the compute unit.
__device__ __forceinline__ void settled_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
// The four kernels above as one workgroup, where the tables are small: entries side by side, a few to a thread, in registers, and barriers instead of launches.
// us a call with its copies, pages of 16 tokens, one head of 32, requests x entries of a table, one workgroup, four launches: 4 x 32: 9.0, 15.8; 64 x 32: 11.2, 17.2; 64 x 64: 12.9, 17.5; 512 x 8: 14.7, 18.0;
// 1024 x 4: 16.2, 20.2; 64 x 80: 13.6, 17.2; 64 x 96: 14.6, 17.4; 384 x 16: 19.3, 18.2; 64 x 128: 15.9, 17.3.
constexpr int kSmallThreads = 1024, kSmallRequests = 1024, kForkEach = 5, kCompactEach = 4;
__global__ __launch_bounds__(kSmallThreads) void fork_small_kernel(ForkParams p) {
  constexpr int kWavesHere = kSmallThreads / 64;
  __shared__ int len[kSmallRequests], parent[kSmallRequests], children[kSmallRequests], heir[kSmallRequests], full[kSmallRequests], held[kSmallRequests];
  __shared__ unsigned long long masks[kWavesHere][kForkEach];
  __shared__ int totals[kWavesHere];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long first = p.free_range[0] > 0 ? p.free_range[0] : 0, end = p.free_range[1] > first ? p.free_range[1] : first;
  if (tid < p.B) {
    len[tid] = held_at(p.lengths, p.lengths_bits, tid, (long long)p.width * p.page);
    parent[tid] = parent_of(p, tid);
    full[tid] = len[tid] / p.page;  // whole pages, and all
    held[tid] = (len[tid] + p.page - 1) / p.page;
    children[tid] = 0;
    heir[tid] = p.B;
  }
  // entry u of a thread: a wave has `each` runs of 64 entries, one behind the other
  const int all = p.B * p.width, each = (all + kSmallThreads - 1) / kSmallThreads, base = wave * (64 * each) + lane;
  const float inv_width = 1.f / (float)p.width;
  auto row_of = [&](int e) { return (int)(((float)e + 0.5f) * inv_width); };  // (below 2^14: off by less than half an entry)
  int id[kForkEach];
#pragma unroll
  for (int u = 0; u < kForkEach; ++u) {
    id[u] = -1;
    if (u < each) {
      const int e = base + u * 64, s = row_of(e);
      if (e < all) id[u] = p.tables[s * p.table_stride + (e - s * p.width)];
    }
  }
  __syncthreads();
  if (tid < p.B && parent[tid] >= 0) {
    atomicAdd(&children[parent[tid]], 1);
    atomicMin(&heir[parent[tid]], parent[tid] == tid ? -1 : tid);
  }
  __syncthreads();
  if (tid < p.B && heir[tid] < 0) heir[tid] = tid;
  // (shares change by atomics, which act in L2: read there)
  auto share = [&](int page) { return __hip_atomic_load(p.shares + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  uint32_t dropped = 0;  // of the thread's entries, those of requests that no one goes on from
#pragma unroll
  for (int u = 0; u < kForkEach; ++u) {
    const int e = base + u * 64, s = u < each && e < all ? row_of(e) : 0, i = e - s * p.width;
    if (u < each && e < all && i < held[s]) {
      p.old[e] = id[u];
      const int more = i < full[s] ? children[s] - 1 : (children[s] > 0 ? 0 : -1);
      if (in_cache(p, id[u])) {
        if (more != 0) atomicAdd(p.shares + id[u], more);
        dropped |= children[s] == 0 ? 1u << u : 0u;
      }
    }
  }
  settled_barrier();
  uint32_t free = 0;
#pragma unroll
  for (int u = 0; u < kForkEach; ++u)
    if (dropped >> u & 1) free |= share(id[u]) < 0 ? 1u << u : 0u;
  settled_barrier();  // (marks are below 0 too: all have looked)
#pragma unroll
  for (int u = 0; u < kForkEach; ++u)
    if (free >> u & 1) atomicMin(p.shares + id[u], mark_of(p, row_of(base + u * 64)));
  settled_barrier();
  int mine = 0;
#pragma unroll
  for (int u = 0; u < kForkEach; ++u) {
    if (u >= each) break;
    const bool in = (free >> u & 1) && share(id[u]) == mark_of(p, row_of(base + u * 64));
    const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
    if (lane == 0) masks[wave][u] = who;
    mine += __builtin_popcountll(who);
  }
  if (lane == 0) totals[wave] = mine;
  __syncthreads();
  const long long room = ring_room(p, first, end);
  int at = 0, freed = 0;
  for (int w = 0; w < kWavesHere; ++w) {
    at += w < wave ? totals[w] : 0;
    freed += totals[w];
  }
#pragma unroll
  for (int u = 0; u < kForkEach; ++u) {
    if (u >= each) break;
    const unsigned long long who = masks[wave][u];
    if (who >> lane & 1) {
      const int to = at + __builtin_popcountll(who & ((1ull << lane) - 1ull));
      if (to < room) p.free_pages[(end + to) % p.free_entries] = id[u];
      __hip_atomic_store(p.shares + id[u], to < room ? 0 : -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    at += __builtin_popcountll(who);
  }
  bool copy = false;
  if (tid < p.B) {
    const int s = parent[tid];
    copy = s >= 0 && heir[s] != tid && full[s] < held[s];
    if (copy) copy = in_cache(p, p.tables[s * p.table_stride + full[s]]);
    p.len[tid] = len[tid];
  }
  const unsigned long long who = __builtin_amdgcn_ballot_w64(copy);
  __syncthreads();  // (the totals have been read)
  if (lane == 0) totals[wave] = __builtin_popcountll(who);
  __syncthreads();
  int place = __builtin_popcountll(who & ((1ull << lane) - 1ull)), copies = 0;
  for (int w = 0; w < kWavesHere; ++w) {
    place += w < wave ? totals[w] : 0;
    copies += totals[w];
  }
  if (tid < p.B) p.place[tid] = copy ? place : -1;
  if (tid == 0) {
    p.range[0] = first;
    p.range[1] = end + (freed < room ? freed : room);
    p.range[2] = copies;
  }
}

// ---- compact ----------------------------------------------------------------------------------------------------------
struct CompactParams {
  const void* lengths;
  void* lengths_to;
  int bits;
  const int* tables;
  long long table_stride;
  int* tables_to;  // [B][width]
  int* shares_to;  // [room]
  int* free_to;    // [room]
  long long* range_to;
  PageRows rows;
  int B, width, page, pages, room;
  // scratch
  unsigned long long* seen;  // [pages]: the lowest request and place (b width + i) that hold a page
  int* number;               // [pages]
  int* of;                   // [room]: the page that a number is of
  int* count;                // [B]: pages of which a request is the first holder
};
__device__ __forceinline__ int held_page(const CompactParams& p, int b, int i) {
  const int id = p.tables[b * p.table_stride + i];
  return (unsigned)id < (unsigned)p.pages ? id : -1;
}
__device__ __forceinline__ int held_pages(const CompactParams& p, int b) { return (held_at(p.lengths, p.bits, b, (long long)p.width * p.page) + p.page - 1) / p.page; }
__global__ __launch_bounds__(kThreads) void compact_clear_kernel(CompactParams p) {
  const long long step = (long long)gridDim.x * kThreads;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < p.pages || i < p.room; i += step) {
    if (i < p.pages) p.seen[i] = ~0ull;
    if (i < p.room) p.shares_to[i] = 0;
  }
}
__global__ __launch_bounds__(kThreads) void compact_mark_kernel(CompactParams p) {
  const int b = blockIdx.x, n = held_pages(p, b);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int id = held_page(p, b, i);
    if (id >= 0) atomicMin(p.seen + id, (unsigned long long)b * p.width + i);
  }
}
__device__ __forceinline__ bool is_first(const CompactParams& p, int b, int i) {
  const int id = held_page(p, b, i);
  return id >= 0 && p.seen[id] == (unsigned long long)b * p.width + i;
}
__global__ __launch_bounds__(kThreads) void compact_count_kernel(CompactParams p) {
  const int b = blockIdx.x, n = held_pages(p, b);
  int sums[1] = {0};
  for (int i = threadIdx.x; i < n; i += kThreads) sums[0] += is_first(p, b, i) ? 1 : 0;
  block_sums(sums);
  if (threadIdx.x == 0) p.count[b] = sums[0];
}
__global__ __launch_bounds__(kThreads) void compact_number_kernel(CompactParams p) {
  const int b = blockIdx.x, tid = threadIdx.x;
  int sums[1] = {0};
  for (int i = tid; i < b; i += kThreads) sums[0] += p.count[i];
  block_sums(sums);
  in_order(
      held_pages(p, b), [&](int i) { return is_first(p, b, i); },
      [&](int i, bool in, int at) {
        if (!in) return;
        const int id = held_page(p, b, i), n = sums[0] + at;
        p.number[id] = n;
        if (n < p.room) p.of[n] = id;
      });
}
// First holders, their number and the pages' numbers as one workgroup, where the tables are small: entries side by side as in a fork, and only the words of held pages cleared.
// us a call, requests x entries of a table, pages, one workgroup, four launches: 4 x 32, 128: 8.0, 11.3; 4 x 32, 65536: 10.8, 12.4; 64 x 16, 1024: 9.3, 12.3; 1024 x 1, 1024: 11.3, 15.4; 64 x 32, 2048: 11.9, 14.0;
// 64 x 64, 4096: 16.6, 16.9; 1024 x 4, 4096: 19.2, 20.7; 64 x 96, 6144: 19.9, 18.4; 64 x 256, 16384: 39.0, 28.5.
constexpr int kSmallRoom = 65536;
__global__ __launch_bounds__(kSmallThreads) void compact_small_kernel(CompactParams p) {
  constexpr int kWavesHere = kSmallThreads / 64;
  __shared__ int held[kSmallRequests];
  __shared__ int totals[kWavesHere];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < p.B) held[tid] = held_pages(p, tid);
  for (int i = tid; i < p.room; i += kSmallThreads) p.shares_to[i] = 0;
  __syncthreads();
  const int all = p.B * p.width, each = (all + kSmallThreads - 1) / kSmallThreads, base = wave * (64 * each) + lane;
  const float inv_width = 1.f / (float)p.width;
  auto row_of = [&](int e) { return (int)(((float)e + 0.5f) * inv_width); };  // (below 2^14: off by less than half an entry)
  int id[kCompactEach];
#pragma unroll
  for (int u = 0; u < kCompactEach; ++u) {
    const int e = base + u * 64, b = u < each && e < all ? row_of(e) : 0, i = e - b * p.width;
    id[u] = u < each && e < all && i < held[b] ? held_page(p, b, i) : -1;
    if (id[u] >= 0) __hip_atomic_store(p.seen + id[u], ~0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  settled_barrier();
#pragma unroll
  for (int u = 0; u < kCompactEach; ++u)
    if (id[u] >= 0) atomicMin(p.seen + id[u], (unsigned long long)(base + u * 64));
  settled_barrier();
  uint32_t firsts = 0;
  int mine = 0;
#pragma unroll
  for (int u = 0; u < kCompactEach; ++u) {
    const unsigned long long e = (unsigned long long)(base + u * 64);
    const bool in = id[u] >= 0 && __hip_atomic_load(p.seen + id[u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == e;
    firsts |= in ? 1u << u : 0u;
    mine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
  }
  if (lane == 0) totals[wave] = mine;
  __syncthreads();
  int at = 0, used = 0;
  for (int w = 0; w < kWavesHere; ++w) {
    at += w < wave ? totals[w] : 0;
    used += totals[w];
  }
#pragma unroll
  for (int u = 0; u < kCompactEach; ++u) {
    const bool in = firsts >> u & 1;
    const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
    if (in) {
      const int number = at + __builtin_popcountll(who & ((1ull << lane) - 1ull));
      p.number[id[u]] = number;
      if (number < p.room) p.of[number] = id[u];
    }
    at += __builtin_popcountll(who);
  }
  if (tid < p.B) p.count[tid] = tid == 0 ? used : 0;  // (what follows takes their sum)
}
// The first B workgroups: tables, lengths and holders; the others: the pages, one after another.
__global__ __launch_bounds__(kThreads) void compact_move_kernel(CompactParams p, int copiers) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < p.B) {
    const int b = blockIdx.x, held = held_at(p.lengths, p.bits, b, (long long)p.width * p.page), n = (held + p.page - 1) / p.page;
    __shared__ int cut;
    if (tid == 0) cut = n;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const int id = held_page(p, b, i);
      if (id >= 0 && p.number[id] >= p.room) atomicMin(&cut, i);
    }
    __syncthreads();
    const int m = cut;
    for (int i = tid; i < p.width; i += kThreads) {
      const int id = i < m ? held_page(p, b, i) : -1, to = id >= 0 ? p.number[id] : -1;
      p.tables_to[(long long)b * p.width + i] = to;
      // (numbers rise along a request's first-held pages: a page in front of the cut is in front of its first holder's too)
      if (to >= 0 && !is_first(p, b, i)) atomicAdd(p.shares_to + to, 1);
    }
    if (tid == 0) {
      const long long after = m < n ? (long long)m * p.page : held;
      if (p.bits == 64) ((long long*)p.lengths_to)[b] = after;
      else ((int*)p.lengths_to)[b] = (int)after;
    }
    return;
  }
  int sums[1] = {0};
  for (int i = tid; i < p.B; i += kThreads) sums[0] += p.count[i];
  block_sums(sums);
  const int at = blockIdx.x - p.B, used = sums[0] < p.room ? sums[0] : p.room;
  for (long long i = (long long)at * kThreads + tid; i < p.room; i += (long long)copiers * kThreads) p.free_to[i] = (int)((i + used) % p.room);
  if (at == 0 && tid == 0) {
    p.range_to[0] = 0;
    p.range_to[1] = p.room - used;
  }
  for (int n = at; n < used; n += copiers) copy_page(p.rows, p.of[n], n, p.page, tid, kThreads);
}
size_t align(size_t n) { return (n + 255) / 256 * 256; }
int check_rows(int dtype, int heads, int D, int page_size, const int64_t* strides, int n, std::initializer_list<const void*> pointers) {
  if (dtype != ADSP_F32 && dtype != ADSP_BF16 && dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  const int es = dtype == ADSP_F32 ? 4 : 2;
  if (heads <= 0 || D <= 0 || page_size <= 0 || D * es % 16 != 0 || (long long)heads * page_size * (D * es / 16) >= (1ll << 30)) return ADSP_ERR_SHAPE;
  uintptr_t all = 0;
  for (const void* x : pointers) {
    if (!x) return ADSP_ERR_NULL;
    all |= (uintptr_t)x;
  }
  int64_t st = 0;
  for (int i = 0; i < n; ++i) st |= strides[i] * es;
  return ((all | (uintptr_t)st) & 15) != 0 ? ADSP_ERR_ALIGN : ADSP_OK;
}
PageRows page_rows(const void* k, const void* v, void* k_to, void* v_to, int heads, int D, const int64_t* from, const int64_t* to, int dtype) {
  const int64_t es = dtype == ADSP_F32 ? 4 : 2;
  PageRows r;
  r.k = (const char*)k;
  r.v = (const char*)v;
  r.k_to = (char*)k_to;
  r.v_to = (char*)v_to;
  r.k_p = from[0] * es, r.k_h = from[1] * es, r.k_s = from[2] * es, r.v_p = from[3] * es, r.v_h = from[4] * es, r.v_s = from[5] * es;
  r.kt_p = to[0] * es, r.kt_h = to[1] * es, r.kt_s = to[2] * es, r.vt_p = to[3] * es, r.vt_h = to[4] * es, r.vt_s = to[5] * es;
  r.heads = heads;
  r.pieces = (int)(D * es / 16);
  return r;
}
bool requests_fit(int B, int width, int page_size) { return B > 0 && B <= kMaxRequests && width > 0 && page_size > 0 && (long long)width * page_size < (1ll << 31); }
}  // namespace
}  // namespace paged
}  // namespace adsp

extern "C" size_t adsp_paged_fork_workspace_bytes(int B, int width) {
  using namespace adsp::paged;
  if (B <= 0 || width <= 0) return 0;
  return 256 + 6 * align((size_t)B * 4) + align((size_t)B * width * 4);
}
extern "C" int adsp_paged_fork(const void* parents, int parents_bits, void* lengths, int lengths_bits, int32_t* block_tables, int64_t table_stride, int32_t* free_pages,
                               int64_t* free_range, int32_t* shares, void* k_pages, void* v_pages, int B, int width, int page_size, int free_entries, int pages,
                               int heads, int D, const int64_t* strides, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace adsp::paged;
  if (!parents || !lengths || !block_tables || !free_pages || !free_range || !shares || !strides) return ADSP_ERR_NULL;
  if (!requests_fit(B, width, page_size) || free_entries <= 0 || pages <= 0 || table_stride < width) return ADSP_ERR_SHAPE;
  if ((parents_bits != 32 && parents_bits != 64) || (lengths_bits != 32 && lengths_bits != 64)) return ADSP_ERR_UNSUPPORTED;
  const int rc = check_rows(dtype, heads, D, page_size, strides, 6, {k_pages, v_pages});
  if (rc != ADSP_OK) return rc;
  if (!workspace || workspace_bytes < adsp_paged_fork_workspace_bytes(B, width) || ((uintptr_t)workspace & 15) != 0) return ADSP_ERR_WORKSPACE;
  ForkParams p;
  p.parents = parents;
  p.lengths = lengths;
  p.parents_bits = parents_bits;
  p.lengths_bits = lengths_bits;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.free_range = (long long*)free_range;
  p.shares = shares;
  p.rows = page_rows(k_pages, v_pages, k_pages, v_pages, heads, D, strides, strides, dtype);
  p.B = B;
  p.width = width;
  p.page = page_size;
  p.free_entries = free_entries;
  p.pages = pages;
  char* at = (char*)workspace;
  p.range = (long long*)at;
  at += 256;
  for (int** x : {&p.len, &p.children, &p.heir, &p.freed, &p.copies, &p.place}) {
    *x = (int*)at;
    at += align((size_t)B * 4);
  }
  p.old = (int*)at;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)B), block(kThreads);
  // a page's rows in slices of 16 KB of K and of V
  const long long bytes = (long long)heads * page_size * p.rows.pieces * 16, slices = (bytes + 16383) / 16384;
  (void)hipGetLastError();
  if (B <= kSmallRequests && (long long)B * width <= kSmallThreads * kForkEach) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kSmallThreads), 0, s, p);
  } else {
    const int columns = (width + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(fork_holders_kernel, dim3((unsigned)((B + kGroup - 1) / kGroup), (unsigned)(columns < 64 ? columns : 64)), block, 0, s, p);
    hipLaunchKernelGGL(fork_mark_kernel, grid, block, 0, s, p);
    hipLaunchKernelGGL(fork_count_kernel, grid, block, 0, s, p);
    hipLaunchKernelGGL(fork_free_kernel, grid, block, 0, s, p);
  }
  hipLaunchKernelGGL(fork_tables_kernel, dim3((unsigned)B, (unsigned)(slices < 64 ? slices : 64)), block, 0, s, p);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}

extern "C" size_t adsp_paged_compact_workspace_bytes(int B, int pages, int room) {
  using namespace adsp::paged;
  if (B <= 0 || pages <= 0 || room <= 0) return 0;
  return align((size_t)pages * 8) + align((size_t)pages * 4) + align((size_t)room * 4) + align((size_t)B * 4);
}
extern "C" int adsp_paged_compact(const void* lengths, int lengths_bits, const int32_t* block_tables, int64_t table_stride, const void* k_pages, const void* v_pages,
                                  void* k_to, void* v_to, void* lengths_to, int32_t* tables_to, int32_t* shares_to, int32_t* free_to, int64_t* range_to, int B,
                                  int width, int page_size, int pages, int room, int heads, int D, const int64_t* strides, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace adsp::paged;
  if (!lengths || !block_tables || !lengths_to || !tables_to || !shares_to || !free_to || !range_to || !strides) return ADSP_ERR_NULL;
  if (!requests_fit(B, width, page_size) || pages <= 0 || room <= 0 || table_stride < width) return ADSP_ERR_SHAPE;
  if (lengths_bits != 32 && lengths_bits != 64) return ADSP_ERR_UNSUPPORTED;
  const int rc = check_rows(dtype, heads, D, page_size, strides, 12, {k_pages, v_pages, k_to, v_to});
  if (rc != ADSP_OK) return rc;
  if (!workspace || workspace_bytes < adsp_paged_compact_workspace_bytes(B, pages, room) || ((uintptr_t)workspace & 15) != 0) return ADSP_ERR_WORKSPACE;
  CompactParams p;
  p.lengths = lengths;
  p.lengths_to = lengths_to;
  p.bits = lengths_bits;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.tables_to = tables_to;
  p.shares_to = shares_to;
  p.free_to = free_to;
  p.range_to = (long long*)range_to;
  p.rows = page_rows(k_pages, v_pages, k_to, v_to, heads, D, strides, strides + 6, dtype);
  p.B = B;
  p.width = width;
  p.page = page_size;
  p.pages = pages;
  p.room = room;
  char* at = (char*)workspace;
  p.seen = (unsigned long long*)at;
  at += align((size_t)pages * 8);
  p.number = (int*)at;
  at += align((size_t)pages * 4);
  p.of = (int*)at;
  at += align((size_t)room * 4);
  p.count = (int*)at;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)B), block(kThreads);
  const int most = pages > room ? pages : room, clear = (most + 1023) / 1024, copiers = room < 4096 ? room : 4096;
  (void)hipGetLastError();
  if (B <= kSmallRequests && (long long)B * width <= kSmallThreads * kCompactEach && room <= kSmallRoom) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kSmallThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL(compact_clear_kernel, dim3((unsigned)(clear < 1024 ? clear : 1024)), block, 0, s, p);
    hipLaunchKernelGGL(compact_mark_kernel, grid, block, 0, s, p);
    hipLaunchKernelGGL(compact_count_kernel, grid, block, 0, s, p);
    hipLaunchKernelGGL(compact_number_kernel, grid, block, 0, s, p);
  }
  hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)(B + copiers)), block, 0, s, p, copiers);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
