// The bookkeeping of a paged cache on the GPU, without a trip to the host: which pages and slots the new tokens of a step take
// (build_tables_kernel), and their keys and values on the way there (write_pages_kernel).
//
// For request b with `held` tokens in the cache and `new` more, pages of P slots and a table of W entries:
//   have = ceil(held / P), need = min(ceil((held + new) / P), W) - have, off = sum of need over the requests in front of it,
//   got = min(max(free - off, 0), need); table[b][have + i] = free page number first + off + i; after = min(held + new, (have + got) P).
// The new tokens lie request behind request; position x of b has slot table[b][x / P] P + x % P, and -1 where x >= after.
// kWithin: only the first `tokens` of the new ones are there; those behind them get no page and are not counted.
#include "common.h"
#include "../../include/adasplash_hip.h"

namespace adsp {
namespace paged {
constexpr int kThreads = 256;
constexpr int kMaxRequests = 8192;

struct TableParams {
  const void *lengths, *fresh;
  int lengths_bits, fresh_bits;
  int32_t* tables;
  long long table_stride;
  const int32_t* free_pages;
  const long long* free_range;
  long long* slots;
  long long* positions;  // or null: each token's place in its request
  void* after;  // as wide as `lengths`
  long long* range_after;
  int B, width, page, free_entries;
  long long tokens;
};

__device__ __forceinline__ long long load_length(const void* x, int bits, int i) {
  const long long l = bits == 64 ? ((const long long*)x)[i] : (long long)((const int*)x)[i];
  return l < 0 ? 0 : l;
}

// Every workgroup forms the two running sums over the requests for itself, in LDS (8 bytes a request, one launch and no second
// trip to memory), and takes its share of the tokens and of the new pages, which it finds by bisection in them.  A new token's page
// is looked up where the table's entry comes from, not in the table, which another workgroup may be about to write.
// What bounds it is latency: lengths, sums, then table or free list.
template <bool kWithin> __global__ __launch_bounds__(kThreads) void build_tables_kernel(TableParams p) {
  extern __shared__ int sums[];
  int* const token_end = sums;        // new tokens up to and including a request's
  int* const page_end = sums + p.B;   // pages likewise
  __shared__ long long part[2][kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long limit = (long long)p.width * p.page;
  const long long first = p.free_range[0] > 0 ? p.free_range[0] : 0;
  long long avail = p.free_range[1] - first;
  avail = avail < 0 ? 0 : (avail > p.free_entries ? p.free_entries : avail);
  auto held_of = [&](int b) {
    const long long l = load_length(p.lengths, p.lengths_bits, b);
    return (int)(l < limit ? l : limit);
  };
  auto fresh_of = [&](int b) {
    const long long l = load_length(p.fresh, p.fresh_bits, b);
    return (int)(l < (1 << 30) ? l : (1 << 30));
  };
  auto pages_of = [&](long long tokens) { return (int)((tokens + p.page - 1) / p.page); };
  auto need_of = [&](int held, int fresh) {
    const long long upto = (long long)held + fresh;
    return pages_of(upto < limit ? upto : limit) - pages_of(held);
  };
  // a thread has `per` requests side by side
  const int per = (p.B + kThreads - 1) / kThreads, b0 = tid * per, b1 = b0 + per < p.B ? b0 + per : p.B;
  long long tokens = 0, need = 0;
  for (int b = b0; b < b1; ++b) {
    const int held = held_of(b), fresh = fresh_of(b);
    tokens += fresh;
    token_end[b] = fresh;
    if constexpr (!kWithin) {
      need += need_of(held, fresh);
      page_end[b] = need_of(held, fresh);
    }
  }
  // (sums beyond 32 bits are cut off: no more tokens than slots and no more pages than the list has are looked for)
  constexpr long long kMost = 0x7fffffff;
  const long long most_tokens = kWithin ? p.tokens : kMost;
  auto scan = [&](long long mine, int which) {
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    if (lane == 63) part[which][wave] = upto;
    return upto - mine;
  };
  long long t0 = scan(tokens, 0), n0 = kWithin ? 0 : scan(need, 1);
  __syncthreads();
  for (int w = 0; w < wave; ++w) t0 += part[0][w];
  auto end_of = [&](int b) {  // of request b's new tokens, t0 before and behind it
    t0 += token_end[b];
    token_end[b] = (int)(t0 < most_tokens ? t0 : most_tokens);
  };
  if constexpr (kWithin) {
    int start = (int)(t0 < most_tokens ? t0 : most_tokens);
    for (int b = b0; b < b1; ++b) {
      end_of(b);
      page_end[b] = need_of(held_of(b), token_end[b] - start);
      need += page_end[b];
      start = token_end[b];
    }
    n0 = scan(need, 1);
    __syncthreads();
  }
  for (int w = 0; w < wave; ++w) n0 += part[1][w];
  long long all_tokens = 0, all_need = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    all_tokens += part[0][w];
    all_need += part[1][w];
  }
  for (int b = b0; b < b1; ++b) {
    if constexpr (!kWithin) end_of(b);
    n0 += page_end[b];
    page_end[b] = (int)(n0 < kMost ? n0 : kMost);
  }
  __syncthreads();
  auto request_of = [&](const int* ends, int x) {  // the first request whose end lies behind x
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (ends[mid] > x) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  auto start_of = [&](const int* ends, int b) { return b > 0 ? ends[b - 1] : 0; };
  auto free_page = [&](long long i) { return p.free_pages[(first + i) % p.free_entries]; };
  const long long step = (long long)gridDim.x * kThreads, at = (long long)blockIdx.x * kThreads + tid;
  // slots
  for (long long i = at; i < p.tokens; i += step) {
    long long slot = -1, place = 0;
    if (i < all_tokens) {
      const int b = request_of(token_end, (int)i), held = held_of(b), have = pages_of(held), off = start_of(page_end, b);
      const long long x = (long long)held + (i - start_of(token_end, b));
      place = x;
      if (x < limit) {
        const int pg = (int)x / p.page;
        int id = -1;
        if (pg < have) id = p.tables[(long long)b * p.table_stride + pg];
        else if (off + (pg - have) < avail) id = free_page(off + (pg - have));
        if (id >= 0) slot = (long long)id * p.page + (int)x % p.page;
      }
    }
    p.slots[i] = slot;
    if (p.positions) p.positions[i] = place;
  }
  // new pages
  const long long pages = all_need < avail ? all_need : avail;
  for (long long i = at; i < pages; i += step) {
    const int b = request_of(page_end, (int)i), col = pages_of(held_of(b)) + (int)(i - start_of(page_end, b));
    p.tables[(long long)b * p.table_stride + col] = free_page(i);
  }
  // lengths behind the step
  for (long long i = at; i < p.B; i += step) {
    const int b = (int)i, held = held_of(b), fresh = kWithin ? token_end[b] - start_of(token_end, b) : fresh_of(b);
    const int off = start_of(page_end, b), need_b = page_end[b] - off;
    long long got = avail - off;
    got = got < 0 ? 0 : (got < need_b ? got : need_b);
    const long long room = (pages_of(held) + got) * p.page, upto = (long long)held + fresh;
    const long long after = upto < room ? upto : room;
    if (p.lengths_bits == 64) ((long long*)p.after)[b] = after;
    else ((int*)p.after)[b] = (int)after;
  }
  if (at == 0) {
    p.range_after[0] = first + pages;
    p.range_after[1] = p.free_range[1];
  }
}

struct WriteParams {
  const char *k, *v;
  char *k_pages, *v_pages;
  const long long* slots;
  long long k_st, k_sh, v_st, v_sh;                   // bytes: token, head
  long long k_sp, k_sph, k_sps, v_sp, v_sph, v_sps;  // bytes: page, head, slot
  long long tokens, n_slots;
  int heads, pieces, page;  // pieces of 16 bytes in a row
};
// A piece of 16 bytes of K and of V to a thread: rows of a token side by side.  Bound by HBM: it reads and writes each byte once.
__global__ __launch_bounds__(256) void write_pages_kernel(WriteParams p) {
  const long long per_token = (long long)p.heads * p.pieces, all = p.tokens * per_token;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    const long long t = i / per_token;
    const int rest = (int)(i - t * per_token), h = rest / p.pieces, c = rest % p.pieces;
    const long long slot = p.slots[t];
    if (slot < 0 || slot >= p.n_slots) continue;
    const long long pg = slot / p.page, in = slot % p.page;
    const u32x4 a = *reinterpret_cast<const u32x4*>(p.k + t * p.k_st + h * p.k_sh + c * 16);
    const u32x4 b = *reinterpret_cast<const u32x4*>(p.v + t * p.v_st + h * p.v_sh + c * 16);
    *reinterpret_cast<u32x4*>(p.k_pages + pg * p.k_sp + h * p.k_sph + in * p.k_sps + c * 16) = a;
    *reinterpret_cast<u32x4*>(p.v_pages + pg * p.v_sp + h * p.v_sph + in * p.v_sps + c * 16) = b;
  }
}
}  // namespace paged
}  // namespace adsp

static int build_tables(bool within, const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                        int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots, void* lengths_after,
                        int64_t* range_after, int B, int width, int page_size, int free_entries, int64_t tokens, int64_t* positions, void* stream) {
  using namespace adsp::paged;
  if (!lengths || !new_tokens || !block_tables || !free_pages || !free_range || !lengths_after || !range_after || (tokens > 0 && !slots))
    return ADSP_ERR_NULL;
  if (B <= 0 || B > kMaxRequests || width <= 0 || page_size <= 0 || free_entries <= 0 || tokens < 0 || tokens >= (1ll << 31) || table_stride < width)
    return ADSP_ERR_SHAPE;
  if ((long long)width * page_size >= (1ll << 31)) return ADSP_ERR_SHAPE;
  if ((lengths_bits != 32 && lengths_bits != 64) || (new_tokens_bits != 32 && new_tokens_bits != 64)) return ADSP_ERR_UNSUPPORTED;
  TableParams p;
  p.lengths = lengths;
  p.fresh = new_tokens;
  p.lengths_bits = lengths_bits;
  p.fresh_bits = new_tokens_bits;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.free_range = (const long long*)free_range;
  p.slots = (long long*)slots;
  p.positions = (long long*)positions;
  p.after = lengths_after;
  p.range_after = (long long*)range_after;
  p.B = B;
  p.width = width;
  p.page = page_size;
  p.free_entries = free_entries;
  p.tokens = tokens;
  const long long most = tokens > B ? tokens : B, groups = (most + 1023) / 1024;  // four items a thread
  (void)hipGetLastError();
  const dim3 grid((unsigned)(groups < 256 ? groups : 256));
  if (within) hipLaunchKernelGGL(build_tables_kernel<true>, grid, dim3(kThreads), (size_t)B * 8, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(build_tables_kernel<false>, grid, dim3(kThreads), (size_t)B * 8, (hipStream_t)stream, p);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
extern "C" int adsp_paged_build_tables(const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                                       int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots,
                                       void* lengths_after, int64_t* range_after, int B, int width, int page_size, int free_entries,
                                       int64_t tokens, void* stream) {
  return build_tables(false, lengths, lengths_bits, new_tokens, new_tokens_bits, block_tables, table_stride, free_pages, free_range, slots, lengths_after,
                      range_after, B, width, page_size, free_entries, tokens, nullptr, stream);
}
extern "C" int adsp_paged_append_tables(const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                                        int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots,
                                        void* lengths_after, int64_t* range_after, int B, int width, int page_size, int free_entries,
                                        int64_t tokens, void* stream) {
  return build_tables(true, lengths, lengths_bits, new_tokens, new_tokens_bits, block_tables, table_stride, free_pages, free_range, slots, lengths_after,
                      range_after, B, width, page_size, free_entries, tokens, nullptr, stream);
}
extern "C" int adsp_paged_append_positions(const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                                           int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots,
                                           void* lengths_after, int64_t* range_after, int B, int width, int page_size, int free_entries,
                                           int64_t tokens, int64_t* positions, void* stream) {
  if (tokens > 0 && !positions) return ADSP_ERR_NULL;
  return build_tables(true, lengths, lengths_bits, new_tokens, new_tokens_bits, block_tables, table_stride, free_pages, free_range, slots, lengths_after,
                      range_after, B, width, page_size, free_entries, tokens, positions, stream);
}

extern "C" int adsp_paged_write(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots, int64_t tokens, int heads, int D,
                                int64_t pages, int page_size, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                int64_t kp_stride_page, int64_t kp_stride_h, int64_t kp_stride_n, int64_t vp_stride_page, int64_t vp_stride_h,
                                int64_t vp_stride_n, int dtype, void* stream) {
  using namespace adsp::paged;
  if (!k || !v || !k_pages || !v_pages || !slots) return ADSP_ERR_NULL;
  if (dtype != ADSP_F32 && dtype != ADSP_BF16 && dtype != ADSP_F16) return ADSP_ERR_DTYPE;
  if (tokens <= 0 || heads <= 0 || D <= 0 || pages <= 0 || page_size <= 0) return ADSP_ERR_SHAPE;
  const int es = dtype == ADSP_F32 ? 4 : 2;
  if (D * es % 16 != 0) return ADSP_ERR_SHAPE;
  if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) != 0) return ADSP_ERR_ALIGN;
  if (((k_stride_t | k_stride_h | v_stride_t | v_stride_h | kp_stride_page | kp_stride_h | kp_stride_n | vp_stride_page | vp_stride_h | vp_stride_n) * es & 15) != 0)
    return ADSP_ERR_ALIGN;
  WriteParams p;
  p.k = (const char*)k;
  p.v = (const char*)v;
  p.k_pages = (char*)k_pages;
  p.v_pages = (char*)v_pages;
  p.slots = (const long long*)slots;
  p.k_st = k_stride_t * es;
  p.k_sh = k_stride_h * es;
  p.v_st = v_stride_t * es;
  p.v_sh = v_stride_h * es;
  p.k_sp = kp_stride_page * es;
  p.k_sph = kp_stride_h * es;
  p.k_sps = kp_stride_n * es;
  p.v_sp = vp_stride_page * es;
  p.v_sph = vp_stride_h * es;
  p.v_sps = vp_stride_n * es;
  p.tokens = tokens;
  p.n_slots = (long long)pages * page_size;
  p.heads = heads;
  p.pieces = D * es / 16;
  p.page = page_size;
  const long long groups = (tokens * heads * p.pieces + 255) / 256;
  (void)hipGetLastError();
  hipLaunchKernelGGL(write_pages_kernel, dim3((unsigned)(groups < (1ll << 22) ? groups : (1ll << 22))), dim3(256), 0, (hipStream_t)stream, p);
  return hipGetLastError() == hipSuccess ? ADSP_OK : ADSP_ERR_LAUNCH;
}
