// Queries and keys of two lengths: instances of the attention kernels whose K and V have rows of their own number (kCross).  In the others the
// keys' side is the queries', and the code is what it is without.
#pragma once
#include <type_traits>

#include "attn_bwd_params.h"
#include "attn_params.h"
#include "common.h"

namespace adsp {

// N and varlen of the parameters are the queries'; no causal mask and no tile mask.
struct KeyLengths {
  const void* varlen_k;
  int varlen_k_bits;
  int Nk;
};
struct AttnCrossParams : AttnParams, KeyLengths {};
struct AttnBwdCrossParams : AttnBwdParams, KeyLengths {
  // few blocks of keys: dK and dV in that many sums over parts of the queries (1: none), fp32 rows [part][dK, dV][B * Hkv * Nk][D]
  int q_parts;
  float* q_part_rows;
  __device__ __forceinline__ float* part_of(int part, int which, int D) const { return q_part_rows + ((size_t)(2 * part + which) * B * Hkv * Nk) * D; }
};
template <bool kCross> using FwdParams = std::conditional_t<kCross, AttnCrossParams, AttnParams>;
template <bool kCross> using BwdParams = std::conditional_t<kCross, AttnBwdCrossParams, AttnBwdParams>;

// What the forward on 32 rows a workgroup keeps of its rows' supports for the gradients: a count a row (kNoList: the row block's lists overflowed), z - tau and keys.
constexpr int kKeptMembers = 128;  // what the forward's lists of a row hold
constexpr uint16_t kNoList = 0xffff;
struct KeptLists {
  float* w;        // [rows][kKeptMembers]
  uint16_t* keys;  // likewise
  uint16_t* counts;
};
__host__ __device__ __forceinline__ size_t kept_lists_bytes(size_t rows) { return rows * (kKeptMembers * 6) + rows * 2; }
__device__ __forceinline__ KeptLists kept_lists(const unsigned char* at, size_t rows) {
  float* const w = reinterpret_cast<float*>(const_cast<unsigned char*>(at));
  uint16_t* const keys = reinterpret_cast<uint16_t*>(w + rows * kKeptMembers);
  return {w, keys, keys + rows * kKeptMembers};
}
// Whether all row blocks (of 32 rows) of a K/V head's queries have lists; all threads of a workgroup of 256.
__device__ __forceinline__ bool all_listed(const KeptLists& kept, size_t q_head0, int group, int N, int L, int tid) {
  const int blocks = (L + 31) / 32;
  int any = 0;
  for (int i = tid; i < group * blocks; i += 256) any |= kept.counts[q_head0 + (size_t)(i / blocks) * N + i % blocks * 32] == kNoList ? 1 : 0;
  return !__syncthreads_or(any);
}

__device__ __forceinline__ int valid_length(const void* varlen, int bits, int b, int N) {
  if (!varlen) return N;
  const long long l = bits == 64 ? ((const long long*)varlen)[b] : (long long)((const int*)varlen)[b];
  return (int)(l < 0 ? 0 : (l > N ? N : l));
}
template <bool kCross, typename P> __device__ __forceinline__ int key_rows(const P& p) {  // rows of K and V in memory
  if constexpr (kCross) return p.Nk;
  else return p.N;
}
template <bool kCross, typename P> __device__ __forceinline__ int key_length(const P& p, int b, int NK) {
  if constexpr (kCross) return valid_length(p.varlen_k, p.varlen_k_bits, b, NK);
  else return valid_length(p.varlen, p.varlen_bits, b, NK);
}
template <bool kCross, typename P> __device__ __forceinline__ bool is_padded(const P& p) {
  if constexpr (kCross) return p.varlen != nullptr || p.varlen_k != nullptr;
  else return p.varlen != nullptr;
}
template <bool kCross, typename P> __device__ __forceinline__ bool is_causal(const P& p) {
  if constexpr (kCross) return false;
  else return p.causal != 0;
}
// What dq and dk are multiplied with.  An item of one key has the weight 1 there whatever the scores are: its queries and key have no gradient, where dP - delta would be the difference
// of two roundings of one number.
template <bool kCross, typename P> __device__ __forceinline__ float gradient_scale(const P& p, int LK) { return kCross && LK == 1 ? 0.f : p.sm_scale; }
// The item at a place of the batch, the valid queries and the valid keys of it.  A workgroup's time goes by the length that it walks along: the keys', or in the
// kernel of dK and dV (`by_queries`) the queries'; batch_item orders a batch by it.  Where no key is, no query is either.
struct TwoLengths {
  int b, L, LK;
};
template <bool kCross, typename P>
__device__ __forceinline__ TwoLengths two_lengths(const P& p, bool by_queries, int pos, int blocks, bool longest_first, int per_cu) {
  if constexpr (!kCross) {
    const BatchItem item = batch_item(p.varlen, p.varlen_bits, p.B, p.N, pos, p.Hkv, blocks, longest_first, per_cu);
    return {item.b, item.L, item.L};
  } else if (by_queries) {
    const BatchItem item = batch_item(p.varlen, p.varlen_bits, p.B, p.N, pos, p.Hkv, blocks, longest_first, per_cu);
    return {item.b, item.L, valid_length(p.varlen_k, p.varlen_k_bits, item.b, p.Nk)};
  } else {
    const BatchItem item = batch_item(p.varlen_k, p.varlen_k_bits, p.B, p.Nk, pos, p.Hkv, blocks, longest_first, per_cu);
    return {item.b, item.L > 0 ? valid_length(p.varlen, p.varlen_bits, item.b, p.N) : 0, item.L};
  }
}

}  // namespace adsp
