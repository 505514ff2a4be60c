/*
 * adasplash_hip.h -- C ABI of the MI355X (gfx950) sparse entmax attention library.
 *
 * Every entry point takes raw device pointers, sizes and scalars, enqueues its kernels on the
 * HIP stream it is given (a hipStream_t passed as void*; NULL = the default stream), never
 * synchronises and never allocates.  The caller owns every buffer, including the workspace; what a call
 * computes depends on its arguments alone.  The return value is an adsp_status; nothing is thrown across
 * the ABI.
 *
 * State the library does hold, none of which carries results from one call to the next:
 *   - per process, the number of workgroups of the persistent kernels that fit the device, looked up on
 *     the first launch of each kernel (one device family per process is assumed: gfx950);
 *   - per device, the address of the 64 MiB scratch array behind adsp_attn_v2_fwd_noalloc, looked up on
 *     that entry point's first call on the device (calls through it share the array: see there);
 *   - the environment, read on every call (comparisons, tests and profiling; unset in normal use):
 *       ADSP_SPARSE=0               every row block of a 16-bit call on the dense kernels (no sparse-support kernels,
 *                                   none of those for short calls); fp32 calls do not look at it
 *       ADSP_BWD_STREAMS=0          the sparse-support dK/dV kernel walks the scores itself instead of taking
 *                                   the dQ kernel's candidate streams
 *       ADSP_PROBE_MAX_SUPPORT=n    the support the probe lets a K/V head's longest rows have before it
 *                                   leaves the head to the dense kernels (default 28; 0: every head)
 *       ADSP_DKDV_MERGE256=n        the share of a causal sequence, in 256ths, from which on the dK/dV kernel serves
 *                                   a key block for all query heads of a K/V head at once (default 80; 0: never).
 *                                   Sizes the backward workspace too: the same value for the size query and the call.
 *
 * The entry points replace the Triton launches inside the reference's autograd wrappers (the
 * reference has no FFI of its own; these are the calls a binding would make in their place):
 *
 *   adsp_entmax_rows_fwd  <- _entmax_triton.forward -> _fwd_entmax
 *                            (adasplash/triton_entmax_v2.py:624-664, kernel :363-536)
 *   adsp_entmax_rows_bwd  <- _entmax_triton.backward -> _bwd_entmax
 *                            (adasplash/triton_entmax_v2.py:667-687, kernel :541-617)
 *   adsp_attn_v2_fwd      <- _sparse_attention.forward -> _get_tau, _get_tau_v2, _get_tau_v3,
 *                            _get_output (adasplash/adasplash_v2.py:1243-1438)
 *   adsp_attn_bwd         <- _sparse_attention.backward -> _bwd_preprocess, _bwd_q_kernel,
 *                            transpose_bmask, _bwd_kv_kernel (adasplash/adasplash_v2.py:1441-1564) and its
 *                            generic-alpha twin (adasplash/adasplash_block_mask.py:1079-1210)
 *   adsp_attn_v1_fwd      <- _sparse_attention.forward -> _get_tau,
 *                            compute_bidxs_and_cubcounts, _get_output
 *                            (adasplash/adasplash_block_mask.py:941-1076)
 */
#ifndef ADASPLASH_HIP_H
#define ADASPLASH_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  ADSP_OK = 0,
  ADSP_ERR_NULL = 1,        /* a required pointer is NULL */
  ADSP_ERR_SHAPE = 2,       /* a dimension is out of the supported range */
  ADSP_ERR_DTYPE = 3,       /* unknown element type */
  ADSP_ERR_ALIGN = 4,       /* a tensor base pointer is not 16-byte aligned */
  ADSP_ERR_UNSUPPORTED = 5, /* parameter combination the kernels do not implement */
  ADSP_ERR_WORKSPACE = 6,   /* workspace missing or smaller than adsp_attn_workspace_bytes() */
  ADSP_ERR_LAUNCH = 7,      /* the HIP runtime refused a launch (hipGetLastError() != success) */
  ADSP_ERR_TOO_LARGE = 8    /* adsp_attn_v2_fwd_noalloc: the problem needs more scratch than the library holds */
} adsp_status;

/* Element types of q/k/v/out and x/y. */
typedef enum { ADSP_F32 = 0, ADSP_BF16 = 1, ADSP_F16 = 2 } adsp_dtype;

/* Library ABI version (bumped when a signature changes). */
int adsp_version(void);

/*
 * Identity of the sources this library was built from: the first 16 hex digits of a SHA-256 over the
 * kernel sources, headers and compiler flags, baked in at build time ("unknown" for a build that did not
 * pass it).  No counterpart in the reference (pure Python, nothing to go stale); the Python loader compares
 * it with the tree it sits in so that a library older than its sources cannot be tested or benchmarked.
 */
const char* adsp_build_id(void);
/* The extra compiler flags of a profiling build (empty for a regular one); they enter adsp_build_id(). */
const char* adsp_build_flags(void);

/* Static, NUL-terminated description of a status code. */
const char* adsp_status_string(int status);

/*
 * Row-wise alpha-entmax over the last dimension: y[r, :] = [(alpha-1) x[r, :] - tau_r]_+^(1/(alpha-1)).
 *   x, y      : contiguous [rows, cols] arrays of `dtype`; y is fully overwritten (zeros included).
 *   alpha     : > 1.  n_iter (>= 0), use_histogram, fast_math: accepted; the solver runs to convergence whatever they say.
 * Replaces the launch at adasplash/triton_entmax_v2.py:650-658.
 */
int adsp_entmax_rows_fwd(const void* x, void* y, int64_t rows, int64_t cols, int dtype, double alpha,
                         int n_iter, int use_histogram, int fast_math, void* stream);

/*
 * Backward of the above: dx = u*dy - (sum(u*dy)/sum(u)) * u with u = y^(2-alpha) on the support.
 * Replaces the launch at adasplash/triton_entmax_v2.py:678-685.
 */
int adsp_entmax_rows_bwd(const void* y, const void* dy, void* dx, int64_t rows, int64_t cols, int dtype,
                         double alpha, void* stream);

/*
 * Bytes of scratch the forward entry points need for these dimensions; 0 for fp32 and for the head dims the
 * sparse-support kernel does not serve (then `workspace` may be NULL).  For the 16-bit types at head dims 64 and 128:
 * the work counters, row-block flags and candidate streams of the sparse-support kernel (up to 1024 slots of 51 KiB;
 * sequences of up to 65536 keys) and a one-byte (fp8 e4m3) copy of K.  The buffer must be 16-byte aligned device
 * memory; its contents need not survive between calls, and two calls that run at the same time need a buffer each.
 * For the block-mask variant pass Hq = Hkv = H.  The size serves any call with these dimensions and is asked for in every
 * one: a short 16-bit call without bmask and supports, whose kernel does not touch the buffer, is refused without it too.
 */
size_t adsp_attn_workspace_bytes(int B, int Hq, int Hkv, int N, int D, int dtype);

/* Number of int32 words per (batch, head) the block mask needs: n_row_blocks * words_per_row. */
size_t adsp_attn_bmask_words(int N);

/* 0 when the backward of such a call needs neither the forward's tile mask nor its supports, so that a caller with no other use
 * for them passes NULL to both (single precision at head dims 64 and 128, and short 16-bit problems there: the call then
 * takes the kernels made for them), else 1. */
int adsp_attn_bwd_reads_bmask(int B, int Hq, int Hkv, int N, int D, int dtype, double alpha, int is_causal);

/*
 * AdaSplash-2 forward: causal entmax-1.5 attention with GQA and right-padded variable lengths.
 *   q, out : [B, Hq, N, D]; k, v : [B, Hkv, N, D], contiguous, Hq % Hkv == 0, D in {16,32,64,128,256}.
 *   taus   : [B, Hq, N] fp32, receives the per-row threshold (rows past the valid length untouched).
 *   bmask  : NULL, or [B, Hq, adsp_attn_bmask_words(N)] int32, receives the per-(128-row, 64-key) tile mask,
 *            bit (c % 32) of word c / 32 of a row block = key tile c holds a non-zero probability.
 *   varlen : NULL, or [B] valid lengths as int32 (varlen_bits = 32) or int64 (varlen_bits = 64);
 *            keys >= length are masked, output rows >= length are written as zeros.
 *   niter  : Halley/bisection refinement passes after the histogram bracket (>= 0).  where the dense kernel serves
 *            a call alone it takes niter + 1 of them, as the reference does (adasplash/adasplash_v2.py:567-611 and
 *            :617-681); behind the sparse-support kernel it takes niter.  That kernel, and those that serve fp32 at head
 *            dims 64 / 128 and short 16-bit calls without bmask, iterate to convergence.
 * Replaces the four launches at adasplash/adasplash_v2.py:1288-1419.
 */
int adsp_attn_v2_fwd(const void* q, const void* k, const void* v, void* out, float* taus, int32_t* bmask,
                     const void* varlen, int varlen_bits, int B, int Hq, int Hkv, int N, int D, int dtype,
                     int niter, void* workspace, size_t workspace_bytes, void* stream);

/*
 * adsp_attn_v2_fwd without a workspace argument, for callers that cannot allocate device memory (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  The
 * scratch memory (control words, flags, candidate streams and fp8 copy of K of the sparse-support kernel)
 * lives in a device array inside the library, 64 MiB on every GPU the library runs on, held until the process ends;
 * problems whose adsp_attn_workspace_bytes() exceeds adsp_attn_v2_fwd_noalloc_max_bytes() are rejected with
 * ADSP_ERR_TOO_LARGE.  The call allocates and frees nothing and records no memset (the kernels clear what must start
 * at zero).  All calls on one GPU share that array: calls that overlap on one GPU (two streams, two threads) race
 * and must be serialised by the caller.  Other arguments, results and status codes as adsp_attn_v2_fwd.
 */
size_t adsp_attn_v2_fwd_noalloc_max_bytes(void);
int adsp_attn_v2_fwd_noalloc(const void* q, const void* k, const void* v, void* out, float* taus, int32_t* bmask,
                             const void* varlen, int varlen_bits, int B, int Hq, int Hkv, int N, int D, int dtype,
                             int niter, void* stream);

/*
 * AdaSplash-1 (block-mask) forward: alpha-entmax attention for any alpha in (1, 2], causal or not,
 * right-padded variable lengths, no GQA (q, k, v share [B, H, N, D]).
 *   tile_counts : NULL, or 2 device uint64 that are incremented by {16x16 score tiles inside the
 *                 causal/valid domain, those that hold a non-zero probability} (for sparsity reports).
 * Other arguments as in adsp_attn_v2_fwd.  Replaces the launches at
 * adasplash/adasplash_block_mask.py:978-1003 and :1024-1054 plus the torch-side list building
 * (:298-320).
 */
int adsp_attn_v1_fwd(const void* q, const void* k, const void* v, void* out, float* taus, int32_t* bmask,
                     const void* varlen, int varlen_bits, int B, int H, int N, int D, int dtype, double alpha,
                     int is_causal, int niter, void* workspace, size_t workspace_bytes,
                     unsigned long long* tile_counts, void* stream);

/*
 * Supports kept for the backward.  No counterpart in the reference (its backward recomputes the scores of every tile of
 * the mask).  The sparse-support forward kernel finds, for every row, the few keys with a non-zero probability; the
 * _keep variants of the two forward entry points leave what they found in `supports` -- per 128-row block of a query
 * head its streams of (score, key) pairs, their lengths, every row's threshold relative to the streams' scores and a
 * flag -- and adsp_attn_bwd_kept, given the same buffer untouched, takes the supports from there instead of walking
 * the scores again.  adsp_attn_supports_bytes() is the size of that buffer (51 KiB per 128 query rows and head plus
 * 4 bytes per row; 0 where nothing is kept: fp32, head dims other than 64 and 128, N > 65536; `supports` may then be
 * NULL).  16-byte aligned device memory owned by the caller; it must hold what the forward wrote for the same
 * q, k, v, varlen until the backward has run.  Row blocks the forward served with its dense kernel keep no supports
 * and the backward walks them as adsp_attn_bwd does; with supports == NULL the three calls are adsp_attn_v2_fwd,
 * adsp_attn_v1_fwd (without tile statistics) and adsp_attn_bwd.
 */
size_t adsp_attn_supports_bytes(int B, int Hq, int Hkv, int N, int D, int dtype);
int adsp_attn_v2_fwd_keep(const void* q, const void* k, const void* v, void* out, float* taus, int32_t* bmask,
                          const void* varlen, int varlen_bits, int B, int Hq, int Hkv, int N, int D, int dtype,
                          int niter, void* workspace, size_t workspace_bytes, void* supports, size_t supports_bytes,
                          void* stream);
int adsp_attn_v1_fwd_keep(const void* q, const void* k, const void* v, void* out, float* taus, int32_t* bmask,
                          const void* varlen, int varlen_bits, int B, int H, int N, int D, int dtype, double alpha,
                          int is_causal, int niter, void* workspace, size_t workspace_bytes, void* supports,
                          size_t supports_bytes, void* stream);
int adsp_attn_bwd_kept(const void* q, const void* k, const void* v, const void* dout, const float* taus,
                       const int32_t* bmask, const void* varlen, int varlen_bits, void* dq, void* dk, void* dv,
                       float* delta, float* zinv, int B, int Hq, int Hkv, int N, int D, int dtype, double alpha,
                       int is_causal, void* workspace, size_t workspace_bytes, const void* supports,
                       size_t supports_bytes, void* stream);

/*
 * Workspace of adsp_attn_bwd in bytes; 0 for fp32 and for the head dims the sparse-support kernels do not serve (then
 * `workspace` may be NULL).  For the 16-bit element types at head dims 64 and 128 (sequences of up to 65536 keys): the
 * counters, flags and candidate streams of the sparse-support backward kernels, 1024 * D bytes of fp32 sums per
 * workgroup (items that are worked off in parts), fp32 partial rows of dk and dv per query head (2 * B * Hq * N * D * 4 bytes;
 * none where Hq == Hkv), and the supports the dq kernel hands to the dk/dv kernel: per query row block of 128 rows
 * 51 KiB of (weights, key) pairs and a table of 4 * ceil(N / 128) + 2 16-bit offsets per wave.
 * 16-byte aligned device memory; contents need not survive between calls; concurrent calls need a buffer each.
 * This is the size that serves any call with these dimensions.
 */
size_t adsp_attn_bwd_workspace_bytes(int B, int Hq, int Hkv, int N, int D, int dtype);

/*
 * The same for a call whose is_causal is known: with a causal mask the dk/dv kernel serves the later key blocks of a
 * sequence (from 5/16 of its length on) for all query heads of a K/V head at once and needs partial rows for the first
 * ones only (about 5/16 of the bytes above), so the workspace is smaller.  adsp_attn_bwd and adsp_attn_bwd_kept accept a
 * workspace of either size.  (No counterpart in the reference, which allocates inside its backward.)
 */
size_t adsp_attn_bwd_workspace_bytes_causal(int B, int Hq, int Hkv, int N, int D, int dtype, int is_causal);

/*
 * Backward of both attention variants: dq, dk, dv for the upstream gradient dout.
 *   q, dout, dq : [B, Hq, N, D]; k, v, dk, dv : [B, Hkv, N, D] (Hq == Hkv for the block-mask variant).
 *   taus, bmask : what the forward wrote for the same inputs (bmask may be NULL: every tile is visited).
 *   delta, zinv : [B, Hq, N] fp32 scratch owned by the caller; receive sum_j u_ij dP_ij / sum_j u_ij and
 *                 1 / sum_j p_ij per query row.
 *   alpha, is_causal : 1.5 / 1 for the AdaSplash-2 path, any alpha in (1, 2] for the block-mask path.
 * Rows of q, k, v and dout past a sequence's valid length are never used, whatever they hold; gradient rows
 * past the valid length are written as zeros.  Replaces the four launches at
 * adasplash/adasplash_v2.py:1456-1562 (delta from out2, dq, mask transpose, dk/dv with the GQA group loop)
 * and adasplash/adasplash_block_mask.py:1079-1210.
 */
int adsp_attn_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus,
                  const int32_t* bmask, const void* varlen, int varlen_bits, void* dq, void* dk, void* dv,
                  float* delta, float* zinv, int B, int Hq, int Hkv, int N, int D, int dtype, double alpha,
                  int is_causal, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Entmax attention of a few queries against a cache of keys (a decoding step): entmax_alpha(q k^T / sqrt(D) + bias) v.
 *   q, out    : contiguous [B, H, q_len, D], q_len <= 16; k, v: [B, H, k_len, D] with unit stride along D and the strides given
 *               (in elements; multiples of 16 bytes), D in {32, 64, 128, 256}; base pointers 16-byte aligned.
 *   varlen    : NULL, or [B] valid key counts (varlen_bits 32 or 64): the first ones of a sequence, or with left_padding the last.
 *   alibi_slopes : NULL, or [H] fp32: adds slope * (key position - query position) to the scores.
 *   is_causal : the queries are the last q_len positions of k_len.
 *   workspace : adsp_attn_decode_workspace_bytes() bytes (the scores in fp32).
 * A query that sees no key gets a row of zeros.  Replaces the dense path of examples/attention.py:34-91 for such calls.
 */
size_t adsp_attn_decode_workspace_bytes(int B, int H, int q_len, int k_len);
int adsp_attn_decode_fwd(const void* q, const void* k, const void* v, void* out, const void* varlen, int varlen_bits,
                         int left_padding, const float* alibi_slopes, int B, int H, int q_len, int k_len, int D,
                         int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_n, int64_t v_stride_b, int64_t v_stride_h,
                         int64_t v_stride_n, int dtype, double alpha, int is_causal, void* workspace, size_t workspace_bytes,
                         void* stream);

/*
 * One new token of every request against its keys in a paged cache: entmax_alpha(q k^T / sqrt(D)) v, split over the keys and joined.
 *   q, out       : contiguous [B, Hq, D], Hq a multiple of Hkv (at most 64 query heads to a K/V head), D in {32, 64, 128, 256}.
 *   k_pages, v_pages : `pages` pages of page_size slots of Hkv heads, unit stride along D, the strides given (in elements;
 *                  multiples of 16 bytes); base pointers 16-byte aligned.  Offsets are formed in 64 bits.
 *   block_tables : [B, table_stride] int32, the pages of a request in the order of its tokens.  An entry outside [0, pages) is a page
 *                  without keys and is never followed.
 *   lengths      : [B] tokens of a request (lengths_bits 32 or 64), the new one among them; cut off at max_length, which the first
 *                  ceil(max_length / page_size) entries of a table have to cover.  A request without keys gets rows of zeros.
 *   alpha in (1, 2].  workspace: adsp_attn_split_workspace_bytes(B, Hq, Hkv, 1, max_length) bytes, 16-byte aligned (8 bytes for each
 *   head and key, of which a few per cent are touched); calls that run at the same time need one each.
 * No counterpart in the reference.
 */
size_t adsp_attn_split_workspace_bytes(int B, int Hq, int Hkv, int q_len, int k_len);
int adsp_attn_paged_fwd(const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* block_tables,
                        int64_t table_stride, const void* lengths, int lengths_bits, int B, int Hq, int Hkv, int D, int pages,
                        int page_size, int max_length, int64_t k_stride_page, int64_t k_stride_h, int64_t k_stride_n,
                        int64_t v_stride_page, int64_t v_stride_h, int64_t v_stride_n, int dtype, double alpha, void* workspace,
                        size_t workspace_bytes, void* stream);

/*
 * The pages and slots that the new tokens of a step take, for B <= 8192 requests with `lengths` tokens in the cache and
 * `new_tokens` more (int32 or int64 each).
 *   block_tables : [B, table_stride] int32, `width` entries in use; the entries of new pages are written, no others.
 *   free_pages   : a ring of free_entries page numbers; entries free_range[0] .. free_range[1] - 1 (modulo free_entries) are free.
 *                  They are handed out in the order of the requests.
 *   slots        : [tokens] int64, the new tokens request behind request: page * page_size + place in it, or -1 for a token that
 *                  got no page (no free one, or none in its table) and for places behind the last token.
 *   tokens       : entries of slots.  Where new_tokens sum to more, those behind them have pages and count like the others, but their slots are not told.
 *   lengths_after: [B], as wide as lengths: the tokens of a request that its pages hold.  range_after: [2] int64, what is free then.
 *                  (Both are buffers of their own: `lengths` and `free_range` stay as they are.)
 * adsp_paged_append_tables: only the first `tokens` of the new tokens are there.  Those behind them get no page, and lengths_after does not count them.
 * No counterpart in the reference.
 */
int adsp_paged_build_tables(const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                            int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots,
                            void* lengths_after, int64_t* range_after, int B, int width, int page_size, int free_entries,
                            int64_t tokens, void* stream);
int adsp_paged_append_tables(const void* lengths, int lengths_bits, const void* new_tokens, int new_tokens_bits, int32_t* block_tables,
                             int64_t table_stride, const int32_t* free_pages, const int64_t* free_range, int64_t* slots,
                             void* lengths_after, int64_t* range_after, int B, int width, int page_size, int free_entries,
                             int64_t tokens, void* stream);

/*
 * Keys and values of new tokens, [tokens, heads, D] with the strides given, to their slots of a paged cache (layout as above).  A slot
 * outside the cache is skipped; no slot may stand twice.  D times the element size has to be a multiple of 16 bytes.
 */
int adsp_paged_write(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots, int64_t tokens, int heads, int D,
                     int64_t pages, int page_size, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                     int64_t kp_stride_page, int64_t kp_stride_h, int64_t kp_stride_n, int64_t vp_stride_page, int64_t vp_stride_h,
                     int64_t vp_stride_n, int dtype, void* stream);

/*
 * Attention of queries to keys of another length (an encoder's states), any alpha in (1, 2], not causal, and its backward.
 *   q, out, dout, dq : contiguous [B, Hq, Nq, D]; k, v, dk, dv : contiguous [B, Hkv, Nk, D]; Hq % Hkv == 0, D in {16, 32, 64, 128, 256},
 *                   lengths from 1 to 1,048,576; base pointers 16-byte aligned.
 *   taus          : [B, Hq, Nq] fp32, the rows' thresholds (NULL where no backward follows); rows past a length untouched.
 *   varlen_q, varlen_k : NULL, or [B] valid lengths (their bits 32 or 64).  Rows of q, k, v and dout past a length may hold anything; output and gradient
 *                   rows past it are written as zeros, and so are the rows of an item without keys.
 *   delta, zinv   : [B, Hq, Nq] fp32 scratch, as in adsp_attn_bwd.
 *   workspace     : adsp_attn_cross_workspace_bytes(..., train = taus != NULL) and adsp_attn_cross_bwd_workspace_bytes(..., kept = supports != NULL) bytes,
 *                   16-byte aligned, 0 for calls that need none (then it may be NULL); contents mean nothing between calls, and calls that run at the
 *                   same time need one each.
 *   supports      : NULL, or adsp_attn_cross_supports_bytes() bytes in which a forward with taus keeps the supports that it found for the backward of the same
 *                   inputs, as adsp_attn_v2_fwd_keep does; without them the backward walks the scores.  A backward takes exactly the bytes that
 *                   adsp_attn_cross_supports_bytes() gives at its time (ADSP_SPARSE changes their layout) and refuses others with ADSP_ERR_WORKSPACE.
 * Replaces the dense path of examples/attention.py:34-91 for q_len != k_len without a causal mask.
 */
size_t adsp_attn_cross_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, int train);
size_t adsp_attn_cross_supports_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha);
size_t adsp_attn_cross_bwd_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, int kept);
int adsp_attn_cross_fwd(const void* q, const void* k, const void* v, void* out, float* taus, const void* varlen_q, int varlen_q_bits,
                        const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha,
                        void* workspace, size_t workspace_bytes, void* supports, size_t supports_bytes, void* stream);
int adsp_attn_cross_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus, const void* varlen_q,
                        int varlen_q_bits, const void* varlen_k, int varlen_k_bits, void* dq, void* dk, void* dv, float* delta, float* zinv,
                        int B, int Hq, int Hkv, int Nq, int Nk, int D, int dtype, double alpha, void* workspace, size_t workspace_bytes,
                        const void* supports, size_t supports_bytes, void* stream);

/*
 * A few queries of each sequence against keys of another length, on the kernels of adsp_attn_paged_fwd: q, out, dout, dq contiguous [B, Hq, q_len, D],
 * k, v, dk, dv contiguous [B, Hkv, k_len, D], (Hq / Hkv) * q_len <= 64, D in {32, 64, 128, 256}, alpha in (1, 2].
 *   varlen_q, varlen_k : NULL, or [B] valid lengths as in adsp_attn_cross_fwd.
 *   workspace : adsp_attn_split_workspace_bytes(B, Hq, Hkv, q_len, k_len) bytes.
 *   taus      : NULL, or [B, Hq, q_len] fp32: the call then leaves in them and in the workspace what adsp_attn_cross_step_bwd takes, which leaves both as they are.
 *   scratch   : adsp_attn_cross_step_bwd_scratch_bytes() bytes, 16-byte aligned.
 */
/* Whether such a call, with its backward where `train` is set, is expected to take less time there than in adsp_attn_cross_fwd and adsp_attn_cross_bwd: 1 or 0. */
int adsp_attn_cross_few_rows(int B, int Hq, int Hkv, int q_len, int k_len, int D, int dtype, int train);
int adsp_attn_cross_step_fwd(const void* q, const void* k, const void* v, void* out, float* taus, const void* varlen_q, int varlen_q_bits,
                             const void* varlen_k, int varlen_k_bits, int B, int Hq, int Hkv, int q_len, int k_len, int D, int dtype,
                             double alpha, void* workspace, size_t workspace_bytes, void* stream);
size_t adsp_attn_cross_step_bwd_scratch_bytes(int B, int Hq, int Hkv, int q_len, int k_len);
int adsp_attn_cross_step_bwd(const void* q, const void* k, const void* v, const void* dout, const float* taus, const void* varlen_q,
                             int varlen_q_bits, const void* varlen_k, int varlen_k_bits, void* dq, void* dk, void* dv, int B, int Hq, int Hkv,
                             int q_len, int k_len, int D, int dtype, double alpha, const void* workspace, size_t workspace_bytes, void* scratch,
                             size_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ADASPLASH_HIP_H */
