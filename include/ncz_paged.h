/* ncz_paged.h -- C ABI of the paged key-value cache in libncz_flash.so
 * (sm_100a): the step from a forward over whole slices (ncz_flash.h) to
 * generating token by token.
 *
 *   ncz_paged_plan    block tables and slot maps from request lengths
 *   ncz_paged_append  new K/V rows into the cache's pages
 *   ncz_paged_decode  attention of one new token per request over the pages
 *
 * The reference has no cache and no decoding step; its attention takes whole
 * K/V slices (src/flash.zig:31-70).
 *
 * A cache is two arrays of pages, K and V: element (page, token, head, d) lies
 * at page * page_stride + token * token_stride + head * head_stride + d, so
 * tokens or heads may be outermost inside a page.  The row of a request's key
 * j is row j % page_size of the page block_table[request][j / page_size]; the
 * slot of a row is page * page_size + row.  All pointers are DEVICE pointers
 * owned by the caller (descriptors and caches are host structs, read during
 * the call only).  Calls are asynchronous on `stream` (NULL = default stream),
 * allocate nothing, and validate before launching.  Return codes are the
 * ncz_status values of ncz_flash.h. */
#ifndef NCZ_PAGED_H
#define NCZ_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element type next to NCZ_DTYPE_F16 (1) and NCZ_DTYPE_BF16 (2): 8-bit
 * floats (4 exponent, 3 mantissa bits, largest value 448), each standing for
 * value * scale of its K or V head. */
#define NCZ_DTYPE_E4M3 3

typedef struct ncz_paged_cache {
    void *k;
    void *v;
    const float *k_scale; /* [kv_heads], NULL = 1; e4m3 only */
    const float *v_scale;
    size_t num_pages;
    size_t page_size; /* any number of rows >= 1 */
    size_t kv_heads; /* at most 65536 */
    size_t head_dim; /* 16 (not e4m3), 32, 64 or 128 */
    size_t k_page_stride, k_token_stride, k_head_stride; /* elements */
    size_t v_page_stride, v_token_stride, v_head_stride;
    int32_t dtype; /* NCZ_DTYPE_F16, NCZ_DTYPE_BF16 or NCZ_DTYPE_E4M3 */
} ncz_paged_cache;

/* The rules every call applies to its cache.  k and v are 16-byte aligned, as
 * is every stride in bytes (else NCZ_ERROR_MISALIGNED); no two rows of K (of
 * V) overlap; at most 2^31 - 1 pages and fewer than 2^31 rows a page. */
int ncz_paged_validate(const ncz_paged_cache *cache);

/* One step's bookkeeping for `requests` requests: request r holds held[r]
 * tokens in the cache and brings added[r] new ones (0 = none this step).
 * Pages are taken from a stack: free_pages[0 .. *free_count) are free, and the
 * i-th page taken, in request order, is free_pages[*free_count - 1 - i].
 *
 *   block_table[r][..]  entries of the pages r needs beyond those it holds
 *   seq_lens[r]         held[r] + added[r] (may be `held` itself)
 *   starts[r]           new tokens of the requests before r; starts[requests]
 *                       their total (clamped to slot_capacity)
 *   slots[t]            slot of new token t, the requests' new tokens packed in
 *                       request order; -1 behind the last one
 *   positions[t]        its position in its request (at most 2^31 - 1); 0 behind the
 *                       last one
 *   *left               pages free after the call (may be `free_count` itself)
 *   status[0..3]        new tokens, pages taken, requests refused, and new
 *                       tokens that slot_capacity left out
 *
 * A request is refused when its lengths are negative, when its tokens would
 * not fit table_width pages, or when the stack no longer holds all the pages it
 * needs (pages asked for by the requests before it count whether or not those
 * got them): its table row and length stay, its slots are -1, and it takes no
 * page.  No other entry of block_table is touched.  A held page whose table
 * entry is negative gives slot -1.  positions, starts and status may be NULL.
 * Apart from the two pairs named, no output may overlap another array (lengths
 * that do are refused).  Arrays are aligned to their elements.
 *
 * Where seq_lens is `held` or left is free_count, 8 SMs do the work, else up to 128:
 * the same time for a step of one token each, twice that for long prompts (98304 new
 * tokens of 48 requests 16.2 and 8.8 us). */
typedef struct ncz_paged_plan_desc {
    const int32_t *held;
    const int32_t *added;
    const int32_t *free_pages;
    const int32_t *free_count;
    int32_t *block_table;
    int32_t *seq_lens;
    int64_t *slots;
    int32_t *positions;
    int32_t *starts;
    int32_t *left;
    int32_t *status;
    size_t requests; /* at most 2^24 */
    size_t table_width;
    size_t table_stride;  /* elements between rows of block_table */
    size_t free_capacity; /* elements of free_pages; *free_count is clamped to it */
    size_t slot_capacity; /* elements of slots and positions */
    size_t page_size;
    int32_t device; /* CUDA ordinal, -1 = current */
    void *stream;
} ncz_paged_plan_desc;

int ncz_paged_plan(const ncz_paged_plan_desc *desc);

/* Writes rows k[t][h][..] and v[t][h][..] of `tokens` new tokens to the slots
 * slots[t]; a slot below 0 or past the cache is skipped.  f16 and bf16 caches
 * take rows of their own type, unchanged.  An e4m3 cache takes f16 or bf16 rows
 * and holds the f32 quotient x / scale[h] rounded to nearest even, values past 448 as 448 (NaN
 * stays NaN).  k and v may have any strides (rows of head_dim elements).  No
 * slot may be given twice in one call: its row would be that of either token,
 * or parts of both.  k and v lie outside the cache, and K and V of the cache are
 * apart (decode takes a cache that is both at once). */
typedef struct ncz_paged_append_desc {
    const void *k;
    const void *v;
    const int64_t *slots;
    size_t tokens;
    size_t k_token_stride, k_head_stride; /* elements */
    size_t v_token_stride, v_head_stride;
    int32_t in_dtype; /* NCZ_DTYPE_F16 or NCZ_DTYPE_BF16 */
    int32_t device;
    void *stream;
} ncz_paged_append_desc;

int ncz_paged_append(const ncz_paged_cache *cache, const ncz_paged_append_desc *desc);

/* Attention of one new token per request: with len = seq_lens[b] (clamped to
 * 0 .. table_width * page_size), for query head h and its K/V head
 * h / (q_heads / kv_heads), over the keys j in [len - window, len) (window 0:
 * [0, len)) whose table entry is a page of the cache:
 *
 *   s_j = scale * q[b][h] . k_j,  o[b][h] = sum_j exp(s_j) v_j / sum_j exp(s_j),
 *   lse[b][h] = ln sum_j exp(s_j)
 *
 * Entries outside [0, num_pages) are absent pages (say, given back once a
 * window has passed them): their keys are left out.  A row without keys gives
 * o = 0 and lse = -infinity.  Nothing in an absent page or behind len affects
 * the result.  Scores, softmax and sums are f32.  bf16 q over an e4m3 cache is held in
 * f16, times a power of two of its row: elements below 2^-17 of the row's largest one are
 * off by at most 2^-25 of that, the others are exact.  P goes to the tensor
 * cores in 16-bit parts: two, but three for bf16 K/V with f32 o and one for
 * e4m3 K/V with bf16 o.  bf16 parts for bf16 K/V; f16 parts else, in which the weight of
 * a key is off by up to 2^-33 of the row's largest as well.
 *
 * q is f16 or bf16 (the cache's type; either for e4m3); o is f32, f16 or bf16;
 * lse may be NULL, else f32 [batch][q_heads].  q and o may have any strides
 * that keep the rows of o apart.  o, lse and workspace overlap nothing else; o in
 * place of q is refused.
 *
 * The lengths are on the device, so the kernel and the grid are chosen by the longest
 * row there may be, table_width * page_size keys (or window, if that is less): a table
 * much wider than its rows costs short rows time (one request of 1000 keys, 8 K/V heads,
 * head_dim 128: 7.1 us with a table of 1024 keys, 8.8 of 2048, 9.8 of 131072).
 *
 * The keys of one request and head are split over CTAs that each leave a
 * partial result in `workspace`, joined by a second kernel.  The workspace is
 * at least the bytes that ncz_paged_decode_workspace reports for the cache and
 * q_heads, 16-byte aligned, for any batch; it needs no initial contents and
 * keeps none.  Calls that may run at the same time (streams, or captured graphs
 * replayed side by side) each need their own; calls on one stream may share one,
 * whichever host threads make them. */
typedef struct ncz_paged_decode_desc {
    const void *q;
    void *o;
    float *lse;
    const int32_t *block_table;
    const int32_t *seq_lens;
    size_t batch; /* at most 2^24 */
    size_t q_heads; /* at most 65536, a multiple of the cache's kv_heads */
    size_t table_width;
    size_t table_stride;                  /* elements between rows of block_table */
    size_t q_batch_stride, q_head_stride; /* elements */
    size_t o_batch_stride, o_head_stride;
    size_t window; /* 0 = every cached key */
    float scale;
    int32_t q_dtype; /* NCZ_DTYPE_F16 or NCZ_DTYPE_BF16 */
    int32_t o_dtype; /* NCZ_DTYPE_F32, NCZ_DTYPE_F16 or NCZ_DTYPE_BF16 */
    void *workspace;
    size_t workspace_bytes;
    int32_t device;
    void *stream;
} ncz_paged_decode_desc;

int ncz_paged_decode(const ncz_paged_cache *cache, const ncz_paged_decode_desc *desc);

/* Synchronises `device` (-1 = current), then reads and clears the bounded-wait
 * status word of its decode kernels: NCZ_SUCCESS, or NCZ_ERROR_DEVICE_TIMEOUT
 * when a wait inside a kernel ran past the wait limit since the last call (that
 * kernel then stopped cleanly; its o and lse are incomplete).  The forward's and the
 * GEMM's status words are their own (ncz_flash_sync_status, ncz_mma_sync_status): a
 * program that checks its steps asks for each kind of kernel it ran. */
int ncz_paged_sync_status(int device);

/* Test hooks (failure detection without a GPU fault), device -1 = current.
 * ncz_paged_test_set_wait_limit: bound of every in-kernel wait in SM cycles (0
 * restores the default, about 2 s).  ncz_paged_test_drop_scores: while enabled,
 * the first CTA of a launch of the tcgen05 kernel (many query heads per K/V head)
 * never announces its first scores, so a wait runs out.  ncz_paged_test_leave_merge:
 * while enabled, one of the four softmax warps of that CTA gives up where its first
 * item ends, as at a wait that ran out, while the others are about to merge. */
int ncz_paged_test_set_wait_limit(int device, uint64_t cycles);
int ncz_paged_test_drop_scores(int device, int enable);
int ncz_paged_test_leave_merge(int device, int enable);

/* Bytes of workspace for ncz_paged_decode on `device` (-1 = current). */
int ncz_paged_decode_workspace(const ncz_paged_cache *cache, size_t q_heads, int device, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* NCZ_PAGED_H */
