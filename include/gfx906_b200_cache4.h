/* Paged 4-bit key/value cache for NVIDIA B200 (sm_100a): C ABI.
 *
 * The cache is device memory of pages x kv_heads x gfx906_b200_cache4_page_bytes(D)
 * bytes, 16-byte aligned. A page holds 64 tokens of one kv head, K and V, each
 * value as an e2m1 code with an e4m3 scale per 16 channels of a token, times
 * one fp32 factor per kv head (k_scale, v_scale; a null pointer means 1). The
 * head dim D is 64 or 128. A slot is page * 64 + place in the page.
 *
 * All pointers are device pointers on the current device; calls are
 * asynchronous on `stream`, allocate nothing and can be captured in CUDA
 * graphs. Status codes are those of gfx906_b200_attn.h. dtype: 0 = fp16,
 * 1 = bf16, 2 = fp32 (reads only). Strides are in elements; rows (the last
 * dimension) are contiguous, start on 16 bytes, and strides are multiples of 8.
 * gfx906_b200_attn_set_sm_limit does not hold for these kernels: their blocks
 * are many and short, and go to any SM that is free.
 */
#ifndef GFX906_B200_CACHE4_H
#define GFX906_B200_CACHE4_H

#include "gfx906_b200_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of one kv head (72 * D), or 0 for an unsupported D. */
GFX906_B200_API int gfx906_b200_cache4_page_bytes(int D);

/* One step of page bookkeeping for `requests` (at most 8192) requests, int32
 * throughout. Request r holds lengths[r] tokens in the pages
 * tables[r * width ...]; counts[r] >= 0 tokens are appended to it, or it has
 * ended (counts[r] < 0) and its pages go back. free_pages is a stack of
 * free_pages_size entries whose first *free_count are free.
 *  1. Pages of ended requests are pushed, in the order of the requests and of
 *     their tables; their new length is 0.
 *  2. In the order of the requests, each that needs more pages gets them off
 *     the top of the stack. A request is refused when its tokens would not fit
 *     its row of the table, when its tokens end behind `tokens`, or when it
 *     needs pages and the requests up to and with it need more than there are.
 * Outputs: query_start [requests + 1], the sums of the counts (refused or not),
 * at most 2^31 - 1;
 * lengths_out [requests]; added [requests], the tokens appended (0: refused or
 * ended); slots and positions [tokens], the slot and position of each token,
 * -1 for tokens of refused requests and behind the last (the slot alone where
 * the page id is negative or has no slots in 31 bits); *free_count_out.
 * tables and free_pages are updated in place, only in entries that the inputs
 * do not use, so a call may be repeated; the other outputs may not alias inputs. */
GFX906_B200_API int gfx906_b200_cache4_plan(int* tables, const int* lengths, const int* counts, int* free_pages,
                                            const int* free_count, int requests, int width, int free_pages_size,
                                            int tokens, int* query_start, int* lengths_out, int* added, int* slots,
                                            int* positions, int* free_count_out, cudaStream_t stream);

/* Writes k and v [tokens, kv_heads, D] (fp16 or bf16) to their slots. Tokens
 * whose slot is outside the cache are skipped; slots are distinct. Per 16
 * channels of a token: scale = e4m3(max|x| / (6 factor)), at least 2^-9 and at
 * most 448, code = e2m1(x / (scale factor)), both to nearest even. Infinities
 * saturate, NaN is held as zero: the cache holds finite numbers only. */
GFX906_B200_API int gfx906_b200_cache4_write(const void* k, const void* v, int dtype, long long k_stride_t,
                                             long long k_stride_h, long long v_stride_t, long long v_stride_h,
                                             int tokens, int kv_heads, int D, void* cache, int pages,
                                             const int* slots, const float* k_scale, const float* v_scale,
                                             cudaStream_t stream);

/* Reads the tokens at `slots` back into contiguous k and v [tokens, kv_heads, D]
 * of the given dtype; zeros for slots outside the cache. */
GFX906_B200_API int gfx906_b200_cache4_read(const void* cache, int pages, const int* slots, const float* k_scale,
                                            const float* v_scale, int tokens, int kv_heads, int D, void* k, void* v,
                                            int dtype, cudaStream_t stream);

/* Attention of new tokens against the cache. Request r's query rows are
 * query_start[r] .. query_start[r + 1] of q [tokens, heads, D] (query_start does
 * not decrease; whatever it holds, no row outside q is touched); it attends to
 * its lengths[r] tokens in tables[r * width ...]. Query head h uses kv head
 * h / (heads / kv_heads). With causal != 0 the last query row sees every
 * token and each row before it one less; rows that see none get zeros. */
typedef struct gfx906_b200_cache4_attn_args {
  const void* q;                    /* [tokens, heads, D], dtype */
  void* o;                          /* [tokens, heads, D], dtype */
  const void* cache;
  const int* tables;                /* [requests, width] */
  const int* lengths;               /* [requests] */
  const int* query_start;           /* [requests + 1] */
  const float* k_scale;             /* [kv_heads] or null */
  const float* v_scale;             /* [kv_heads] or null */
  long long q_stride_t, q_stride_h; /* elements */
  long long o_stride_t, o_stride_h;
  int dtype;                        /* 0 = fp16, 1 = bf16 */
  int tokens, heads, kv_heads, D;
  int pages, requests, width;       /* requests <= 8192 */
  int max_tokens;                   /* no request has more query rows (a hint for the schedule) */
  int causal;
  int zero_rest;                    /* 1: zero the rows of o behind the last request, 0: leave them */
  float scale;                      /* finite */
} gfx906_b200_cache4_attn_args;

/* Scratch bytes that gfx906_b200_cache4_attn needs for these arguments (only
 * sizes are read); 256-byte aligned device memory, contents irrelevant. Calls
 * that may overlap on the GPU need workspaces of their own. */
GFX906_B200_API size_t gfx906_b200_cache4_attn_workspace_size(const gfx906_b200_cache4_attn_args* args);
GFX906_B200_API int gfx906_b200_cache4_attn(const gfx906_b200_cache4_attn_args* args, void* workspace,
                                            size_t workspace_bytes, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GFX906_B200_CACHE4_H */
