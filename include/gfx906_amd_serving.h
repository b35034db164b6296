/* C ABI of the serving operators of libgfx906_amd_attn.so: norms of queries and
 * keys with the position rotation, a paged key/value cache held in 8 bits with the
 * attention over it, the attention weights of its blocks and eviction by them. No
 * counterpart in the reference. (Pages and slots: kv4_plan_pages in
 * gfx906_amd_attn.h, whose requests, tables and lengths these calls share.)
 *
 * Pointers are device pointers, strides are in elements; int arguments named here
 * as device arrays are read on the GPU and not checked by the host; any value is
 * safe (see each). Calls are asynchronous on `stream`, return 0, 1 for a rejected
 * argument (nothing launched) or 2 for a HIP error, and set the *_last_error() of
 * the calling thread.
 */
#ifndef GFX906_AMD_SERVING_H
#define GFX906_AMD_SERVING_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KV8_DTYPE_F16 0
#define KV8_DTYPE_BF16 1
#define KV8_MAX_REQUESTS 4096
#define KV8_BLOCK 64 /* tokens of a head that share a scale */

/* -- Norms of queries and keys for each head, with the position rotation.
 *
 * For every row x of q [B, S, Hq, D] and of k [B, S, Hk, D] (fp16 or bf16; strides
 * {batch, token, head}, head dim contiguous, D a multiple of 8 up to 512; either
 * may have no heads and null pointers):
 *   y = x / sqrt(mean(x^2) + eps) * weight      (q_weight, k_weight: [D] or NULL for 1)
 * then pairs of the first R dims are turned by the angle whose cosine and sine are
 * in row p of cos and sin ([N, R/2] fp32, rows angle_stride apart):
 *   (y_i, y_j) <- (c y_i - s y_j, s y_i + c y_j)
 * i, j = 2n, 2n + 1 (neighbours != 0; R a multiple of 8) or n, n + R/2 (R a multiple
 * of 16). p is positions[b][s] (strides {batch, token}) or, where positions is NULL, s;
 * a row whose position lies outside 0 .. N-1 gets NaN in its turned dims. R = 0: no rotation.
 * Everything in fp32, rounded once. weight_f32: the weights are fp32, else of the
 * rows' type. Rows are 16-byte aligned, strides multiples of 8, rows of angles 16-byte aligned;
 * the results' rows must not overlap each other; q_out may be q, and k_out k (with equal strides).
 */
int qk_norm_rotate(const void* q, const void* k, void* q_out, void* k_out,
                   const long long* q_strides, const long long* k_strides,
                   const long long* q_out_strides, const long long* k_out_strides, int dtype, int B,
                   int S, int Hq, int Hk, int D, const void* q_weight, const void* k_weight,
                   int weight_f32, float eps, const float* cos, const float* sin,
                   long long angle_stride, int N, int R, int neighbours, const int* positions,
                   const long long* p_strides, hipStream_t stream);
const char* qk_norm_rotate_last_error(void);

/* -- A key/value cache held in 8 bits.
 *
 * Keys and values are E4M3 numbers (OCP: bias 7, largest 448, 0x7f NaN) times a scale
 * that the 64 tokens of a block share for a kv head, a power of two from 2^-15 to 2^7, in
 * pages of `page` tokens (64, 128 or 256), for head dims of 64 or 128:
 *   k codes [pages, Hkv, page, D] bytes
 *   v codes [pages, Hkv, page/64, D, 64] bytes; token t of a block at place
 *           16 ((t >> 2) & 3) + 8 (t >> 5) + 4 ((t >> 4) & 1) + (t & 3), so that a lane
 *           reads the 16 tokens of a dim that it has in the matrix product
 *   scales  [pages, Hkv, page/64] fp32, of k and of v
 * Every number that a cache holds is one of fp16 and of bf16 too, so attention works on
 * what is held. A block's scale is the least that holds its largest finite |x| as 448
 * scales or less; finite values past 448 * 2^7 = 57344 are held as that, infinite and NaN ones
 * as NaN. Codes are the nearest, ties to even.
 */

/* Stores rows cu_new[b] .. cu_new[b+1] of k and v ([T, Hkv, D]; strides {token, head},
 * multiples of 8, 16-byte aligned rows) as the last tokens of request b, which holds lens[b]
 * tokens, the new ones among them, in pages table[b][...] (cu_new NULL: row b, T = B). A block
 * with older tokens keeps its scale or takes a larger one, to which the older tokens' codes are
 * rounded; what a block held behind them does not count. Rows past the request's
 * length or in pages outside [0, pages) or behind the table's last column are not stored; cu_new
 * is taken as clamped to 0 .. T. No block may be written for two requests. weights: NULL, or as in
 * kv8_weigh: 0 is written for blocks whose first token is stored. */
int kv8_store(const void* k, const void* v, const long long* k_strides, const long long* v_strides,
              int dtype, int T, int B, int Hkv, int D, void* k_codes, float* k_scales, void* v_codes,
              float* v_scales, int pages, int page, const int* table, long long table_stride, int W,
              const int* lens, const int* cu_new, float* weights, hipStream_t stream);

/* Reads rows slots[t] (page * `page` + place in it) into contiguous k and v [T, Hkv, D]; a
 * slot outside the cache reads as zeros. */
int kv8_load(void* k, void* v, int dtype, int T, int Hkv, int D, const int* slots,
             const void* k_codes, const float* k_scales, const void* v_codes,
             const float* v_scales, int pages, int page, hipStream_t stream);

/* o = softmax(scale q k^T) v over the cache, as kv4_attn: T query rows q [T, Hq, D], rows
 * cu_q[b] .. cu_q[b+1] of request b (cu_q NULL: row b, T = B), whose lens[b] tokens lie in pages
 * table[b][...]; query head h reads kv head h / (Hq / Hkv). With causal != 0 the n queries of a
 * request are its last n tokens and see no later one. A row that sees no key, or only such of score
 * -inf, is 0; a token that a row does not see adds nothing to it, whatever it holds. Keys in
 * pages outside [0, pages) or behind the table's last column weigh nothing; cu_q is taken as
 * clamped to 0 .. T. Rows outside every request, and queries past the first max_q of one, are left
 * as they were. lse: NULL, or fp32 [T, Hq], the logarithm of the sum of exp(scale q k) over the
 * row's keys (-inf where it sees none). q and o: strides {token, head}, head dim contiguous, q's
 * rows 16-byte and o's 8-byte aligned; o's must not overlap each other, q or the cache. workspace:
 * 16-byte aligned, kv8_attn_workspace_bytes() bytes, with max_len = W * page (and max_q = 1 where
 * cu_q is NULL); its content is neither read before it is written nor kept. */
size_t kv8_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int D, int max_q, int max_len);
int kv8_attn(const void* q, void* o, float* lse, const long long* q_strides,
             const long long* o_strides, int dtype, int T, int B, int Hq, int Hkv, int D,
             const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales,
             int pages, int page, const int* table, long long table_stride, int W, const int* lens,
             const int* cu_q, int max_q, float scale, int causal, void* workspace,
             size_t workspace_bytes, hipStream_t stream);

/* -- Accumulated attention weights of the cache's blocks, and eviction by them. */

/* weights[page][kv head][block] += sum of exp(scale q k - lse) over the block's tokens, the
 * queries of its request that see them and the query heads of the kv head: with kv8_attn's
 * arguments and its lse [T, Hq] (packed fp32), the attention that the block's tokens got.
 * weights: fp32 [pages, Hkv, page/64]. Queries past the first max_q of a request do not count. Rows
 * of lse -inf add nothing. Sums are fp32 in an order that sizes alone set; where requests share
 * a page, their sums are added in any order. workspace: kv8_weigh_workspace_bytes() bytes (max_q = 1
 * where cu_q is NULL; may be 0), 4-byte aligned. */
size_t kv8_weigh_workspace_bytes(int T, int B, int Hq, int Hkv, int max_q, int W, int page);
int kv8_weigh(float* weights, const void* q, const long long* q_strides, int dtype, const float* lse,
              int T, int B, int Hq, int Hkv, int D, const void* k_codes, const float* k_scales,
              int pages, int page, const int* table, long long table_stride, int W, const int* lens,
              const int* cu_q, int max_q, float scale, int causal, void* workspace,
              size_t workspace_bytes, hipStream_t stream);

/* Every request with more than keep[b] pages (n = ceil(lens[b] / page) of at most W) gives back
 * n - keep[b] of them (fewer, where fewer may go): those of least weight among its pages first ..
 * n - recent - 1, of equal ones the earlier. A page's weight is the sum of weights[page] (fp32
 * [pages, Hkv, page/64]) over heads and blocks in fp64, NaN counting as largest; table entries
 * outside [0, pages) weigh least. The row closes up in place (-1 behind the last page that stays), lens_out[b]
 * = lens[b] less the evicted pages' tokens. The pages given back, in the order of the requests and
 * of their rows, go before free_pages[*used], from where kv4_plan_pages takes pages:
 * into free_pages[*used_out .. *used), *used_out = *used less their number; *lost counts
 * those that had no room (the earlier ones go in). first >= 0, recent >= 1: the last page, which
 * may be short, always stays. workspace: kv8_evict_workspace_bytes(), 8-byte aligned. */
size_t kv8_evict_workspace_bytes(int B, int W);
int kv8_evict(const float* weights, int pages, int Hkv, int page, int* table,
              long long table_stride, int W, const int* lens, const int* keep, int B, int first,
              int recent, int* free_pages, int n_free, const int* used, int* lens_out, int* used_out,
              int* lost, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Message for the last failed kv8_* call on the calling thread, or NULL. */
const char* kv8_last_error(void);

#ifdef __cplusplus
}
#endif

#endif
