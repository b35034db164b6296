/* C ABI of the MI355X (gfx950) key/value cache held in 4 bits: pages and slots
 * from request lengths, storing and reading rows, and attention over the
 * cache. No counterpart in the reference, whose attention reads fp16 tensors.
 *
 * Cache. Keys and values are E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
 * negatives) with one E8M0 scale (2^(byte - 127); 255 is NaN) per 32 head dims
 * of a token (the OCP MX format MXFP4), in pages of `page` tokens (64, 128 or
 * 256), for head dims of 64 or 128:
 *   codes  [pages, Hkv, page, D/2] bytes; dim 2i in the low, 2i+1 in the high
 *          nibble of byte i
 *   scales [pages, Hkv, page/64, 16, D/32, 4] bytes; the scale of dims
 *          32j..32j+31 of a page's token 64a + 16c + b at [a, b, j, c], so that a
 *          lane reads the scales of four 16-token tiles as one dword
 * A block of 32 values x is stored with scale byte E - 2, E the biased fp32
 * exponent of max |x| (at least 1; 255, a block of NaN, where some x is infinite
 * or NaN), as the nearest codes, ties to even, saturating at 6 scales. fp16
 * rows hold 16384 <= max |x| <= 65504 as well; a cache of bf16 rows read as fp16
 * gives infinities for values past 65504.
 *
 * Lengths, slots, tables and other int arguments named here as device arrays
 * are read on the GPU and not checked by the host; any value is safe (see each).
 * All pointers are device pointers; calls are asynchronous on `stream`, return
 * 0, 1 for a rejected argument (nothing launched) or 2 for a HIP error, and set
 * kv4_last_error() for the calling thread.
 */
#ifndef GFX906_AMD_KV4_H
#define GFX906_AMD_KV4_H

#include <stddef.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KV4_DTYPE_F16 0
#define KV4_DTYPE_BF16 1
#define KV4_MAX_REQUESTS 4096

/* Pages and slots for new tokens. Request b holds lens[b] tokens, in pages
 * table[b][0 .. ceil(lens[b] / page)), and gets new_lens[b] more (negative counts are
 * taken as 0). Requests take the pages they lack from free_pages[*used ..), in
 * request order; written are
 *   table[b][...]   the new pages (rows table_stride apart; W columns)
 *   slots[0..n_slots)  page * `page` + place of every new token, requests one after
 *                   another; -1 for a token without a page (the free list or the
 *                   table's row ended, or a held page is negative) and behind the last
 *   cu_new[0..B]    first slot of every request, and their number (int32; saturates)
 *   lens_out[b]     lens[b] + new_lens[b]
 *   used_out        *used + the pages lacked, at most n_free
 *   missing         pages that could not be taken: the free list ended (table
 *                   entry -1), or the table's row did (its place in the free list is
 *                   passed over)
 * The arrays written must not overlap those read, except table. */
int kv4_plan_pages(const int* lens, const int* new_lens, int* table, long long table_stride, int W,
                   const int* free_pages, int n_free, const int* used, int B, int page,
                   int n_slots, int* slots, int* cu_new, int* lens_out, int* used_out,
                   int* missing, hipStream_t stream);

/* Stores rows t of k and v ([T, Hkv, D], fp16 or bf16; strides {token, head} in
 * elements, head dim contiguous, 16-byte aligned rows) at slots[t]; a slot outside
 * [0, pages * page) stores nothing. Slots of stored rows must differ: two rows with
 * one slot leave some mix of both there. */
int kv4_store(const void* k, const void* v, const long long* k_strides, const long long* v_strides,
              int dtype, int T, int Hkv, int D, const int* slots, void* k_codes, void* k_scales,
              void* v_codes, void* v_scales, int pages, int page, hipStream_t stream);

/* Reads rows slots[t] of the cache into contiguous k and v [T, Hkv, D]; a slot
 * outside the cache reads as zeros. */
int kv4_load(void* k, void* v, int dtype, int T, int Hkv, int D, const int* slots,
             const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
             int pages, int page, hipStream_t stream);

/* o = softmax(scale q k^T) v over the cache, for T query rows q [T, Hq, D] of B
 * requests: rows cu_q[b] .. cu_q[b+1] belong to request b (cu_q NULL: row b, T = B),
 * whose lens[b] tokens lie in pages table[b][...]. Query head h reads kv head
 * h / (Hq / Hkv). With causal != 0 the n queries of a request are its last n tokens
 * and see no later one; otherwise they see all of its tokens. A row that sees no key, or
 * only such of score -inf, is 0; a token that a row does not see adds nothing to it, whatever
 * it holds. Keys in pages outside [0, pages) or behind the table's last column weigh
 * nothing; cu_q is taken as clamped to 0 .. T. Rows outside every request, and queries
 * past the first max_q of one, are left as they were. q and o: strides {token, head} in
 * elements, head dim contiguous, q's rows 16-byte and o's 8-byte aligned; o's must
 * not overlap each other, q or the cache. workspace: 16-byte aligned,
 * kv4_attn_workspace_bytes() bytes, with max_len = W * page (and max_q = 1 where cu_q is
 * NULL); its content is neither read before it is written nor kept. */
size_t kv4_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int D, int max_q, int max_len);
int kv4_attn(const void* q, void* o, const long long* q_strides, const long long* o_strides,
             int dtype, int T, int B, int Hq, int Hkv, int D, const void* k_codes,
             const void* k_scales, const void* v_codes, const void* v_scales, int pages, int page,
             const int* table, long long table_stride, int W, const int* lens, const int* cu_q,
             int max_q, float scale, int causal, void* workspace, size_t workspace_bytes,
             hipStream_t stream);

/* Message for the last failed call on the calling thread, or NULL. */
const char* kv4_last_error(void);

#ifdef __cplusplus
}
#endif

#endif
