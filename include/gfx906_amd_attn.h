/* C ABI of the MI355X (gfx950) flash-attention forward, and at the end of
 * forms of it for long contexts (a 4-bit key/value cache, sparse attention) and of
 * what serves them: head norms with rotation, an 8-bit cache, eviction.
 *
 * All pointers are device pointers. For launch() and attn_fwd() the tensors
 * are contiguous fp16:
 *   q, o : [B, H, Sq,  D]
 *   k, v : [B, H, Skv, D]
 * attn_fwd_ex() also takes bf16 and per-tensor strides.
 * D must be <= 64 and a multiple of 8, or 128, or 512. Sq != Skv is allowed.
 * o[b,h,i,:] = sum_j softmax_j(scale * <q[b,h,i,:], k[b,h,j,:]>) v[b,h,j,:],
 * rounded to the element type; rows with Skv == 0 are written as zeros. A
 * score of -inf weighs nothing; a row of nothing else is NaN (0 for D = 128).
 * Calls are asynchronous on `stream`. The only state kept between calls is
 * the static scratch of the calls that split key ranges without a caller
 * workspace (launch(), attn_fwd(), attn_fwd_split_static(), and conv3d_fwd()
 * and launch_conv3d(), which split reductions in it): a device array
 * of attn_split_scratch_capacity() bytes that is part of the library's code
 * object, so it is held on every GPU where the library's kernels are loaded,
 * until the process ends. Each call takes a part of it. Calls that use the
 * same part are ordered on the GPU whatever their streams (each waits for the
 * previous one); different streams get different parts while these last, and
 * their calls may run side by side. A call under stream capture neither waits
 * nor is waited for: a graph that contains one is ordered only by the stream
 * it is launched on, and must not run concurrently with other streams' calls
 * that use the scratch.
 */
#ifndef GFX906_AMD_ATTN_H
#define GFX906_AMD_ATTN_H

#include <stddef.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types for attn_fwd_ex(). */
#define ATTN_DTYPE_F16 0
#define ATTN_DTYPE_BF16 1

/* Drop-in for the reference entry point of the same name and signature:
 * declared at attn.cpp:4-5, defined at attn_kernel.hip:710-742. Returns
 * nothing; on a rejected argument or launch failure no kernel runs and the
 * reason is available from attn_last_error(). When B*H*Sq is too small to
 * fill the GPU (a one-head VAE attention), or fills it a whole number of times
 * and a little more, it splits key ranges as attn_fwd_split_static() does, in
 * the static scratch. */
void launch(const void* q, const void* k, const void* v, void* o,
            int B, int H, int Sq, int Skv, int D, float scale, hipStream_t stream);

/* Same computation as launch(), returning 0 on success, 1 for a rejected
 * argument (nothing launched) and 2 for a HIP launch error. It replaces the
 * launch-then-check sequence of the reference binding (attn.cpp:17-19), which
 * has no error path of its own. */
int attn_fwd(const void* q, const void* k, const void* v, void* o,
             int B, int H, int Sq, int Skv, int D, float scale, hipStream_t stream);

/* attn_fwd() for fp16 or bf16 (dtype = ATTN_DTYPE_F16 / ATTN_DTYPE_BF16,
 * the same type for q, k, v and o) and strided tensors, never splitting the
 * key range over workgroups. Each *_strides
 * points to four element strides {batch, head, sequence, head dim} of that
 * tensor, or is NULL for the contiguous layout. Strides are non-negative;
 * input strides may be 0 (a tensor broadcast over batch or heads) but no two
 * elements of o may share an address. Two layouts are accepted:
 *  - head dim contiguous (stride 1) for q, k, v and o: q, k, v 16-byte
 *    aligned with other strides multiples of 8 elements, o 8-byte aligned
 *    with multiples of 4; k/v sequence strides at most 2^24;
 *  - D == 512 with token-contiguous k and v (sequence stride 1, head-dim
 *    stride not 1), as in a [b, c, h*w] activation viewed as
 *    [b, 1, h*w, c]: k, v 16-byte aligned, batch/head/head-dim strides
 *    multiples of 8, Skv % 8 == 0, (D-1)*stride_d + Skv < 2^30 per head;
 *    q and o then take any strides (2-byte aligned).
 * Return codes as attn_fwd(). No counterpart in the reference, whose hook
 * casts bf16 to fp16 and back (deploy/gfx906_attention.py:71-75, 99-100) and
 * whose binding copies strided inputs (attn.cpp:15), including the VAE's
 * transposed views (deploy/gfx906_attention.py:102-104). */
int attn_fwd_ex(const void* q, const void* k, const void* v, void* o,
                int B, int H, int Sq, int Skv, int D, float scale, hipStream_t stream,
                int dtype, const long long* q_strides, const long long* k_strides,
                const long long* v_strides, const long long* o_strides);

/* Bytes of device workspace attn_fwd_split() takes for this problem on the
 * current device: 0 when no split pays (the call then runs as attn_fwd_ex()),
 * else room for the partial results of the split key ranges: of every row
 * when the problem's workgroups do not fill the GPU, of the last rows alone
 * (at most 96 MiB) when they fill it a whole number of times and a little
 * more. No counterpart in the reference. */
size_t attn_split_workspace_bytes(int B, int H, int Sq, int Skv, int D);

/* attn_fwd_ex() that, when B*H*Sq is too small to fill the GPU (a VAE
 * attention over one head, short problems) or leaves its last round of
 * workgroups nearly empty, splits key ranges over more workgroups: each
 * writes its unnormalised partial output and running max/sum to `workspace` (device memory, 16-byte aligned, at least
 * attn_split_workspace_bytes() bytes; may be NULL when that is 0) and a
 * second kernel merges them into o. Same arguments and return codes as
 * attn_fwd_ex(), plus 1 for a missing or short workspace (problems that fill
 * the GPU then run unsplit instead). Results agree with
 * attn_fwd_ex() to fp32 rounding of the merge (not bit for bit). Calls on one
 * workspace must not overlap. No counterpart in the reference. */
int attn_fwd_split(const void* q, const void* k, const void* v, void* o,
                   int B, int H, int Sq, int Skv, int D, float scale, hipStream_t stream,
                   int dtype, const long long* q_strides, const long long* k_strides,
                   const long long* v_strides, const long long* o_strides,
                   void* workspace, size_t workspace_bytes);

/* attn_fwd_split() that allocates nothing: the split partial results go to
 * the library's static scratch (attn_split_scratch_capacity() bytes, 96 MiB,
 * on every GPU where the library's kernels are loaded, held until the
 * process ends). For callers that cannot allocate device memory: code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc.
 * The split count is the best one whose partial results fit the scratch:
 * the same as attn_fwd_split()'s whenever attn_split_workspace_bytes() <=
 * capacity (then the results are bit-identical), fewer splits or none
 * otherwise. Problems that do not split use no scratch. Calls that use the
 * same part of the scratch are ordered across streams (see the top of this
 * file); under stream capture the first such call on a device must have
 * been made outside capture (it sets the scratch up), else status 1; problems
 * that fill the GPU do not use the scratch under capture and run unsplit. Same
 * arguments and return codes as attn_fwd_split() otherwise. No counterpart
 * in the reference. */
int attn_fwd_split_static(const void* q, const void* k, const void* v, void* o,
                          int B, int H, int Sq, int Skv, int D, float scale, hipStream_t stream,
                          int dtype, const long long* q_strides, const long long* k_strides,
                          const long long* v_strides, const long long* o_strides);

/* attn_fwd_split() on row copies of token-contiguous q, k and v (D = 512, o
 * token-contiguous too; any other strides, alignment and counts): the tensors
 * are first transposed into `copies` (16-byte aligned,
 * attn_row_copies_bytes() bytes, one launch) and the row-contiguous kernel
 * runs on those. For layouts that attn_fwd_split() does not read in place,
 * and faster than reading in place from about 5500 tokens. No counterpart in
 * the reference. */
size_t attn_row_copies_bytes(int B, int H, int Sq, int Skv, int D);
int attn_fwd_split_copied(const void* q, const void* k, const void* v, void* o, int B, int H,
                          int Sq, int Skv, int D, float scale, hipStream_t stream, int dtype,
                          const long long* q_strides, const long long* k_strides,
                          const long long* v_strides, const long long* o_strides, void* workspace,
                          size_t workspace_bytes, void* copies, size_t copies_bytes);

/* Bytes of the static scratch attn_fwd_split_static() uses. No counterpart in
 * the reference. */
size_t attn_split_scratch_capacity(void);

/* Message for the last failed launch()/attn_fwd()/attn_fwd_ex()/
 * attn_fwd_split()/attn_fwd_split_static() on the calling thread, or NULL if
 * the last call succeeded. No counterpart in the reference, whose launch()
 * (attn_kernel.hip:710-742) never reports errors. */
const char* attn_last_error(void);

/* -- A key/value cache held in 4 bits: pages and slots from request lengths,
 * storing and reading rows, and attention over the cache. No counterpart in the reference, whose attention reads fp16 tensors.
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
 * it holds (of an infinite value that it does see, with a weight that the element type rounds
 * to 0, comes an infinity or NaN). Keys in pages outside [0, pages) or behind the table's last column weigh
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

/* -- Sparse attention: every block of 128 query rows
 * reads a few blocks of keys, which a score of block means selects. No counterpart
 * in the reference, whose attention reads every key.
 *
 * Calls are asynchronous on `stream`, return 0, 1 for a rejected argument (nothing
 * launched) or 2 for a HIP error, and set sparse_last_error() for the calling
 * thread. Pointers are device pointers, strides in elements {batch, head,
 * sequence}, head dims contiguous, D 64 or 128, key blocks of 64 or 128 rows.
 */

#define SPARSE_DTYPE_F16 0
#define SPARSE_DTYPE_BF16 1
#define SPARSE_Q_BLOCK 128
#define SPARSE_MAX_BLOCKS 32768 /* key blocks of a head */
#define SPARSE_MAX_COUNT 2048   /* blocks chosen for a query block */

/* means[b][h][j][:] = mean of rows j*block .. of x [B, H, S, D] (the last block
 * may be short), summed in fp64 and rounded once to fp32; packed. x's rows are
 * 16-byte aligned. */
int sparse_block_means(const void* x, const long long* strides, int dtype, int B, int H, int S,
                       int D, int block, float* means, hipStream_t stream);

/* index[b][h][i][0..count): the key blocks of query block i, ascending, -1 behind
 * the last. Taken are those with the largest product of q_means[b][h][i] and
 * k_means[b][h / (Hq/Hkv)][j] (NaN counts as largest, equal products by the lower index).
 * A product is added up in fp64, within 2^-48 sum |q k| of the exact one and always in the
 * same order: sizes and the entry point do not change a choice. Means are packed fp32 [B, Hq, ceil(Sq/128), D] and
 * [B, Hkv, ceil(Skv/block), D], 16-byte aligned. With causal != 0 query row r stands at key position
 * r + Skv - Sq; blocks past the query block's last position are never taken, and
 * those that hold its own positions always (count must be at least 128/block + 1,
 * or their number where Sq < 128). workspace: sparse_select_workspace_bytes() bytes. */
size_t sparse_select_workspace_bytes(int B, int Hq, int Sq, int Skv, int block);
int sparse_select(const float* q_means, const float* k_means, int B, int Hq, int Hkv, int Sq,
                  int Skv, int D, int block, int count, int causal, int* index, void* workspace,
                  size_t workspace_bytes, hipStream_t stream);

/* The same from the query rows q [B, Hq, Sq, D] themselves (16-byte aligned), whose means
 * over 128 rows are taken as sparse_block_means does. workspace:
 * sparse_choose_workspace_bytes() bytes (0 for few query blocks, which take one kernel). */
size_t sparse_choose_workspace_bytes(int B, int Hq, int Sq, int Skv, int D, int block);
int sparse_choose(const void* q, const long long* q_strides, int dtype, const float* k_means, int B,
                  int Hq, int Hkv, int Sq, int Skv, int D, int block, int count, int causal,
                  int* index, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* o = softmax(scale q k^T) v over the keys of the blocks in index (as
 * sparse_select writes it, [B, Hq, ceil(Sq/128), count]; read on the GPU and not
 * checked by the host: an entry outside 0 .. ceil(Skv/block)-1, or not above every
 * valid entry before it, is passed over). causal as above. A row that sees no key,
 * or only such of score -inf, is 0; a key that a row does not see adds nothing to it, whatever
 * it holds (infinite values that it does see: as in kv4_attn). q, k, v: rows 16-byte aligned (k's and v's
 * apart, their strides at most 2^22); o: 8-byte, rows that do not overlap each other, k, v or
 * index; o may be q (the same rows).
 * workspace: 16-byte aligned, sparse_attn_workspace_bytes() bytes (may be 0). */
size_t sparse_attn_workspace_bytes(int B, int Hq, int Sq, int Skv, int D, int block, int count);
int sparse_attn(const void* q, const void* k, const void* v, void* o, const long long* q_strides,
                const long long* k_strides, const long long* v_strides,
                const long long* o_strides, int dtype, int B, int Hq, int Hkv, int Sq, int Skv,
                int D, float scale, const int* index, int block, int count, int causal,
                void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Message for the last failed call on the calling thread, or NULL. */
const char* sparse_last_error(void);

/* -- Serving operators around the caches: norms of queries and keys with the position rotation, a
 * paged key/value cache held in 8 bits with the attention over it, the attention weights of its blocks
 * and eviction by them. No counterpart in the reference. (Pages and slots: kv4_plan_pages above, whose
 * requests, tables and lengths these calls share.)
 *
 * Pointers are device pointers, strides are in elements; int arguments named here as device arrays
 * are read on the GPU and not checked by the host; any value is safe (see each). Calls are asynchronous
 * on `stream`, return 0, 1 for a rejected argument (nothing launched) or 2 for a HIP error, and set the
 * *_last_error() of the calling thread.
 */

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
 * a page, their sums are added in any order. Refused: max_q * Hq / Hkv of 2^30 and more, and tables of 2^26
 * and more blocks over all requests and kv heads. workspace: kv8_weigh_workspace_bytes() bytes (max_q = 1
 * where cu_q is NULL; may be 0), 4-byte aligned. */
size_t kv8_weigh_workspace_bytes(int T, int B, int Hq, int Hkv, int max_q, int W, int page);
int kv8_weigh(float* weights, const void* q, const long long* q_strides, int dtype, const float* lse,
              int T, int B, int Hq, int Hkv, int D, const void* k_codes, const float* k_scales,
              int pages, int page, const int* table, long long table_stride, int W, const int* lens,
              const int* cu_q, int max_q, float scale, int causal, void* workspace,
              size_t workspace_bytes, hipStream_t stream);

/* Every request with more than keep[b] pages (n = ceil(lens[b] / page) of at most W) loses
 * n - keep[b] of them (fewer, where fewer may go): those of least weight among its pages first ..
 * n - recent - 1, of equal ones the earlier. A page's weight is the sum of weights[page] (fp32
 * [pages, Hkv, page/64]) over heads and blocks in fp64, NaN counting as largest. A table entry
 * outside [0, pages), as kv4_plan_pages leaves where the free list ends, goes before all of them.
 * The row closes up in place (-1 behind the last page that stays), lens_out[b] = lens[b] less the
 * tokens of all that went. The pages that went, in the order of the requests and
 * of their rows, go before free_pages[*used], from where kv4_plan_pages takes pages:
 * into free_pages[*used_out .. *used), *used_out = *used less their number; *lost counts
 * those that had no room (the earlier ones go in). Entries that name no page count in none of the
 * three. first >= 0, recent >= 1: the last page, which
 * may be short, always stays. lens_out, used_out and lost must not overlap each other or anything else that is
 * passed (what one request's work writes, another's may still read). workspace:
 * kv8_evict_workspace_bytes(), 8-byte aligned. */
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
