/* C ABI of the MI355X (gfx950) sparse attention: every block of 128 query rows
 * reads a few blocks of keys, which a score of block means selects. No counterpart
 * in the reference, whose attention reads every key.
 *
 * Calls are asynchronous on `stream`, return 0, 1 for a rejected argument (nothing
 * launched) or 2 for a HIP error, and set sparse_last_error() for the calling
 * thread. Pointers are device pointers, strides in elements {batch, head,
 * sequence}, head dims contiguous, D 64 or 128, key blocks of 64 or 128 rows.
 */
#ifndef GFX906_AMD_SPARSE_H
#define GFX906_AMD_SPARSE_H

#include <stddef.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

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
 * k_means[b][h / (Hq/Hkv)][j] (fp64; NaN counts as largest, equal products by the
 * lower index). Means are packed fp32 [B, Hq, ceil(Sq/128), D] and
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
 * it holds. q, k, v: rows 16-byte aligned (k's and v's
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

#ifdef __cplusplus
}
#endif

#endif
