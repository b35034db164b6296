// Sparse attention for AMD MI355X (gfx950): means of row blocks, the choice of key
// blocks by the product of means, and attention over the chosen blocks. The entry
// points are described in gfx906_amd_sparse.h.
//
// The choice is an output (and decides what is read), so it must not hang on the
// order of a sum: block sums are taken in fp64, where sums of 128 fp16 values are
// exact, and rounded once to fp32; products of two fp32 are exact in fp64 and add
// up there. Scores of different blocks closer than 1e-15 relative are as good as
// never seen; equal ones go by the index.
#include "longctx.h"

#include <algorithm>

#include "gfx906_amd_sparse.h"

namespace {

using namespace gfx906_amd::longctx;

thread_local LastError g_err;

constexpr int kQBlock = SPARSE_Q_BLOCK;

// -- block means ----------------------------------------------------------------------

struct MeansArgs {
    const void* x;
    long long sb, sh, ss;
    float* means;
    int H, S, D, block, nb;
};

// One wave per block of rows and 64 dims.
template <class T>
__global__ void __launch_bounds__(64) means_kernel(const MeansArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int j = blockIdx.x, bh = blockIdx.y, d = blockIdx.z * 64 + threadIdx.x;
    const int b = bh / a.H, h = bh - b * a.H;
    const int r0 = j * a.block, r1 = min(a.S, r0 + a.block);
    const T* x = (const T*)a.x + b * a.sb + h * a.sh + d;
    double sum = 0.0;
    for (int r = r0; r < r1; ++r) sum += (double)(float)x[r * a.ss];
    a.means[((long long)bh * a.nb + j) * a.D + d] = (float)(sum / (r1 - r0));
#endif
}

// -- choice ---------------------------------------------------------------------------

struct SelectArgs {
    const float* qm;
    const float* km;
    double* score;
    int* index;
    int Hq, Hkv, Sq, Skv, D, block, nq, nk, count, causal;
};

// Key blocks a query block may take (the first `seen`), and the first of those that
// it always takes (`own`; seen without causal).
struct Reach {
    int seen, own;
};
__host__ __device__ inline Reach reach(int i, int Sq, int Skv, int block, int nk, int causal) {
    if (!causal) return {nk, nk};
    const long long first = (long long)i * kQBlock + Skv - Sq;
    const long long last = ((long long)i * kQBlock + kQBlock < Sq ? (long long)i * kQBlock + kQBlock
                                                                    : Sq) -
                           1 + Skv - Sq;
    if (last < 0) return {0, 0};
    return {(int)(last / block) + 1, (int)((first < 0 ? 0 : first) / block)};
}

// One workgroup per query block: all scores, then every block counts those ranked
// before it, then the chosen ones are written in order.
__global__ void __launch_bounds__(256) select_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float qs[128];
    __shared__ int base, wave_n[4];
    const int i = blockIdx.x, bh = blockIdx.y, t = threadIdx.x;
    const int b = bh / a.Hq, h = bh - b * a.Hq, kvh = b * a.Hkv + h / (a.Hq / a.Hkv);
    const Reach r = reach(i, a.Sq, a.Skv, a.block, a.nk, a.causal);
    const long long row = (long long)bh * a.nq + i;
    double* score = a.score + row * a.nk;
    int* out = a.index + row * a.count;
    if (t < a.D) qs[t] = a.qm[row * a.D + t];
    if (t == 0) base = 0;
    __syncthreads();
    for (int j = t; j < r.seen; j += 256) {
        const float* k = a.km + ((long long)kvh * a.nk + j) * a.D;
        double s = 0.0;
        for (int d = 0; d < a.D; ++d) s = fma((double)qs[d], (double)k[d], s);
        score[j] = s != s || j >= r.own ? INFINITY : s;
    }
    __syncthreads();
    __threadfence_block();
    for (int j0 = 0; j0 < r.seen; j0 += 256) {
        const int j = j0 + t;
        bool take = false;
        if (j < r.seen) {
            const double s = score[j];
            int before = 0;
            for (int u = 0; u < r.seen; ++u) {
                const bool mine = u >= r.own, me = j >= r.own;
                before += mine != me ? mine : score[u] > s || (score[u] == s && u < j);
            }
            take = before < a.count;
        }
        const unsigned long long m = __ballot(take);
        if ((t & 63) == 0) wave_n[t >> 6] = __popcll(m);
        __syncthreads();
        int at = base + __popcll(m & ((1ull << (t & 63)) - 1));
        for (int w = 0; w < t >> 6; ++w) at += wave_n[w];
        if (take && at < a.count) out[at] = j;
        __syncthreads();
        if (t == 0) base += wave_n[0] + wave_n[1] + wave_n[2] + wave_n[3];
        __syncthreads();
    }
    for (int j = base + t; j < a.count; j += 256) out[j] = -1;
#endif
}

// -- attention ------------------------------------------------------------------------

struct Strides {
    long long b, h, s;
};

struct AttnArgs {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    Strides sq, sk, sv, so;
    const int* index;
    int Hq, Hkv, Sq, Skv, D, block, nq, nk, count, causal;
    float scale;
};

// One wave per query row: 64 keys at a time, a score per lane, then a pair of dims
// per lane.
template <class T>
__global__ void __launch_bounds__(64) attn_rows_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float qs[128], ps[64];
    const int row = blockIdx.x, bh = blockIdx.y, lane = threadIdx.x;
    const int b = bh / a.Hq, h = bh - b * a.Hq, hk = h / (a.Hq / a.Hkv);
    const T* q = (const T*)a.q + b * a.sq.b + h * a.sq.h + row * a.sq.s;
    const T* k = (const T*)a.k + b * a.sk.b + hk * a.sk.h;
    const T* v = (const T*)a.v + b * a.sv.b + hk * a.sv.h;
    T* o = (T*)a.o + b * a.so.b + h * a.so.h + row * a.so.s;
    const int* list = a.index + ((long long)bh * a.nq + row / kQBlock) * a.count;
    for (int d = lane; d < a.D; d += 64) qs[d] = (float)q[d];
    __syncthreads();
    const long long seen = a.causal ? (long long)row + a.Skv - a.Sq + 1 : a.Skv;
    float m = kNoMax, l = 0.f, o0 = 0.f, o1 = 0.f;
    int last = -1;
    for (int e = 0; e < a.count; ++e) {
        const int blk = list[e];
        if (blk <= last || blk >= a.nk) continue;
        last = blk;
        for (int u = 0; u < a.block; u += 64) {
            const long long j0 = (long long)blk * a.block + u, j = j0 + lane;
            const long long end = min(seen, (long long)a.Skv);
            float s = -INFINITY;
            if (j < end) {
                s = 0.f;
                for (int d = 0; d < a.D; ++d) s += qs[d] * (float)k[j * a.sk.s + d];
                s *= a.scale * kLog2e;
            }
            const float mn = fmaxf(m, wave_max(s)), w = exp2f(m - mn), p = exp2f(s - mn);
            l = l * w + wave_sum(p);
            o0 *= w;
            o1 *= w;
            m = mn;
            ps[lane] = p;
            __syncthreads();
            if (2 * lane < a.D)
                for (int i = 0; i < 64 && j0 + i < end; ++i) {
                    o0 += ps[i] * (float)v[(j0 + i) * a.sv.s + 2 * lane];
                    o1 += ps[i] * (float)v[(j0 + i) * a.sv.s + 2 * lane + 1];
                }
            __syncthreads();
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    if (2 * lane < a.D) {
        o[2 * lane] = (T)(o0 * inv);
        o[2 * lane + 1] = (T)(o1 * inv);
    }
#endif
}

// -- host -----------------------------------------------------------------------------

int check_sizes(int B, int H, int S, int D, int block, const char* who) {
    if (B < 0 || H < 0 || S < 0 || S >= (1 << 30) || (long long)B * H > 65535)
        return g_err.fail("%s: negative sizes, a sequence of 2^30 or more, or more than 65535 heads",
                          who);
    if (D != 64 && D != 128) return g_err.fail("%s: head dim must be 64 or 128", who);
    if (block != 64 && block != 128) return g_err.fail("%s: blocks have 64 or 128 rows", who);
    return 0;
}

int blocks_of(int S, int block) { return (S + block - 1) / block; }

int check_strides(const long long* s, const void* p, size_t bytes, int mult, const char* who) {
    for (int i = 0; i < 3; ++i)
        if (s[i] < 0 || s[i] % mult)
            return g_err.fail("%s: strides must be non-negative multiples of %d elements", who, mult);
    if (!aligned(p, bytes)) return g_err.fail("%s: tensors must be %d-byte aligned", who, (int)bytes);
    return 0;
}

}  // namespace

extern "C" const char* sparse_last_error(void) { return g_err.get(); }

extern "C" int sparse_block_means(const void* x, const long long* strides, int dtype, int B, int H,
                                  int S, int D, int block, float* means, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_sizes(B, H, S, D, block, "sparse_block_means")) return 1;
    if (dtype != SPARSE_DTYPE_F16 && dtype != SPARSE_DTYPE_BF16)
        return g_err.fail("sparse_block_means: bad dtype");
    if (B == 0 || H == 0 || S == 0) return 0;
    if (!x || !strides || !means) return g_err.fail("sparse_block_means: null argument");
    if (check_strides(strides, x, 16, 8, "sparse_block_means")) return 1;
    const int nb = blocks_of(S, block);
    const MeansArgs a{x, strides[0], strides[1], strides[2], means, H, S, D, block, nb};
    const dim3 grid(nb, B * H, D / 64);
    if (dtype == SPARSE_DTYPE_F16)
        hipLaunchKernelGGL(means_kernel<f16>, grid, dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL(means_kernel<bf16>, grid, dim3(64), 0, stream, a);
    return g_err.launched("sparse_block_means", hipGetLastError());
}

extern "C" size_t sparse_select_workspace_bytes(int B, int Hq, int Sq, int Skv, int block) {
    if (B <= 0 || Hq <= 0 || Sq <= 0 || Skv <= 0 || block <= 0) return 0;
    return (size_t)B * Hq * blocks_of(Sq, kQBlock) * blocks_of(Skv, block) * sizeof(double);
}

extern "C" int sparse_select(const float* q_means, const float* k_means, int B, int Hq, int Hkv,
                             int Sq, int Skv, int D, int block, int count, int causal, int* index,
                             void* workspace, size_t workspace_bytes, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_sizes(B, Hq, Sq, D, block, "sparse_select") ||
        check_sizes(B, Hkv, Skv, D, block, "sparse_select"))
        return 1;
    if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
        return g_err.fail("sparse_select: query heads must be a multiple of kv heads");
    if (blocks_of(Skv, block) > SPARSE_MAX_BLOCKS)
        return g_err.fail("sparse_select: at most %d key blocks", SPARSE_MAX_BLOCKS);
    if (count < 1 || count > SPARSE_MAX_COUNT)
        return g_err.fail("sparse_select: count must be 1 .. %d", SPARSE_MAX_COUNT);
    if (B == 0 || Hq == 0 || Sq == 0) return 0;
    if (!q_means || !index || (Skv > 0 && !k_means))
        return g_err.fail("sparse_select: null argument");
    // Blocks that hold the positions of a query block: the most over all of them.
    const int own = (std::min(Sq, kQBlock) + block - 2) / block + 1;
    if (causal && count < own)
        return g_err.fail("sparse_select: count must be at least %d, the blocks that hold a query "
                          "block's own positions", own);
    const size_t need = sparse_select_workspace_bytes(B, Hq, Sq, Skv, block);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return g_err.fail("sparse_select: workspace misaligned or smaller than "
                          "sparse_select_workspace_bytes()");
    SelectArgs a{q_means, k_means, (double*)workspace, index, Hq, Hkv, Sq, Skv, D, block,
                 blocks_of(Sq, kQBlock), blocks_of(Skv, block), count, causal};
    hipLaunchKernelGGL(select_kernel, dim3(a.nq, B * Hq), dim3(256), 0, stream, a);
    return g_err.launched("sparse_select", hipGetLastError());
}

extern "C" size_t sparse_attn_workspace_bytes(int B, int Hq, int Sq, int Skv, int D, int block,
                                              int count) {
    (void)B, (void)Hq, (void)Sq, (void)Skv, (void)D, (void)block, (void)count;
    return 0;
}

extern "C" int sparse_attn(const void* q, const void* k, const void* v, void* o,
                           const long long* q_strides, const long long* k_strides,
                           const long long* v_strides, const long long* o_strides, int dtype, int B,
                           int Hq, int Hkv, int Sq, int Skv, int D, float scale, const int* index,
                           int block, int count, int causal, void* workspace,
                           size_t workspace_bytes, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_sizes(B, Hq, Sq, D, block, "sparse_attn") ||
        check_sizes(B, Hkv, Skv, D, block, "sparse_attn"))
        return 1;
    if (dtype != SPARSE_DTYPE_F16 && dtype != SPARSE_DTYPE_BF16)
        return g_err.fail("sparse_attn: bad dtype");
    if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
        return g_err.fail("sparse_attn: query heads must be a multiple of kv heads");
    if (blocks_of(Skv, block) > SPARSE_MAX_BLOCKS)
        return g_err.fail("sparse_attn: at most %d key blocks", SPARSE_MAX_BLOCKS);
    if (count < 1 || count > SPARSE_MAX_COUNT)
        return g_err.fail("sparse_attn: count must be 1 .. %d", SPARSE_MAX_COUNT);
    if (!(scale > -INFINITY && scale < INFINITY))
        return g_err.fail("sparse_attn: scale must be finite");
    if (B == 0 || Hq == 0 || Sq == 0) return 0;
    if (!q || !o || !index || (Skv > 0 && (!k || !v)) || !q_strides || !k_strides || !v_strides ||
        !o_strides)
        return g_err.fail("sparse_attn: null argument");
    if (check_strides(q_strides, q, 16, 8, "sparse_attn") ||
        check_strides(k_strides, k, 16, 8, "sparse_attn") ||
        check_strides(v_strides, v, 16, 8, "sparse_attn") ||
        check_strides(o_strides, o, 8, 4, "sparse_attn"))
        return 1;
    if (k_strides[2] > (1 << 22) || v_strides[2] > (1 << 22))
        return g_err.fail("sparse_attn: k/v sequence stride above 2^22 elements");
    const long long oe[3] = {B, Hq, Sq};
    if (!rows_apart(o_strides, oe, 3, D)) return g_err.fail("sparse_attn: o's rows overlap");
    (void)workspace, (void)workspace_bytes;
    auto st = [](const long long* s) { return Strides{s[0], s[1], s[2]}; };
    const AttnArgs a{q, k, v, o, st(q_strides), st(k_strides), st(v_strides), st(o_strides), index,
                     Hq, Hkv, Sq, Skv, D, block, blocks_of(Sq, kQBlock), blocks_of(Skv, block),
                     count, causal, scale};
    if (dtype == SPARSE_DTYPE_F16)
        hipLaunchKernelGGL(attn_rows_kernel<f16>, dim3(Sq, B * Hq), dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL(attn_rows_kernel<bf16>, dim3(Sq, B * Hq), dim3(64), 0, stream, a);
    return g_err.launched("sparse_attn", hipGetLastError());
}
