// Sparse attention for AMD MI355X (gfx950): means of row blocks, the choice of key
// blocks by the product of means, and attention over the chosen blocks. The entry
// points are described in gfx906_amd_attn.h.
//
// The choice is an output (and decides what is read), so it must be the same by whichever
// kernel it is made. Block sums are taken in fp64, exact for fp16 rows (and for bf16 rows
// unless the values of a dim lie more than 38 octaves apart), by block_sum() alone, and rounded
// once to fp32. Products of two such means are exact in fp64; both kernels that add them up do
// it in one order (kChain): blocks whose scores differ by less than its error, 2^-48 sum |q k|,
// may change places against exact sums, but alike in every call. Equal sums go by the index.
#include "longctx_tile.h"

#include <algorithm>
#include <type_traits>

#include "gfx906_amd_attn.h"

namespace {

using namespace gfx906_amd::longctx;

thread_local LastError g_err;

constexpr int kQBlock = SPARSE_Q_BLOCK;

// -- block means ----------------------------------------------------------------------

struct MeansArgs {
    const void* x;
    long long sb, sh, ss;
    float* means;
    int H, S, block, nb;
    long long blocks;  // of all heads
};

#if defined(__HIP_DEVICE_COMPILE__)
// Column sums of `rows` rows, V dims a lane, N loads in flight: D/8 lanes beside each other
// take a row, a wave 512/D rows at a time, and the lanes that hold the same dims add up at the
// end (all of them have the sum). A dim's sum is added up in the same order whatever V and N.
// x: the lane's dims of the first row.
template <int D, int V, int N, class T>
__device__ __forceinline__ void block_sum(const T* x, long long stride, int rows, double (&sum)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    constexpr int LPR = D / 8, RPL = 64 / LPR;
    const int r = (threadIdx.x & 63) / LPR;
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.0;
    for (int t = 0; t < rows; t += N * RPL) {
        vec v[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int row = t + n * RPL + r;
            v[n] = vec{};
            if (row < rows) v[n] = *reinterpret_cast<const vec*>(x + row * stride);
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += (double)(float)v[n][e];
    }
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += __shfl_xor(sum[e], o);
}
#endif

// One wave per block of rows, 16 bytes a lane: a load takes 4 (D = 128) or 8 (D = 64) whole rows.
// Bound by the bytes of x: 16 heads of 16384, D = 128, 17 us
// (4.0 TB/s), and 13 where the last-level cache holds rows.
template <int D, class T>
__global__ void __launch_bounds__(256) means_kernel(const MeansArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LPR = D / 8;
    const int lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.blocks) return;
    const int j = (int)(id % a.nb), bh = (int)(id / a.nb), b = bh / a.H, h = bh - b * a.H;
    const int r0 = j * a.block, rows = min(a.block, a.S - r0);
    const int c = lane % LPR, r = lane / LPR;
    double sum[8];
    block_sum<D, 8, 16>((const T*)a.x + b * a.sb + h * a.sh + r0 * a.ss + c * 8, a.ss, rows, sum);
    if (r == 0) {
        float* m = a.means + id * D + c * 8;
        f32x4 lo, hi;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = (float)(sum[e] / rows);
            hi[e] = (float)(sum[e + 4] / rows);
        }
        *reinterpret_cast<f32x4*>(m) = lo;
        *reinterpret_cast<f32x4*>(m + 4) = hi;
    }
#endif
}

// -- choice ---------------------------------------------------------------------------

struct SelectArgs {
    const float* qm;
    const float* km;
    double* score;
    int* index;
    int Hq, Hkv, Sq, Skv, D, block, nq, nk, count, causal;
    long long rows;  // query blocks of all heads
    const void* q;   // choose_one_kernel: the query rows, and their strides
    long long qb, qh, qs;
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

// Scores of a kv head's query rows (row r: query block r / G of query head r % G of the
// head's group) and key blocks, on the fp64 matrix pipe: a wave keeps 16 rows and goes
// through tiles of 16 key blocks. In step s of a tile lane group g supplies dim
// g D/4 + s, so that a lane reads D/4 consecutive floats of its row.
//
// Order of a score's sum (here and in choose_one_kernel): v_mfma_f64_16x16x4 adds its four
// products to the accumulator one after another, each rounded once, as four fmas do. kChain
// steps make a chain of 4 kChain dims that starts at 0, and chains are added pairwise, neighbours
// first.
//
// 8 heads, 1024 x 1024 blocks, D = 64: 33 us, for 67 MB of scores; 16 heads, 128 x 256, 8.4.
//
// grid: row tiles, kv heads of all batches, shares of the key tiles; 4 waves.
constexpr int kChain = 4;
template <int D>
__global__ void __launch_bounds__(256) score_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int N = D / 4;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int G = a.Hq / a.Hkv, rows = G * a.nq, r0 = blockIdx.x * 16;
    const int b = blockIdx.y / a.Hkv, hk = blockIdx.y - b * a.Hkv;
    const int tiles = (a.nk + 15) / 16, step = 4 * gridDim.z;
    // Row of the score matrix (of all heads) that tile row r stands for.
    auto row_of = [&](int r) {
        const int qb = r / G;
        return ((long long)b * a.Hq + hk * G + (r - qb * G)) * a.nq + qb;
    };
    double q[N];
    {
        const int r = min(r0 + i, rows - 1);
        const float* p = a.qm + row_of(r) * D + g * N;
#pragma unroll
        for (int s = 0; s < N; s += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(p + s);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[s + e] = x[e];
        }
    }
    const float* km = a.km + (long long)blockIdx.y * a.nk * D + g * N;
    for (int t = blockIdx.z * 4 + (threadIdx.x >> 6); t < tiles; t += step) {
        const float* p = km + (long long)min(16 * t + i, a.nk - 1) * D;
        f32x4 k[N / 4];
#pragma unroll
        for (int s = 0; s < N / 4; ++s) k[s] = *reinterpret_cast<const f32x4*>(p + 4 * s);
        f64x4 sum[N / kChain];
#pragma unroll
        for (int x = 0; x < N / kChain; ++x) {
            f64x4 c = {};
#pragma unroll
            for (int s = x * kChain; s < (x + 1) * kChain; ++s)
                c = __builtin_amdgcn_mfma_f64_16x16x4f64(q[s], (double)k[s / 4][s % 4], c, 0, 0, 0);
            sum[x] = c;
        }
#pragma unroll
        for (int o = 1; o < N / kChain; o *= 2)
#pragma unroll
            for (int x = 0; x < N / kChain; x += 2 * o) sum[x] += sum[x + o];
        // (accumulator element e: row 4 e + l/16, column l%16)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = r0 + 4 * e + g, j = 16 * t + i;
            if (r < rows && j < a.nk) a.score[row_of(r) * a.nk + j] = sum[0][e];
        }
    }
#endif
}

// The choice of one row by WAVES waves, K scores a lane (wave w: the w-th run of 64 K
// key blocks). Scores become 64-bit integers of the same order (0: not to be taken;
// all ones: always), and the count-th largest is found bit by bit from the top, until
// exactly `count` lie at or above the bits so far, or their last bit is set: then
// scores equal to it fill up in the order of their index. The upper 32 bits go first, by
// themselves; the lower ones matter only among scores whose upper bits are the bound's.
// Everything stays in registers; a step is a compare and a population count per 64 scores
// (and, with several waves, an exchange through LDS). 8192 rows of 1024 scores: 36 us; 2048 of
// 256: 6.6.
#if defined(__HIP_DEVICE_COMPILE__)
template <int WAVES, int K, class Score>
__device__ __forceinline__ void choose(const SelectArgs& a, const Reach& r, Score score, int* out,
                                       int (*part)[WAVES]) {
    typedef unsigned long long u64;
    const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
    const int base = wave * 64 * K + lane;
    unsigned hi[K], lo[K];
#pragma unroll
    for (int n = 0; n < K; ++n) {
        const int j = base + 64 * n;
        u64 key = 0;
        if (j < r.seen) {
            const double s = score(j) + 0.0;  // -0 becomes +0
            const u64 bits = (u64)__double_as_longlong(s != s ? INFINITY : s);
            key = j >= r.own ? ~0ull : bits >> 63 ? ~bits : bits | 1ull << 63;
        }
        hi[n] = (unsigned)(key >> 32);
        lo[n] = (unsigned)key;
    }
    int turn = 0;
    auto popc = [](u64 x) { return (int)__popcll(x); };  // (unsigned, else)
    // Sum over the waves of a wave-uniform count; `before`: that of the waves before.
    auto total = [&](int mine, int* before) {
        if (WAVES == 1) {
            if (before) *before = 0;
            return mine;
        }
        if (lane == 0) part[turn][wave] = mine;
        __syncthreads();
        int sum = 0, pre = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int x = part[turn][w];
            sum += x;
            pre += w < wave ? x : 0;
        }
        turn ^= 1;
        if (before) *before = pre;
        return sum;
    };
    // (every key that may be taken is at least 2^51: its upper half is not 0)
    auto upper = [&](unsigned x) {
        int n = 0;
#pragma unroll
        for (int m = 0; m < K; ++m) n += popc(__ballot(hi[m] >= x));
        return total(n, nullptr);
    };
    unsigned bar_hi = 0, bar_lo = 0;  // the bound: all above it, and `ties` of those equal to it
    auto lower = [&](unsigned x) {
        int n = 0;
#pragma unroll
        for (int m = 0; m < K; ++m) n += popc(__ballot(hi[m] == bar_hi && lo[m] >= x));
        return total(n, nullptr);
    };
    int ties = 0;
    if (upper(1) > a.count) {
        bool done = false;
        for (int bit = 31; bit >= 0 && !done; --bit) {
            const unsigned x = bar_hi | 1u << bit;
            const int n = upper(x);
            if (n >= a.count) bar_hi = x;
            done = n == a.count;
        }
        if (done) {  // all whose upper half is at least bar_hi
            bar_hi -= 1;
            bar_lo = ~0u;
        } else {
            const int need = a.count - (bar_hi == ~0u ? 0 : upper(bar_hi + 1));
            for (int bit = 31; bit >= 0 && !done; --bit) {
                const unsigned x = bar_lo | 1u << bit;
                const int n = lower(x);
                if (n >= need) bar_lo = x;
                done = n == need;
            }
            if (done)
                bar_lo -= 1;
            else
                ties = need - (bar_lo == ~0u ? 0 : lower(bar_lo + 1));
        }
    }
    auto over = [&](int n) { return hi[n] > bar_hi || (hi[n] == bar_hi && lo[n] > bar_lo); };
    auto even = [&](int n) { return ties > 0 && hi[n] == bar_hi && lo[n] == bar_lo; };
    int above = 0, equal = 0;
#pragma unroll
    for (int n = 0; n < K; ++n) {
        above += popc(__ballot(over(n)));
        equal += popc(__ballot(even(n)));
    }
    int ties_before;
    total(equal, &ties_before);
    int ties_left = max(0, ties - ties_before);
    int at;
    const int all = total(above + min(equal, ties_left), &at);
    const u64 below = (1ull << lane) - 1;
#pragma unroll
    for (int n = 0; n < K; ++n) {
        const u64 eq = __ballot(even(n));
        const bool take = over(n) || (even(n) && popc(eq & below) < ties_left);
        const u64 mk = __ballot(take);
        if (take) out[at + popc(mk & below)] = base + 64 * n;
        at += popc(mk);
        ties_left = max(0, ties_left - popc(eq));
    }
    for (int e = all + (WAVES == 1 ? lane : (int)threadIdx.x); e < a.count; e += 64 * WAVES)
        out[e] = -1;
}
#endif

template <int WAVES, int K>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) select_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ int part[2][WAVES];
    const long long row = WAVES == 1 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= a.rows) return;  // (a whole wave; with several, never)
    const Reach r = reach((int)(row % a.nq), a.Sq, a.Skv, a.block, a.nk, a.causal);
    const double* score = a.score + row * a.nk;
    choose<WAVES, K>(a, r, [&](int j) { return score[j]; }, a.index + row * a.count, part);
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// Adds up N = 4 or 8 neighbouring lanes, pairwise (DPP moves within rows of 16: a swap of
// neighbours, of pairs, and a mirror of what is then equal in halves).
template <int CTRL>
__device__ __forceinline__ double dpp_add(double x) {
    const long long b = __double_as_longlong(x);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, true);
    return x + __longlong_as_double((long long)((unsigned long long)(unsigned)hi << 32 | (unsigned)lo));
}
template <int N>
__device__ __forceinline__ double lanes_sum(double x) {
    x = dpp_add<0xB1>(x);   // quad_perm [1, 0, 3, 2]
    x = dpp_add<0x4E>(x);   // quad_perm [2, 3, 0, 1]
    if constexpr (N == 8) x = dpp_add<0x141>(x);  // row_half_mirror
    return x;
}
#endif

// The choice straight from the query rows: mean, scores and choice of a query block in one
// workgroup, of up to 4096 key blocks, where the launches of three kernels outweigh that every
// block reads all key means (one_kernel below). Four waves take the mean; then
// D/16 lanes take a row of the key means, a chain of score_kernel's order each. 64 heads of
// one query, 512 blocks: 11 to 13 us, and 19 in three kernels.
template <int D, class T>
__global__ void __launch_bounds__(512) choose_one_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    // dims of a lane group in score_kernel; lanes a row, rows at a time
    constexpr int N = D / 4, LPR = N / kChain, ROWS = 512 / LPR;
    static_assert(kChain == 4, "a chain is a 16-byte load of every group");
    __shared__ double score[4096];
    __shared__ __attribute__((aligned(16))) float qs[D];
    __shared__ int part[2][8];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int bh = blockIdx.x / a.nq, i = blockIdx.x - bh * a.nq, b = bh / a.Hq, h = bh - b * a.Hq;
    const int kvh = b * a.Hkv + h / (a.Hq / a.Hkv);
    if (wave < 4) {  // D/4 dims a wave
        const int rows = min(kQBlock, a.Sq - i * kQBlock), d = 2 * (wave * (D / 8) + tid % (D / 8));
        double sum[2];
        block_sum<D, 2, kQBlock * D / 512>(
            (const T*)a.q + b * a.qb + h * a.qh + (long long)i * kQBlock * a.qs + d, a.qs, rows, sum);
        if (tid % 64 < D / 8) *reinterpret_cast<f32x2*>(qs + d) =
            f32x2{(float)(sum[0] / rows), (float)(sum[1] / rows)};
    }
    __syncthreads();
    const int c = tid % LPR, r0 = tid / LPR;
    double qd[4][4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) qd[g][e] = qs[g * N + c * 4 + e];
    const Reach r = reach(i, a.Sq, a.Skv, a.block, a.nk, a.causal);
    const float* km = a.km + (long long)kvh * a.nk * D + c * 4;
    // U rows a lane at a time: 512 in all, or 128 of a short sequence (512 queries of 32 heads, 64
    // blocks, D = 128: 8.8 us a call, and 10.6 with 512).
    auto rows_by = [&](auto per) __attribute__((always_inline)) {
        constexpr int U = decltype(per)::value;
        for (int j0 = r0; j0 < r.seen; j0 += U * ROWS) {
            f32x4 x[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float* p = km + (long long)min(j0 + u * ROWS, r.seen - 1) * D;
#pragma unroll
                for (int g = 0; g < 4; ++g) x[u][g] = *reinterpret_cast<const f32x4*>(p + g * N);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                double s = 0.0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int g = 0; g < 4; ++g) s = fma(qd[g][e], (double)x[u][g][e], s);
                s = lanes_sum<LPR>(s);
                const int j = j0 + u * ROWS;
                if (c == 0 && j < r.seen) score[j] = s;
            }
        }
    };
    if (r.seen <= 128)
        rows_by(std::integral_constant<int, 128 / ROWS>{});
    else
        rows_by(std::integral_constant<int, 512 / ROWS>{});
    __syncthreads();
    int* out = a.index + (long long)blockIdx.x * a.count;
    auto at = [&](int j) { return score[j]; };
    if (a.nk <= 512) {  // one wave: no exchange between waves in a step
        if (wave == 0) choose<1, 8>(a, r, at, out, (int(*)[1])part);
    } else {
        choose<8, 8>(a, r, at, out, part);
    }
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
    float c, qsign;  // log2_scale(); a negative scale negates q
    // Lists are split in nsplit ranges of a query block's entries; a range writes its
    // unnormalised O (fp32) and (m, l) to the workspace, at row range * rows + row of
    // all heads' rows, and combine_kernel merges them.
    int nsplit;
    long long rows;
    float* ws_o;
    float* ws_ml;
};

#if defined(__HIP_DEVICE_COMPILE__)
// Where the results of one row go: the output, or the workspace of a split range.
template <class T>
__device__ __forceinline__ void store_pair(const AttnArgs& a, T* orow, long long wrow, int d,
                                           float x, float y, float inv, bool split) {
    if (split) {
        *reinterpret_cast<f32x2*>(a.ws_o + wrow * a.D + d) = f32x2{x, y};
    } else {
        *reinterpret_cast<typename Elem<T>::x2*>(orow + d) = Elem<T>::cvt2(x * inv, y * inv);
    }
}

// One row over the blocks whose first keys are list[e0..e1), by one wave: 64 keys at a time, a score per
// lane, then a pair of dims per lane. Keys the row does not see are not touched at
// all, so that what they hold cannot reach it.
template <int D, class T>
__device__ __attribute__((noinline)) void attend_row(const AttnArgs& a, const T* q, const T* k,
                                                     const T* v, T* orow, long long wrow,
                                                     const int* list, int e0, int e1,
                                                     int seen) {
    const int lane = threadIdx.x & 63;
    float m = kNoMax, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int e = e0; e < e1; ++e)
        for (int u = 0; u < a.block; u += 64) {
            const int j0 = list[e] + u, j = j0 + lane;
            float s = -INFINITY;
            if (j < seen) {
                s = 0.f;
                for (int d = 0; d < D; ++d) s = fmaf((float)q[d], (float)k[j * a.sk.s + d], s);
                s *= a.c * a.qsign;
            }
            const float mn = max2(m, wave_max(s)), w = exp2f(m - mn), p = exp2f(s - mn);
            l = l * w + wave_sum(p);
            o0 *= w;
            o1 *= w;
            m = mn;
            for (int i = 0; i < 64 && j0 + i < seen; ++i) {
                const float pi = __shfl(p, i);
                if (2 * lane < D) {
                    o0 = fmaf(pi, (float)v[(j0 + i) * a.sv.s + 2 * lane], o0);
                    o1 = fmaf(pi, (float)v[(j0 + i) * a.sv.s + 2 * lane + 1], o1);
                }
            }
        }
    if (2 * lane < D)
        store_pair(a, orow, wrow, 2 * lane, o0, o1, l != 0.f ? 1.f / l : 0.f, a.nsplit > 1);
    if (a.nsplit > 1 && lane == 0) *reinterpret_cast<f32x2*>(a.ws_ml + 2 * wrow) = f32x2{m, l};
}

// Workgroup w's place in a grid of n: the dispatcher deals workgroups out to the 8
// XCDs in turn; where 8 divides n, consecutive units go to one XCD, whose L2 then
// streams the keys of as few heads as possible.
__device__ __forceinline__ int xcd_order(int w, int n) {
    return (n & 7) == 0 ? (w & 7) * (n >> 3) + (w >> 3) : w;
}
#endif

// Attention of one query block (128 rows, 32 a wave) over its listed key blocks.
//
// The list is read first and the first keys of its valid entries gathered in LDS. Then the
// waves walk the listed keys in tiles of 32, software-pipelined as attn_fwd_pipe: the step
// of tile j issues the PV products of tile j-1 and the QK products of tile j+1 around
// the softmax of tile j. K and V tiles come by loads to LDS into rings of four, K three
// and V two steps ahead, whose waits are counted: one barrier a step. Tiles of 32 (16 KB of
// K and V at D = 128) instead of attn_fwd_pipe's 64 let two workgroups of four waves share
// a CU's LDS, for lists of 128 rows instead of 256.
//
// Steps go four to a round, a whole number of blocks, so that which entry of the list a
// tile belongs to is known when the kernel is compiled; entries are read a round ahead.
// Tiles past the list load zeros (their offset is past the descriptor's range) and are
// masked, so that loads and waits stay static. One descriptor serves a head's K (or V) of
// less than 2^31 bytes; with FAR it is made anew for every tile.
//
// A tile with masked keys is checked for infinite and NaN values of V (which a weight of 0
// would not keep out of the sums); where there are any the wave does its rows again by
// attend_row.
//
// 16 heads of 16384 tokens, 32 blocks of 64, D = 128: 259 us (1060 TFLOP/s, where a library
// product of 8192 reaches 1130; 293 in the first calls of a process): the matrix pipe is busy for
// 56 % of the clocks, the vector unit for 46, LDS for 27, at 1.98 GHz. 8 heads of 131072, 64 blocks
// of 128, D = 64: 2.25 ms (977): 60, 72 and 27 % at 1.71 GHz, with twice the exponentials a product.
// So the matrix and the vector unit's work, which the two waves of a SIMD overlap in part, and the
// clock that the card keeps under it (2.4 GHz at most) bound it, not LDS. Single queries are bound
// by the blocks' bytes (138 MB in 21 us).
template <int D, class T, int TPB, bool FAR>
__global__ void __launch_bounds__(256, 2) attn_tile_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using W = Tile<D, T>;
    using x8 = typename W::x8;
    constexpr int NU = W::NU, RB = W::RB, BYTES = W::BYTES;
    constexpr int LPT = BYTES / 1024 / 4;  // loads a wave and tile
    constexpr int kWait = 0x0F70 | ((4 * LPT) & 15) | (((4 * LPT) >> 4) << 14);
    constexpr int EPR = 4 / TPB;           // entries a round
    constexpr int kNoKey = 0x7fffff00;     // the key of tiles past the list
    __shared__ __attribute__((aligned(1024))) char k0[BYTES];
    __shared__ __attribute__((aligned(1024))) char k1[BYTES];
    __shared__ __attribute__((aligned(1024))) char k2[BYTES];
    __shared__ __attribute__((aligned(1024))) char k3[BYTES];
    __shared__ __attribute__((aligned(1024))) char v0[BYTES];
    __shared__ __attribute__((aligned(1024))) char v1[BYTES];
    __shared__ __attribute__((aligned(1024))) char v2[BYTES];
    __shared__ __attribute__((aligned(1024))) char v3[BYTES];
    __shared__ int list[SPARSE_MAX_COUNT];
    __shared__ int n_list;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    // (uniform, and kept in scalar registers: divisions run on the vector unit, and
    // descriptors made from vector registers would be read in loops)
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int unit = xcd_order(blockIdx.x, gridDim.x);
    const int qi = uni(unit / a.nsplit), range = unit - qi * a.nsplit;
    const int bh = uni(qi / a.nq), qb = qi - bh * a.nq;
    const int b = uni(bh / a.Hq), h = bh - b * a.Hq, hk = uni(h / uni(a.Hq / a.Hkv));
    const T* Q = (const T*)a.q + b * a.sq.b + h * a.sq.h;
    const T* K = (const T*)a.k + b * a.sk.b + hk * a.sk.h;
    const T* V = (const T*)a.v + b * a.sv.b + hk * a.sv.h;
    const int row0 = qb * kQBlock + wave * 32;  // this lane's rows: row0 + 16 nb + i
    const bool active = row0 < a.Sq;            // (wave-uniform)

    W w;
    w.init(lane);
    const unsigned neg = a.qsign < 0.f ? 0x80008000u : 0u;
    int lim[2];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
        const int row = row0 + 16 * nb + i;
        lim[nb] = a.causal ? min(a.Skv, row + a.Skv - a.Sq + 1) : a.Skv;
#pragma unroll
        for (int s = 0; s < W::NQ; ++s) {
            u32x4 x = {};
            if (row < a.Sq)
                x = *reinterpret_cast<const u32x4*>(Q + row * a.sq.s + 32 * s + 8 * g);
            w.qf[nb][s] = __builtin_bit_cast(x8, x ^ neg);
        }
    }
    // Keys below this one are seen by every row of the wave.
    const int all_see = a.causal ? min(a.Skv, row0 + a.Skv - a.Sq + 1) : a.Skv;

    // The valid entries of the list: above every valid one before them, in range, and
    // (causal) not behind every row of the query block.
    if (wave == 0) {
        const int* src = a.index + ((long long)bh * a.nq + qb) * a.count;
        const int reach = a.causal
                              ? min(a.nk, (int)((min(a.Sq, (qb + 1) * kQBlock) - 1LL + a.Skv - a.Sq +
                                                 a.block) / a.block))
                              : a.nk;
        int last = -1, n = 0;
        for (int e0 = 0; e0 < a.count; e0 += 64) {
            const int e = e0 + lane;
            const int x = e < a.count ? src[e] : -1;
            const bool in = x >= 0 && x < a.nk;
            int top = in ? x : -1;  // running max, inclusive
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(top, o);
                if (lane >= o) top = max(top, y);
            }
            int before = __shfl_up(top, 1);
            before = max(last, lane ? before : -1);
            const bool take = in && x > before && x < reach;
            const unsigned long long mk = __ballot(take);
            if (take) list[n + (int)__popcll(mk & ((1ull << lane) - 1))] = x * (TPB * 32);
            n += (int)__popcll(mk);
            last = max(last, __shfl(top, 63));
        }
        if (lane == 0) n_list = n;
    }
    for (int z = tid; z < BYTES / 16; z += 256) *reinterpret_cast<u32x4*>(v3 + 16 * z) = u32x4{};
    __syncthreads();
    const int n_all = uni(n_list);
    // (at most 2048 entries and 512 ranges)
    const int e0 = uni(n_all * range / a.nsplit), e1 = uni(n_all * (range + 1) / a.nsplit);
    const int ntiles = (e1 - e0) * TPB;

    const unsigned kss = (unsigned)(a.sk.s * 2), vss = (unsigned)(a.sv.s * 2);
    unsigned koff[LPT], voff[LPT];
#pragma unroll
    for (int n = 0; n < LPT; ++n) {
        const int u = (wave + 4 * n) * 64 + lane, r = u / NU, s = u % NU;
        koff[n] = r * kss + (s ^ kswz<NU>(r)) * 16;
        voff[n] = r * vss + (s ^ vswz<NU>(r)) * 16;
    }
    auto span = [&](int rows, unsigned ss) {  // bytes of the first rows
        return rows > 0 ? (int)((rows - 1) * ss + 2 * D) : 0;
    };
    const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)K, 0, FAR ? 0 : uni(span(a.Skv, kss)), 0x00020000);
    const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)V, 0, FAR ? 0 : uni(span(a.Skv, vss)), 0x00020000);
    // First key of a list entry, and the offsets of its rows in K and V.
    struct Entry {
        int key;
        unsigned k, v;
    };
    auto entry = [&](int e, int key) __attribute__((always_inline)) {
        Entry x;
        x.key = e < e1 ? uni(key) : kNoKey;
        x.k = e < e1 ? x.key * kss : kOutOfRange;
        x.v = e < e1 ? x.key * vss : kOutOfRange;
        return x;
    };
    auto listed = [&](int e) { return list[min(e, SPARSE_MAX_COUNT - 1)]; };
    // Loads a tile of K or V: tile `sub` of entry x.
    auto issue = [&](auto is_v, const Entry& x, int sub, char* dst) __attribute__((always_inline)) {
        constexpr bool kV = decltype(is_v)::value;
        const unsigned ss = kV ? vss : kss;
        __amdgpu_buffer_rsrc_t r = kV ? vrs : krs;
        unsigned at = (kV ? x.v : x.k) + 32 * sub * ss;
        if constexpr (FAR) {
            const int key = x.key + 32 * sub;
            const int rows = min(a.Skv - key, 32);
            r = __builtin_amdgcn_make_buffer_rsrc(
                (void*)((kV ? V : K) + (rows > 0 ? key : 0) * (kV ? a.sv.s : a.sk.s)), 0,
                uni(span(rows, ss)), 0x00020000);
            at = 0;
        }
#pragma unroll
        for (int n = 0; n < LPT; ++n)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (GFX906_LDS void*)(dst + (wave + 4 * n) * 1024), 16, (kV ? voff : koff)[n] + at, 0,
                0, 0);
    };
    using IsK = std::false_type;
    using IsV = std::true_type;

    bool redo = false;
    if (ntiles > 0) {
        f32x4 Sa[2][2], Sb[2][2];
        x8 Pa[2], Pb[2];
        Pb[0] = x8{};
        Pb[1] = x8{};
        // Entries of tiles j .. j+8, j the round's first tile.
        constexpr int NE = 8 / TPB + 1;
        Entry q[NE];
#pragma unroll
        for (int n = 0; n < NE; ++n) q[n] = entry(e0 + n, listed(e0 + n));
        int ahead[EPR], enext = e0 + NE;  // entries of the next round, read and not yet taken
#pragma unroll
        for (int n = 0; n < EPR; ++n) ahead[n] = listed(enext + n);
        bool hidden = false;  // tile j-1 had masked keys
        issue(IsK{}, q[0], 0, k0);
        issue(IsK{}, q[1 / TPB], 1 % TPB, k1);
        issue(IsK{}, q[2 / TPB], 2 % TPB, k2);
        issue(IsV{}, q[0], 0, v0);
        issue(IsK{}, q[3 / TPB], 3 % TPB, k3);
        issue(IsV{}, q[1 / TPB], 1 % TPB, v1);
        __builtin_amdgcn_s_waitcnt(kWait);
        lds_barrier();
        if (active) w.qk(k0, Sa);
        lds_barrier();
        issue(IsK{}, q[4 / TPB], 4 % TPB, k0);
        issue(IsV{}, q[2 / TPB], 2 % TPB, v2);

        // Tile n of the round: V of the tile before in vp, K of the next in kn; K of the
        // fifth and V of the third after it go where those were.
        auto step = [&](auto nth, const char* vp, const char* kn, char* kfree, char* vfree,
                        f32x4 (&S)[2][2], f32x4 (&Sn)[2][2], const x8 (&Pp)[2], x8 (&P)[2])
            __attribute__((always_inline)) {
            constexpr int n = decltype(nth)::value;
            if (active) {
                if (__builtin_expect(hidden, 0)) redo |= not_finite<D, T>(vp, lane);
                const int key = q[n / TPB].key + 32 * (n % TPB);
                hidden = key + 32 > all_see;
                if (__builtin_expect(hidden, 0)) w.mask(S, key, lim, g);
                w.turn(vp, Pp, kn, Sn, S, P, a.c);
            }
            __builtin_amdgcn_s_waitcnt(kWait);
            lds_barrier();
            issue(IsK{}, q[(n + 5) / TPB], (n + 5) % TPB, kfree);
            issue(IsV{}, q[(n + 3) / TPB], (n + 3) % TPB, vfree);
        };
        using N0 = std::integral_constant<int, 0>;
        using N1 = std::integral_constant<int, 1>;
        using N2 = std::integral_constant<int, 2>;
        using N3 = std::integral_constant<int, 3>;
        for (int j = 0; j < ntiles; j += 4) {
            step(N0{}, v3, k1, k1, v3, Sa, Sb, Pb, Pa);
            step(N1{}, v0, k2, k2, v0, Sb, Sa, Pa, Pb);
            step(N2{}, v1, k3, k3, v1, Sa, Sb, Pb, Pa);
            step(N3{}, v2, k0, k0, v2, Sb, Sa, Pa, Pb);
#pragma unroll
            for (int n = 0; n < NE; ++n)
                q[n] = n + EPR < NE ? q[n + EPR] : entry(enext + n + EPR - NE, ahead[n + EPR - NE]);
            enext += EPR;
#pragma unroll
            for (int n = 0; n < EPR; ++n) ahead[n] = listed(enext + n);
        }
        if (active) {
            if (hidden) redo |= not_finite<D, T>(v3, lane);
            w.pv(v3, Pb);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // loads past the end, before LDS is released
    }
    if (!active) return;

    T* O = (T*)a.o + b * a.so.b + h * a.so.h;
    const long long wbase = range * a.rows + (long long)bh * a.Sq;
    if (__builtin_expect(redo, 0)) {
        // The arguments where they lie (a reference to `a` would put it in memory).
        const AttnArgs& ka = *(const AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
        for (int r = row0; r < min(row0 + 32, a.Sq); ++r)
            attend_row<D, T>(ka, Q + r * a.sq.s, K, V, O + r * a.so.s, wbase + r, list, e0, e1,
                             a.causal ? min(a.Skv, r + a.Skv - a.Sq + 1) : a.Skv);
        return;
    }
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
        const int row = row0 + 16 * nb + i;
        const float l = quad_sum(w.lacc[nb][0]);
        if (row >= a.Sq) continue;
        if (a.nsplit > 1) {
            float* wo = a.ws_o + (wbase + row) * D;
#pragma unroll
            for (int ob = 0; ob < W::NO; ++ob)
                *reinterpret_cast<f32x4*>(wo + 16 * ob + 4 * g) = w.oacc[ob][nb];
            if (g == 0) *reinterpret_cast<f32x2*>(a.ws_ml + 2 * (wbase + row)) = f32x2{w.m[nb], l};
            continue;
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;
        T* op = O + row * a.so.s;
#pragma unroll
        for (int ob = 0; ob < W::NO; ++ob) {
            const f32x4 x = w.oacc[ob][nb] * inv;
            const auto lo = Elem<T>::cvt2(x[0], x[1]), hi = Elem<T>::cvt2(x[2], x[3]);
            *reinterpret_cast<u32x2*>(op + 16 * ob + 4 * g) =
                u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
        }
    }
#endif
}

// Merges the ranges of a row, four dims a lane.
template <class T>
__global__ void __launch_bounds__(256) combine_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int dq = a.D / 4;
    const long long row = id / dq;
    const int d = (int)(id - row * dq) * 4;
    if (row >= a.rows) return;
    // (eight ranges' loads at a time: one after another they took 6 us for 8 ranges)
    constexpr int U = 8;
    float m = kNoMax, l = 0.f;
    f32x4 acc = {};
    for (int s = 0; s < a.nsplit; s += U) {
        f32x2 ml[U];
        f32x4 p[U];
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const long long r = min(s + n, a.nsplit - 1) * a.rows + row;
            ml[n] = *reinterpret_cast<const f32x2*>(a.ws_ml + 2 * r);
            p[n] = *reinterpret_cast<const f32x4*>(a.ws_o + r * a.D + d);
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            if (s + n >= a.nsplit) continue;
            const float mn = max2(m, ml[n][0]);
            const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(ml[n][0] - mn);
            acc = acc * f + p[n] * e;
            l = l * f + ml[n][1] * e;
            m = mn;
        }
    }
    acc *= l != 0.f ? 1.f / l : 0.f;
    const int bh = (int)(row / a.Sq), r = (int)(row - (long long)bh * a.Sq), b = bh / a.Hq;
    T* o = (T*)a.o + b * a.so.b + (bh - b * a.Hq) * a.so.h + r * a.so.s + d;
    const auto lo = Elem<T>::cvt2(acc[0], acc[1]), hi = Elem<T>::cvt2(acc[2], acc[3]);
    *reinterpret_cast<u32x2*>(o) =
        u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
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

// Ranges the lists are split in: enough for two workgroups a CU, of 8 tiles or more (a tile takes
// about 0.65 us, the merge 5).
int split_count(int B, int Hq, int Sq, int Skv, int block, int count) {
    const long long units = (long long)B * Hq * blocks_of(Sq, kQBlock);
    const int entries = std::min(count, blocks_of(Skv, block));
    if (units >= 256 || entries <= 1) return 1;
    const int most = std::max(1, entries * (block / 32) / 8);
    return (int)std::min<long long>(most, 512 / units);
}

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
    const long long blocks = (long long)B * H * nb;
    const MeansArgs a{x, strides[0], strides[1], strides[2], means, H, S, block, nb, blocks};
    if (!launchable((blocks + 3) / 4, 256)) return g_err.fail("sparse_block_means: too many blocks");
    const dim3 grid((unsigned)((blocks + 3) / 4));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a); };
    if (dtype == SPARSE_DTYPE_F16)
        D == 64 ? go(means_kernel<64, f16>) : go(means_kernel<128, f16>);
    else
        D == 64 ? go(means_kernel<64, bf16>) : go(means_kernel<128, bf16>);
    return g_err.launched("sparse_block_means", hipGetLastError());
}

extern "C" size_t sparse_select_workspace_bytes(int B, int Hq, int Sq, int Skv, int block) {
    if (B <= 0 || Hq <= 0 || Sq <= 0 || Skv <= 0 || block <= 0) return 0;
    return (size_t)B * Hq * blocks_of(Sq, kQBlock) * blocks_of(Skv, block) * sizeof(double);
}

namespace {

// Checks that sparse_select and sparse_choose share; `who` names the caller.
int check_choice(const void* q, const float* k_means, int B, int Hq, int Hkv, int Sq, int Skv, int D,
                 int block, int count, int causal, const int* index, const char* who) {
    if (check_sizes(B, Hq, Sq, D, block, who) || check_sizes(B, Hkv, Skv, D, block, who)) return 1;
    if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
        return g_err.fail("%s: query heads must be a multiple of kv heads", who);
    if (blocks_of(Skv, block) > SPARSE_MAX_BLOCKS)
        return g_err.fail("%s: at most %d key blocks", who, SPARSE_MAX_BLOCKS);
    if (count < 1 || count > SPARSE_MAX_COUNT)
        return g_err.fail("%s: count must be 1 .. %d", who, SPARSE_MAX_COUNT);
    if (B == 0 || Hq == 0 || Sq == 0) return 0;
    if (!q || !index || (Skv > 0 && !k_means)) return g_err.fail("%s: null argument", who);
    if (!aligned(k_means, 16)) return g_err.fail("%s: means must be 16-byte aligned", who);
    // Blocks that hold the positions of a query block: the most over all of them.
    const int own = (std::min(Sq, kQBlock) + block - 2) / block + 1;
    if (causal && count < own)
        return g_err.fail("%s: count must be at least %d, the blocks that hold a query block's own "
                          "positions", who, own);
    if (!launchable((long long)B * Hq * blocks_of(Sq, kQBlock), 1024))
        return g_err.fail("%s: too many query blocks", who);
    return 0;
}

SelectArgs select_args(const float* q_means, const float* k_means, int B, int Hq, int Hkv, int Sq,
                       int Skv, int D, int block, int count, int causal, int* index, void* scores) {
    SelectArgs a{};
    a.qm = q_means;
    a.km = k_means;
    a.score = (double*)scores;
    a.index = index;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.Sq = Sq;
    a.Skv = Skv;
    a.D = D;
    a.block = block;
    a.nq = blocks_of(Sq, kQBlock);
    a.nk = blocks_of(Skv, block);
    a.count = count;
    a.causal = causal;
    a.rows = (long long)B * Hq * a.nq;
    return a;
}

}  // namespace

extern "C" int sparse_select(const float* q_means, const float* k_means, int B, int Hq, int Hkv,
                             int Sq, int Skv, int D, int block, int count, int causal, int* index,
                             void* workspace, size_t workspace_bytes, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_choice(q_means, k_means, B, Hq, Hkv, Sq, Skv, D, block, count, causal, index,
                     "sparse_select"))
        return 1;
    if (B == 0 || Hq == 0 || Sq == 0) return 0;
    if (!aligned(q_means, 16)) return g_err.fail("sparse_select: means must be 16-byte aligned");
    const size_t need = sparse_select_workspace_bytes(B, Hq, Sq, Skv, block);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return g_err.fail("sparse_select: workspace misaligned or smaller than "
                          "sparse_select_workspace_bytes()");
    const SelectArgs a = select_args(q_means, k_means, B, Hq, Hkv, Sq, Skv, D, block, count, causal,
                                     index, workspace);
    if (a.nk > 0) {
        const int x = (int)(((long long)Hq / Hkv * a.nq + 15) / 16), y = B * Hkv;
        const int tiles = (a.nk + 15) / 16;
        // Shares of the key tiles: enough workgroups for the GPU, a tile a wave at least.
        const int z = (int)std::max<long long>(
            1, std::min<long long>((tiles + 3) / 4, 1024 / std::max(1LL, (long long)x * y)));
        const dim3 grid(x, y, z);
        if (D == 64)
            hipLaunchKernelGGL(score_kernel<64>, grid, dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL(score_kernel<128>, grid, dim3(256), 0, stream, a);
    }
    const dim3 quads((unsigned)((a.rows + 3) / 4)), singles((unsigned)a.rows);
    if (a.nk <= 256)
        hipLaunchKernelGGL((select_kernel<1, 4>), quads, dim3(256), 0, stream, a);
    else if (a.nk <= 512)
        hipLaunchKernelGGL((select_kernel<1, 8>), quads, dim3(256), 0, stream, a);
    else if (a.nk <= 1024)
        hipLaunchKernelGGL((select_kernel<1, 16>), quads, dim3(256), 0, stream, a);
    else if (a.nk <= 16384)
        hipLaunchKernelGGL((select_kernel<16, 16>), singles, dim3(1024), 0, stream, a);
    else
        hipLaunchKernelGGL((select_kernel<16, 32>), singles, dim3(1024), 0, stream, a);
    return g_err.launched("sparse_select", hipGetLastError());
}

namespace {
// Whether a choice is choose_one_kernel's: its workgroups together read at most so many bytes
// of key means (640 query blocks of 79 key blocks, D = 128, 26 MB: the whole call takes 87.5 us in
// one kernel and 87.2 in three; 2048 of 256, 268 MB: 45 against 31 for the choice alone).
constexpr double kOneBytes = 2.0e7;
bool one_kernel(int B, int Hq, int Sq, int Skv, int D, int block) {
    const double nk = blocks_of(Skv, block);
    return nk <= 4096 && (double)B * Hq * blocks_of(Sq, kQBlock) * nk * D * 4 <= kOneBytes;
}
size_t means_bytes(int B, int Hq, int Sq, int D) {
    return ((size_t)B * Hq * blocks_of(Sq, kQBlock) * D * sizeof(float) + 255) & ~(size_t)255;
}
}  // namespace

extern "C" size_t sparse_choose_workspace_bytes(int B, int Hq, int Sq, int Skv, int D, int block) {
    if (B <= 0 || Hq <= 0 || Sq <= 0 || D <= 0 || block <= 0 ||
        one_kernel(B, Hq, Sq, Skv, D, block))
        return 0;
    return means_bytes(B, Hq, Sq, D) + sparse_select_workspace_bytes(B, Hq, Sq, Skv, block);
}

extern "C" int sparse_choose(const void* q, const long long* q_strides, int dtype,
                             const float* k_means, int B, int Hq, int Hkv, int Sq, int Skv, int D,
                             int block, int count, int causal, int* index, void* workspace,
                             size_t workspace_bytes, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_choice(q, k_means, B, Hq, Hkv, Sq, Skv, D, block, count, causal, index,
                     "sparse_choose"))
        return 1;
    if (dtype != SPARSE_DTYPE_F16 && dtype != SPARSE_DTYPE_BF16)
        return g_err.fail("sparse_choose: bad dtype");
    if (B == 0 || Hq == 0 || Sq == 0) return 0;
    if (!q_strides) return g_err.fail("sparse_choose: null argument");
    if (check_strides(q_strides, q, 16, 8, "sparse_choose")) return 1;
    const size_t need = sparse_choose_workspace_bytes(B, Hq, Sq, Skv, D, block);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return g_err.fail("sparse_choose: workspace misaligned or smaller than "
                          "sparse_choose_workspace_bytes()");
    if (!one_kernel(B, Hq, Sq, Skv, D, block)) {
        float* means = (float*)workspace;
        const size_t used = means_bytes(B, Hq, Sq, D);
        const int rc =
            sparse_block_means(q, q_strides, dtype, B, Hq, Sq, D, kQBlock, means, stream);
        return rc ? rc
                  : sparse_select(means, k_means, B, Hq, Hkv, Sq, Skv, D, block, count, causal,
                                  index, (char*)workspace + used, workspace_bytes - used, stream);
    }
    SelectArgs a = select_args(nullptr, k_means, B, Hq, Hkv, Sq, Skv, D, block, count, causal, index,
                               nullptr);
    a.q = q;
    a.qb = q_strides[0];
    a.qh = q_strides[1];
    a.qs = q_strides[2];
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.rows), dim3(512), 0, stream, a);
    };
    if (dtype == SPARSE_DTYPE_F16)
        D == 64 ? go(choose_one_kernel<64, f16>) : go(choose_one_kernel<128, f16>);
    else
        D == 64 ? go(choose_one_kernel<64, bf16>) : go(choose_one_kernel<128, bf16>);
    return g_err.launched("sparse_choose", hipGetLastError());
}

extern "C" size_t sparse_attn_workspace_bytes(int B, int Hq, int Sq, int Skv, int D, int block,
                                              int count) {
    if (B <= 0 || Hq <= 0 || Sq <= 0 || Skv <= 0 || D <= 0 || block <= 0 || count <= 0) return 0;
    const int n = split_count(B, Hq, Sq, Skv, block, count);
    return n <= 1 ? 0 : (size_t)n * B * Hq * Sq * (D + 2) * sizeof(float);
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
    if (!good_scale(scale))
        return g_err.fail("sparse_attn: scale must be finite, and below 2.3e38");
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
    if (Skv > 1 && (k_strides[2] < D || v_strides[2] < D))
        return g_err.fail("sparse_attn: k/v rows overlap");
    const long long oe[3] = {B, Hq, Sq};
    if (!rows_apart(o_strides, oe, 3, D)) return g_err.fail("sparse_attn: o's rows overlap");
    const size_t need = sparse_attn_workspace_bytes(B, Hq, Sq, Skv, D, block, count);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return g_err.fail("sparse_attn: workspace misaligned or smaller than "
                          "sparse_attn_workspace_bytes()");
    auto st = [](const long long* s) { return Strides{s[0], s[1], s[2]}; };
    AttnArgs a{q, k, v, o, st(q_strides), st(k_strides), st(v_strides), st(o_strides), index,
               Hq, Hkv, Sq, Skv, D, block, blocks_of(Sq, kQBlock), blocks_of(Skv, block), count,
               causal, log2_scale(scale), scale < 0.f ? -1.f : 1.f,
               Skv > 0 ? split_count(B, Hq, Sq, Skv, block, count) : 1, (long long)B * Hq * Sq,
               nullptr, nullptr};
    if (a.nsplit > 1) {
        a.ws_o = (float*)workspace;
        a.ws_ml = a.ws_o + (size_t)a.nsplit * a.rows * D;
    }
    const long long grid = (long long)a.nq * B * Hq * a.nsplit;
    if (!launchable(grid, 256)) return g_err.fail("sparse_attn: too many query blocks");
    auto go = [&](auto kernel, auto combine) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, stream, a);
        if (a.nsplit > 1)
            hipLaunchKernelGGL(combine, dim3((unsigned)((a.rows * (D / 4) + 255) / 256)), dim3(256),
                               0, stream, a);
    };
    // Whether a head's K or V takes 2^31 bytes or more.
    const bool far = std::max(a.sk.s, a.sv.s) * 2 * Skv >= (1LL << 31);
    auto pick = [&](auto d, auto t) {
        constexpr int kD = decltype(d)::value;
        using E = decltype(t);
        if (block == 64)
            far ? go(attn_tile_kernel<kD, E, 2, true>, combine_kernel<E>)
                : go(attn_tile_kernel<kD, E, 2, false>, combine_kernel<E>);
        else
            far ? go(attn_tile_kernel<kD, E, 4, true>, combine_kernel<E>)
                : go(attn_tile_kernel<kD, E, 4, false>, combine_kernel<E>);
    };
    if (dtype == SPARSE_DTYPE_F16)
        D == 64 ? pick(std::integral_constant<int, 64>{}, f16{})
                : pick(std::integral_constant<int, 128>{}, f16{});
    else
        D == 64 ? pick(std::integral_constant<int, 64>{}, bf16{})
                : pick(std::integral_constant<int, 128>{}, bf16{});
    return g_err.launched("sparse_attn", hipGetLastError());
}
