// Requests over a paged cache and how the attention's work is dealt out, as the kernels of
// the 4-bit (kv4_kernel.hip) and the 8-bit cache (kv8_*.hip) take them. Functions are templates
// on a kernel's arguments `a`: those with cu, lens (device arrays), T, W, max_q, causal, and
// c.page, c.pages of the cache; from the row tiles on with the plan's fields too.
#pragma once

#include <algorithm>

#include "longctx.h"

namespace gfx906_amd {
namespace longctx {

constexpr int kPagedRequests = 4096;  // requests of a call at most
// Requests of up to so many query rows a kv head go to attn_few_kernel, in tiles of 32 that
// read the cache again, the others to the prompt kernels. One request behind 16384 tokens, 8 kv
// heads, us here / there: 128 rows 32 / 70, 256 42 / 69, 384 53 / 71; 8 requests behind 4096,
// 4 kv heads: 256 rows 44 / 58, 384 76 / 64.
constexpr int kFewRows = 256;

// A run is at least kPromptRun units: two prompts of 200 queries behind 800 tokens, 16/4 heads, 30
// us in the prompt kernels with 5, 37 with 8, 53 with 16.
constexpr int kTileRows = 128, kPromptStart = 4;  // (of the 4-bit cache's tiles)
constexpr long long kPromptRun = kPromptStart + 1;
constexpr int kSelfTiles = 1024, kSelfRequests = 256;  // SELF (attn_prompt_kernel)

#if defined(__HIP_DEVICE_COMPILE__)
// Loads of arrays that no kernel of a call writes, through the scalar cache where the
// index is uniform.
typedef const __attribute__((address_space(4))) int* ConstInts;
template <class A>
__device__ __forceinline__ int cu_at(const A& a, int b) {
    return a.cu ? min(max(((ConstInts)a.cu)[b], 0), a.T) : b;
}

// A request: its query rows first .. first + n - 1 of which the first m are computed,
// its tokens, and how many of them the table's columns hold.
struct Request {
    int first, n, m;
    long long len;
    int keys;
};
template <class A>
__device__ __forceinline__ Request request(const A& a, int b) {
    Request r;
    r.first = cu_at(a, b);
    r.n = max(0, cu_at(a, b + 1) - r.first);
    r.m = min(r.n, a.max_q);
    r.len = max(0, ((ConstInts)a.lens)[b]);
    r.keys = a.c.pages ? (int)min(r.len, (long long)a.W * a.c.page) : 0;
    return r;
}
// Keys that the query at place i of its request sees.
template <class A>
__device__ __forceinline__ int seen_by(const A& a, const Request& r, int i) {
    return a.causal ? (int)max(0LL, min((long long)r.keys, r.len - r.n + i + 1)) : r.keys;
}

// Row tiles of a request, and the 64-key chunks that tile rt reads.
template <int ROWS, class A>
__device__ __forceinline__ int tiles_of(const A& a, const Request& r) {
    const long long rows = (long long)r.m * a.G;
    return rows > a.few_rows ? (int)((rows + ROWS - 1) / ROWS) : 0;
}
template <int ROWS, class A>
__device__ __forceinline__ int tile_end(const A& a, const Request& r, int rt) {
    const long long last = min((long long)r.m * a.G, (rt + 1LL) * ROWS) - 1;
    return seen_by(a, r, (int)(last / a.G));
}
template <int ROWS, class A>
__device__ __forceinline__ int tile_chunks(const A& a, const Request& r, int rt) {
    return (tile_end<ROWS>(a, r, rt) + 63) / 64;
}
#endif

// Tiles of all requests and their units (chunks, and kPromptStart for the start and the
// merge of a tile that has any), summed up. One workgroup.
template <int ROWS, class A>
__global__ void __launch_bounds__(1024) prompt_plan_kernel(const A a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ int first[kPagedRequests + 1];
    __shared__ long long part[1024];
    const int t = threadIdx.x;
    auto scan = [&](long long x) {  // inclusive, over the workgroup
        part[t] = x;
        __syncthreads();
        for (int o = 1; o < 1024; o <<= 1) {
            const long long y = t >= o ? part[t - o] : 0;
            __syncthreads();
            part[t] += y;
            __syncthreads();
        }
        return part[t];
    };
    const int per = (a.B + 1023) / 1024, b0 = min(a.B, t * per), b1 = min(a.B, b0 + per);
    // (requests whose rows overlap could have more tiles than there is room for)
    auto cap = [&](long long x) { return (int)min(x, (long long)a.p_tiles); };
    long long n = 0;
    for (int b = b0; b < b1; ++b) n += tiles_of<ROWS>(a, request(a, b));
    n = scan(n) - n;
    for (int b = b0; b < b1; ++b) {
        first[b] = a.p_first[b] = cap(n);
        n += tiles_of<ROWS>(a, request(a, b));
    }
    __syncthreads();
    const int all = cap(part[1023]);
    if (t == 0) first[a.B] = a.p_first[a.B] = all;
    __syncthreads();

    const int run = (all + 1023) / 1024, i0 = min(all, t * run), i1 = min(all, i0 + run);
    int b = 0;
    for (int hi = a.B - 1; b < hi;) {  // the last request that starts at or before tile i0
        const int mid = (b + hi + 1) / 2;
        if (first[mid] <= i0)
            b = mid;
        else
            hi = mid - 1;
    }
    for (int pass = 0; pass < 2; ++pass) {
        long long sum = pass ? part[t] : 0;
        int x = b;
        Request r = request(a, x);
        for (int i = i0; i < i1; ++i) {
            while (i >= first[x + 1]) r = request(a, ++x);
            if (pass) {
                a.p_cost[i] = sum;
                a.p_req[i] = x;
            }
            const int c = tile_chunks<ROWS>(a, r, i - first[x]);
            sum += c ? c + kPromptStart : 0;
        }
        if (!pass) {
            __syncthreads();
            const long long before = scan(sum) - sum;
            if (t == 1023) a.p_cost[all] = before + sum;
            __syncthreads();
            part[t] = before;
        }
    }
#endif
}

constexpr int kGroups = 256, kMinUnits = 8;
// Tables of up to so many tokens go to the DIRECT form, and twice as many where there are heads
// enough for the GPU. One query each, 8 kv heads, us DIRECT / in runs: 1 request of 1000 tokens
// 8.5 / 13.4, of 2000 12.0 / 13.5, of 4000 19.5 / 13.8; 32 requests of 2000 16.3 / 24.2, of 4000
// 25.9 / 30.2, of 100 .. 4000 20.5 / 20.7.
constexpr int kDirectTokens = 2048, kDirectHeads = 256;
// How attn_few_kernel is launched.
struct FewPlan {
    int nb, tiles, groups;
    int start;          // units that a head's start counts
    bool direct, many;  // many: heads lie in 32 runs or more, if all requests are as long
    long long units;
    size_t o_off, ml_off, bytes;  // of the workspace
};
// ml: floats of a row's statistics; start: units that the start of a head of up to 16 rows counts;
// far: how many times as far DIRECT reaches where there are heads enough.
inline FewPlan few_plan(int B, int G, int Hkv, int D, int max_q, int max_len, int ml = 2,
                        int start = 16, int far = 2) {
    FewPlan p{};
    const long long rows = std::min<long long>((long long)max_q * G, kFewRows);
    p.nb = rows > 16 ? 2 : 1;
    p.tiles = (int)((rows + 16 * p.nb - 1) / (16 * p.nb));
    const long long segs = (long long)B * Hkv * p.tiles;
    // (a unit of 32 rows takes about as long as two of 16. 32 requests of 100 .. 16384 tokens,
    // one query each: 36.1 us with 8 units, 28.8 with 16, 30.5 with 24; 131072 tokens with 32
    // rows: 22.5 with 8, 24.0 with 16)
    p.start = p.nb == 1 ? start : 8;
    p.units = segs * ((std::max(max_len, 1) + 63LL) / 64 + p.start);
    p.direct = max_len <= (segs >= kDirectHeads ? far : 1) * kDirectTokens && segs < (1LL << 31);
    if (p.direct) return p;
    // A workgroup a CU, with a unit a wave at least. (Three of four waves, with 8 units for a
    // start: 32 ragged requests 29.3 us and not 28.8, 32 of 4000 tokens 33.5 and not 30.)
    p.groups = (int)std::max(1LL, std::min<long long>(kGroups, p.units / (kMinUnits + p.start) + 1));
    p.many = p.groups / segs >= 32;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.o_off = up((size_t)(B + 1) * sizeof(int));
    p.ml_off = p.o_off + (size_t)2 * p.groups * 16 * p.nb * D * sizeof(float);
    p.bytes = p.ml_off + (size_t)2 * p.groups * 16 * p.nb * ml * sizeof(float);
    return p;
}

// How attn_prompt_kernel is launched, and its part of the workspace behind the few
// rows' one. tiles: the most there can be of T queries. rows: of a tile; groups: workgroups.
struct PromptPlan {
    bool used;
    int groups, tiles;
    bool self;
    size_t cost_off, req_off, o_off, ml_off, bytes;
};
inline PromptPlan prompt_plan(int T, int B, int G, int D, int max_q, size_t after, int ml = 2,
                              int rows = kTileRows, int groups = 512) {
    PromptPlan p{};
    p.used = (long long)max_q * G > kFewRows;
    if (!p.used) return p;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.groups = groups;
    p.tiles = (int)std::min<long long>((long long)T * G / rows + B, (1LL << 27));
    p.cost_off = up(after) + up((size_t)(B + 1) * sizeof(int));
    p.self = p.tiles <= kSelfTiles && B <= kSelfRequests;
    p.req_off = p.cost_off + up((size_t)(p.tiles + 1) * sizeof(long long));
    p.o_off = p.req_off + up((size_t)p.tiles * sizeof(int));
    p.ml_off = p.o_off + (size_t)2 * p.groups * rows * D * sizeof(float);
    p.bytes = p.ml_off + (size_t)2 * p.groups * rows * ml * sizeof(float);
    return p;
}

}  // namespace longctx
}  // namespace gfx906_amd
