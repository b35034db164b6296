// Requests over a paged cache, as the kernels of the 4-bit (kv4_kernel.hip) and the 8-bit
// cache (kv8_*.hip) take them. Functions are templates on a kernel's arguments `a`: those
// with cu, lens (device arrays), T, W, max_q, causal, and c.page, c.pages of the cache.
#pragma once

#include "longctx.h"

#if defined(__HIP_DEVICE_COMPILE__)

namespace gfx906_amd {
namespace longctx {

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

}  // namespace longctx
}  // namespace gfx906_amd

#endif
