// Key/value cache in 4 bits for AMD MI355X (gfx950): pages and slots from
// request lengths, storing and reading rows, attention over the cache. The
// format and the entry points are described in gfx906_amd_attn.h.
//
// gfx950 converts between E2M1 pairs with an E8M0 scale and fp16, bf16 or fp32
// in one instruction (v_cvt_scalef32_*), rounding to nearest even and
// saturating, so the format costs half an instruction a value to read.
#include "longctx_tile.h"

#include <algorithm>
#include <type_traits>

#include "gfx906_amd_attn.h"

namespace {

using namespace gfx906_amd::longctx;

thread_local LastError g_err;

constexpr int kMaxRequests = KV4_MAX_REQUESTS;
// Requests of up to so many query rows a kv head go to attn_few_kernel, in tiles of 32 that
// read the cache again, the others to the prompt kernels. One request behind 16384 tokens, 8 kv
// heads, us here / there: 128 rows 32 / 70, 256 42 / 69, 384 53 / 71; 8 requests behind 4096,
// 4 kv heads: 256 rows 44 / 58, 384 76 / 64.
constexpr int kFewRows = 256;

// The cache as kernels see it. Offsets of rows are 64-bit: a cache may hold more
// than 2^32 bytes.
struct Cache {
    const uint8_t* kc;
    const uint8_t* ks;
    const uint8_t* vc;
    const uint8_t* vs;
    int pages, page, Hkv, D;
};

#if defined(__HIP_DEVICE_COMPILE__)
// Byte of the codes of token t (of its page), and of its first scale (the scale
// of 32 dims j is at 4 j further on).
__device__ __forceinline__ long long code_at(const Cache& c, long long page, int h, int t) {
    return ((page * c.Hkv + h) * c.page + t) * (c.D / 2);
}
__device__ __forceinline__ long long scale_at(const Cache& c, long long page, int h, int t) {
    const long long tok16 = (page * c.Hkv + h) * (c.page / 64) * 16 + (t >> 6) * 16 + (t & 15);
    return tok16 * (c.D / 32) * 4 + ((t >> 4) & 3);
}
// Eight codes in the element type (rounded to it where it does not hold them).
template <class T>
__device__ __forceinline__ typename Elem<T>::x8 expand(unsigned w, float s) {
    typename Elem<T>::x2 p[4];
    if constexpr (__is_same(T, f16)) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    }
    auto u = [](typename Elem<T>::x2 x) { return __builtin_bit_cast(unsigned, x); };
    return __builtin_bit_cast(typename Elem<T>::x8, u32x4{u(p[0]), u(p[1]), u(p[2]), u(p[3])});
}
// The two codes of a byte, rounded to the element type as expand() does.
template <class T>
__device__ __forceinline__ f32x2 expand_pair(unsigned byte, float s) {
    if constexpr (__is_same(T, f16))
        return __builtin_convertvector(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(byte, s, 0), f32x2);
    else
        return __builtin_convertvector(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(byte, s, 0), f32x2);
}
#endif

// -- pages and slots ------------------------------------------------------------------

struct PlanArgs {
    const int* lens;
    const int* new_lens;
    int* table;
    long long table_stride;
    const int* free_pages;
    const int* used;
    int *slots, *cu_new, *lens_out, *used_out, *missing;
    int W, n_free, B, page, n_slots;
};

// Every workgroup adds up all requests (each of the 256 threads a run of them, then a
// scan over the threads) and serves its share of the slots and of the requests' table
// rows. Entries that are read (held pages) and written (new ones) are different, so
// workgroups need no order. Bound by latency: lengths are read once and kept in LDS, where
// a slot finds its request by bisection; sums are 64-bit and kept saturated to 31 bits, as
// no slot or page past that is used. Nothing waits for a store, and a slot has a thread and a
// request's new pages 16 lanes of their own: 64 requests, one token each, 3.7 us; 6.3 with a wave a
// request, four slots a thread and the missing pages counted at the end.
__global__ void __launch_bounds__(256) plan_pages_kernel(const PlanArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ int len[kMaxRequests];       // cached tokens
    __shared__ int tok0[kMaxRequests + 1];  // first slot of a request
    __shared__ int pg0[kMaxRequests + 1];   // pages taken before a request
    __shared__ long long part[2][4];
    constexpr long long kCap = 0x7fffffff;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, B = a.B, P = a.page;
    const int sh = P == 64 ? 6 : P == 128 ? 7 : 8;
    auto pages = [&](long long n) { return (n + P - 1) >> sh; };
    auto cap = [&](long long x) { return (int)min(x, kCap); };
    const int per = (B + 255) / 256, b0 = min(B, t * per), b1 = min(B, b0 + per);
    long long n = 0, p = 0;
    for (int b = b0; b < b1; ++b) {
        const long long have = max(0, a.lens[b]), more = max(0, a.new_lens[b]);
        len[b] = (int)have;
        tok0[b] = (int)more;  // (turned into the first slot below)
        n += more;
        p += pages(have + more) - pages(have);
    }
    const int used = max(0, a.used[0]);
    long long sn = n, sp = p;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(sn, o), y = __shfl_up(sp, o);
        if (lane >= o) {
            sn += x;
            sp += y;
        }
    }
    if (lane == 63) {
        part[0][wave] = sn;
        part[1][wave] = sp;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        sn += part[0][w];
        sp += part[1][w];
    }
    if (t == 255) {
        tok0[B] = cap(sn);
        pg0[B] = cap(sp);
    }
    n = sn - n;
    p = sp - p;
    for (int b = b0; b < b1; ++b) {
        const long long have = len[b], more = tok0[b];
        tok0[b] = cap(n);
        pg0[b] = cap(p);
        n += more;
        p += pages(have + more) - pages(have);
    }
    __syncthreads();

    // (new tokens of a request: from its first slot to the next request's; where those are
    // saturated, from memory again)
    auto more_of = [&](int b) -> long long {
        return tok0[b + 1] < kCap ? tok0[b + 1] - tok0[b] : max(0, a.new_lens[b]);
    };
    if (blockIdx.x == 0) {
        // Pages of columns behind the table take their place in the free list too.
        long long lost = 0;
        for (int b = b0; b < b1; ++b) {
            const long long held = pages(len[b]), need = pages(len[b] + more_of(b)) - held;
            const long long in_row = max(0LL, min(need, a.W - held));
            lost += need - max(0LL, min(in_row, (long long)a.n_free - used - pg0[b]));
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) lost += __shfl_xor(lost, o);
        if (lane == 0) part[0][wave] = lost;
        __syncthreads();
        if (t == 0) {
            a.missing[0] = cap(part[0][0] + part[0][1] + part[0][2] + part[0][3]);
            a.used_out[0] = max(used, (int)min((long long)used + pg0[B], (long long)a.n_free));
        }
    }

    // Page of place k of request b's row, or -1.
    auto fresh = [&](int b, long long k) -> int {
        const long long f = (long long)used + pg0[b] + (k - pages(len[b]));
        return k < a.W && f < a.n_free ? a.free_pages[f] : -1;
    };
    const int stride = gridDim.x * 256, gt = blockIdx.x * 256 + t;
    for (long long s = gt; s < a.n_slots; s += stride) {
        int slot = -1;
        if (s < tok0[B]) {
            int lo = 0, hi = B - 1;  // last request whose first slot is at most s
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (tok0[mid] <= s)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            const long long pos = (long long)len[lo] + (s - tok0[lo]), k = pos >> sh;
            const int page = k >= pages(len[lo]) ? fresh(lo, k)
                             : k < a.W           ? a.table[lo * a.table_stride + k]
                                                 : -1;
            const long long at = (long long)page * P + (pos & (P - 1));
            if (page >= 0 && at <= kCap) slot = (int)at;
        }
        a.slots[s] = slot;
    }
    for (int b = gt; b <= B; b += stride) {
        a.cu_new[b] = tok0[b];
        if (b < B) a.lens_out[b] = cap(len[b] + more_of(b));
    }
    for (int b = gt / 16; b < B; b += stride / 16) {
        const long long last = min(pages(len[b] + more_of(b)), (long long)a.W);
        for (long long k = pages(len[b]) + (lane & 15); k < last; k += 16)
            a.table[b * a.table_stride + k] = fresh(b, k);
    }
#endif
}

// -- storing and reading rows ---------------------------------------------------------

struct RowArgs {
    const void* k;
    const void* v;
    void* ko;
    void* vo;
    long long kt, kh, vt, vh;  // strides of k and v: token, head
    const int* slots;
    Cache c;
    unsigned n;  // blocks of 32 values (store) or pieces of 8 (load) in k, and in v
};

#if defined(__HIP_DEVICE_COMPILE__)
// Piece id of K or V, 2^ds pieces in a row: piece d of head h of row t.
struct Piece {
    unsigned t;
    int h, d;
};
__device__ __forceinline__ Piece piece(const Cache& c, unsigned id, int ds) {
    const unsigned row = id >> ds, t = row / (unsigned)c.Hkv;
    return {t, (int)(row - t * c.Hkv), (int)(id & ((1u << ds) - 1))};
}
#endif

// A lane stores a block of 32 values: four 16-byte loads in flight, no exchange. Bound by
// bytes: 16384 rows of 16 heads, D = 128, 41 us (4.1 TB/s), and 34 where the last-level cache
// holds rows; there a lane per 8 values, with the block's maximum exchanged between four, takes 45.
// grid.y: K, V.
template <class T>
__global__ void __launch_bounds__(256) store_kernel(const RowArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using x8 = typename Elem<T>::x8;
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.n) return;
    const bool is_v = blockIdx.y;
    const Piece p = piece(a.c, id, a.c.D == 128 ? 2 : 1);
    const int slot = a.slots[p.t];
    if (slot < 0 || slot >= a.c.pages * (long long)a.c.page) return;
    const T* src = is_v ? (const T*)a.v + p.t * a.vt + p.h * a.vh
                        : (const T*)a.k + p.t * a.kt + p.h * a.kh;
    x8 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const x8*>(src + 32 * p.d + 8 * i);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        top = max(top, __float_as_uint((float)x[i / 8][i % 8]) & 0x7fffffffu);
    const unsigned e = top >> 23, byte = e == 255 ? 255 : (unsigned)max(1, (int)e - 2);
    const float s = e8m0(byte);
    u32x4 w = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)x[i][j];
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], f[0], f[1], s, 0);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], f[2], f[3], s, 1);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], f[4], f[5], s, 2);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], f[6], f[7], s, 3);
    }
    const int page = slot / a.c.page, tok = slot % a.c.page;
    uint8_t* codes = const_cast<uint8_t*>(is_v ? a.c.vc : a.c.kc);
    uint8_t* scales = const_cast<uint8_t*>(is_v ? a.c.vs : a.c.ks);
    *reinterpret_cast<u32x4*>(codes + code_at(a.c, page, p.h, tok) + 16 * p.d) = w;
    scales[scale_at(a.c, page, p.h, tok) + 4 * p.d] = (uint8_t)byte;
#endif
}

// Rows back: a lane per 8 values, so that a wave's 16-byte stores are contiguous; 34 us
// for as many rows, and 45 with a lane per 32 values.
template <class T>
__global__ void __launch_bounds__(256) load_kernel(const RowArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.n) return;
    const bool is_v = blockIdx.y;
    const Piece p = piece(a.c, id, a.c.D == 128 ? 4 : 3);
    const int slot = a.slots[p.t];
    unsigned w = 0;
    float s = 1.f;
    if (slot >= 0 && slot < a.c.pages * (long long)a.c.page) {
        const int page = slot / a.c.page, tok = slot % a.c.page;
        w = *reinterpret_cast<const unsigned*>((is_v ? a.c.vc : a.c.kc) +
                                               code_at(a.c, page, p.h, tok) + 4 * p.d);
        s = e8m0((is_v ? a.c.vs : a.c.ks)[scale_at(a.c, page, p.h, tok) + (p.d & ~3)]);
    }
    reinterpret_cast<typename Elem<T>::x8*>(is_v ? a.vo : a.ko)[id] = expand<T>(w, s);
#endif
}

// -- attention ------------------------------------------------------------------------

struct AttnArgs {
    const void* q;
    void* o;
    long long qt, qh, ot, oh;  // strides: token, head
    Cache c;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* cu;  // NULL: one query a request
    int W, T, B, Hq, G, max_q, causal;
    float scale, qsign;  // log2_scale(); a negative scale negates q
    int few_rows, tiles;  // requests of at most so many query rows a kv head go to attn_few_kernel
    // attn_few_kernel's partial results: two slots a workgroup (below).
    int groups, min_units, start_units;
    int* starts;  // [B + 1]: first unit of every request; units a workgroup
    float* ws_o;        // [slot][row][D]
    float* ws_ml;       // [slot][row][2]
    // The same of attn_prompt_kernel, and its plan.
    int p_groups, p_tiles;  // p_tiles: room for so many tiles
    int* p_first;         // [B + 1]: first tile of every request
    long long* p_cost;    // [tiles + 1]: units before a tile, of one kv head
    int* p_req;           // [tiles]: request of a tile
    float* p_o;
    float* p_ml;
};

#if defined(__HIP_DEVICE_COMPILE__)
// Loads of arrays that no kernel of a call writes, through the scalar cache where the
// index is uniform.
typedef const __attribute__((address_space(4))) int* ConstInts;
__device__ __forceinline__ int cu_at(const AttnArgs& a, int b) {
    return a.cu ? min(max(((ConstInts)a.cu)[b], 0), a.T) : b;
}

// A request: its query rows first .. first + n - 1 of which the first m are computed,
// its tokens, and how many of them the table's columns hold.
struct Request {
    int first, n, m;
    long long len;
    int keys;
};
__device__ __forceinline__ Request request(const AttnArgs& a, int b) {
    Request r;
    r.first = cu_at(a, b);
    r.n = max(0, cu_at(a, b + 1) - r.first);
    r.m = min(r.n, a.max_q);
    r.len = max(0, ((ConstInts)a.lens)[b]);
    r.keys = a.c.pages ? (int)min(r.len, (long long)a.W * a.c.page) : 0;
    return r;
}
// Keys that the query at place i of its request sees.
__device__ __forceinline__ int seen_by(const AttnArgs& a, const Request& r, int i) {
    return a.causal ? (int)max(0LL, min((long long)r.keys, r.len - r.n + i + 1)) : r.keys;
}

// Whether a scale byte may stand for an infinite or NaN value in element type T.
template <class T>
constexpr unsigned kScaleLimit = __is_same(T, f16) ? 141u : 253u;

// One query row over the keys t0 .. t1 - 1 of its request, by one wave: 64 keys at a
// time, a score per lane, then a pair of dims per lane. Keys the row does not see are
// not touched at all, so that what they hold cannot reach it. Keys and values are those of the
// matrix kernels, rounded to the element type: whether a row is done here depends on tokens
// that it does not see, and a value past fp16's range must be the same infinity either way.
template <int D, class T>
__device__ void attend_row(const AttnArgs& a, const T* q, int hk, int b, int t0, int t1, T* o) {
    const int lane = threadIdx.x & 63;
    float m = kNoMax, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = t0; j0 < t1; j0 += 64) {
        const int page = a.table[b * a.table_stride + j0 / a.c.page], j = j0 + lane;
        if (page < 0 || page >= a.c.pages) continue;
        float s = -INFINITY;
        if (j < t1) {
            const long long ca = code_at(a.c, page, hk, j % a.c.page);
            const long long sa = scale_at(a.c, page, hk, j % a.c.page);
            s = 0.f;
            for (int i = 0; i < D / 2; ++i) {
                const f32x2 x =
                    expand_pair<T>((unsigned)a.c.kc[ca + i], e8m0(a.c.ks[sa + 4 * (i / 16)]));
                s = fmaf((float)q[2 * i], x[0], s);
                s = fmaf((float)q[2 * i + 1], x[1], s);
            }
            s *= a.scale * a.qsign;
        }
        const float mn = max2(m, wave_max(s)), w = exp2f(m - mn), p = exp2f(s - mn);
        l = l * w + wave_sum(p);
        o0 *= w;
        o1 *= w;
        m = mn;
        for (int i = 0; i < 64 && j0 + i < t1; ++i) {
            const float pi = __shfl(p, i);
            if (2 * lane < D) {
                const int t = (j0 + i) % a.c.page;
                const f32x2 x =
                    expand_pair<T>((unsigned)a.c.vc[code_at(a.c, page, hk, t) + lane],
                                   e8m0(a.c.vs[scale_at(a.c, page, hk, t) + 4 * (lane / 16)]));
                o0 = fmaf(pi, x[0], o0);
                o1 = fmaf(pi, x[1], o1);
            }
        }
    }
    if (2 * lane < D) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        *reinterpret_cast<typename Elem<T>::x2*>(o + 2 * lane) = Elem<T>::cvt2(o0 * inv, o1 * inv);
    }
}

// Whether one of the tokens seen .. end - 1 of request b may hold an infinite or NaN
// value: a weight of 0 would not keep that out of the sum of a row that does not see it. For a
// wave.
template <int D, class T>
__device__ __forceinline__ bool may_spoil(const AttnArgs& a, int b, int hk, int seen, int end) {
    bool bad = false;
    for (int e = threadIdx.x & 63; e < (end - seen) * (D / 32); e += 64) {
        const int t = seen + e / (D / 32), page = a.table[b * a.table_stride + t / a.c.page];
        if ((unsigned)page < (unsigned)a.c.pages)
            bad |= a.c.vs[scale_at(a.c, page, hk, t % a.c.page) + e % (D / 32) * 4] >= kScaleLimit<T>;
    }
    return __any(bad);
}

// A lane's part of 16 cache rows: 32 (D = 128) or 16 dims of row l%16, D/32 dwords.
template <int D>
struct Codes {
    unsigned w[D / 32];
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (D == 128) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p);
            w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(p);
            w[0] = x[0], w[1] = x[1];
        }
    }
};
#endif

// Attention of requests with few query rows (single tokens, drafts), bound by the
// bytes of the cache.
//
// Work is counted in units of 64 tokens of one kv head of one request (and of one tile
// of 16 NB query rows: a token's G heads share the keys). The lengths lie on the GPU, so
// every workgroup adds up all requests' units and takes an equal run of them, which may
// end inside a head and span several: a ragged batch fills the GPU as an even one does.
// Within a run the eight waves take every eighth unit of a head, each with its own
// running max and sums, and are merged through LDS. A head that lies in one run is
// finished there; of others each run writes unnormalised O and (m, l) to a slot of the
// workspace (2 w + 1 of workgroup w for the run that begins the head, 2 w for the
// others), which few_combine_kernel merges.
//
// A wave reads 16 keys as 16 bytes a lane: lane group g has dims g D/4 .. of key l%16 (at
// D = 128 one scale block), converts them in registers, and they are the matrix operand
// as they stand: the dims of a step are split over the lane groups alike for K and
// Q, whatever their order. V goes through LDS in the element type (8 KB a wave), as the
// second product sums over keys. The next unit's K codes are loaded once the scores of
// one are done, its V codes at the end, so that neither needs registers twice (two units ahead,
// in twice the registers, measured 31.3 us a call and not 28.6 on the batch below).
//
// DIRECT: short tables. One workgroup a head, no runs, no slots and no second kernel.
//
// 32 requests of 100 .. 16384 tokens, 8 kv heads of 128, one query each: 26 us and 5 for the
// merge (103 MB: 3.3 TB/s in all); 131072 tokens, 2 kv heads, 32 rows: 17 and 6, of which the bytes
// take 7, with two units a wave. 262144 tokens take 26 and 524288 36, 2.6 us more for every unit a
// wave, and 16384 tokens (34 workgroups) still 15: some ten of the 17 are a run's start (the search,
// Q, first loads) and end (eight waves' merge, partial results); 1024 tokens, 16 heads of 64, in
// DIRECT: 7.
template <int D, class T, int NB, bool DIRECT>
__global__ void __launch_bounds__(512, D == 64 && NB == 1 ? 4 : 2) attn_few_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using W = Tile<D, T, NB>;
    using x8 = typename W::x8;
    constexpr int R = 16 * NB, DW = D / 32, NW = 8, NT = 64 * NW;
    __shared__ __attribute__((aligned(1024))) char stage[NW][W::BYTES];
    __shared__ float ml_s[NW][R][2];
    __shared__ int run0[NT + 1];
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

    // Units of a request (the host has checked that all of them fit an int).
    struct Units {
        int chunks, tiles;
    };
    auto units_of = [&](const Request& r) {
        const int rows = (int)min((long long)r.m * a.G, 1LL << 30);
        Units u{0, 0};
        if (rows > 0 && rows <= a.few_rows) {
            u.chunks = (r.keys + 63) / 64;
            u.tiles = (rows + R - 1) / R;
        }
        return u;
    };
    // (a head's start and merge cost as much as a.start_units units)
    auto count = [&](const Units& u) {
        return u.chunks ? (u.chunks + a.start_units) * u.tiles * a.c.Hkv : 0;
    };
    int b = 0, start = 0, u0 = 0, hi = 1;
    if constexpr (!DIRECT) {
        const int per_run = (a.B + NT - 1) / NT;
        int n = 0;
        for (int x = tid * per_run; x < min(a.B, (tid + 1) * per_run); ++x)
            n += count(units_of(request(a, x)));
        int sum = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 63) ml_s[wave][0][0] = __int_as_float(sum);
        __syncthreads();
        for (int w = 0; w < wave; ++w) sum += __float_as_int(ml_s[w][0][0]);
        run0[tid + 1] = sum;
        if (tid == 0) run0[0] = 0;
        __syncthreads();
        const int all = run0[NT];
        const int per = max(a.min_units, uni((int)((unsigned)(all + a.groups - 1) / (unsigned)a.groups)));
        if (blockIdx.x == 0) {
            n = run0[tid];
            for (int x = tid * per_run; x < min(a.B, (tid + 1) * per_run); ++x) {
                a.starts[x] = n;
                n += count(units_of(request(a, x)));
            }
            if (tid == 0) a.starts[a.B] = per;
        }
        // (the last run may end past 2^31 before it is cut)
        const long long lo = (long long)blockIdx.x * per;
        if (lo >= all) return;
        u0 = (int)lo;
        hi = (int)min((long long)all, lo + per);
        if (run0[tid] <= u0 && u0 < run0[tid + 1]) found = tid;
        __syncthreads();
        b = uni(found) * per_run;
        start = uni(run0[uni(found)]);
    }

    while (u0 < hi) {
        Request req;
        int chunks, c0, c1, hk, rt;
        bool whole;
        long long slot = 0;
        if constexpr (DIRECT) {  // grid: requests x kv heads x row tiles
            const int seg = uni(blockIdx.x / a.tiles);
            rt = blockIdx.x - seg * a.tiles;
            b = uni(seg / a.c.Hkv);
            hk = seg - b * a.c.Hkv;
            req = request(a, b);
            if (rt * R >= (long long)req.m * a.G || (long long)req.m * a.G > a.few_rows) return;
            chunks = (req.keys + 63) / 64;
            c0 = 0;
            c1 = chunks;
            whole = true;
            u0 = hi;
        } else {
            req = request(a, b);
            Units un = units_of(req);
            while (start + count(un) <= u0) {
                start += count(un);
                req = request(a, ++b);
                un = units_of(req);
            }
            chunks = un.chunks;
            const int each = chunks + a.start_units;
            const int s = uni((int)((unsigned)(u0 - start) / (unsigned)each));
            const int p0 = u0 - start - s * each, p1 = min(each, p0 + (hi - u0));
            u0 += p1 - p0;
            c0 = max(0, p0 - a.start_units);
            c1 = p1 - a.start_units;
            if (c1 <= 0) continue;  // (the run ends before the head's first unit)
            hk = uni((int)((unsigned)s / (unsigned)un.tiles));
            rt = s - hk * un.tiles;
            whole = c0 == 0 && c1 == chunks;
            slot = 2LL * blockIdx.x + (c0 == 0 ? 1 : 0);
        }

        // This lane's query rows (16 nb + i of the tile): Q fragments and keys seen.
        W w;
        w.init(lane);
        int lim[NB];
        const int rows = req.m * a.G;
        const unsigned neg = a.qsign < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int r = rt * R + 16 * nb + i, tok = r / a.G, h = hk * a.G + r - tok * a.G;
            const bool ok = r < rows;
            lim[nb] = ok ? seen_by(a, req, tok) : 0;
            const T* q = (const T*)a.q + (req.first + tok) * a.qt + h * a.qh + g * (D / 4);
#pragma unroll
            for (int n = 0; n < DW; ++n) {
                u32x4 x = {};
                if (ok) x = *reinterpret_cast<const u32x4*>(q + 8 * n);
                w.qf[nb][n] = __builtin_bit_cast(x8, x ^ neg);
            }
        }
        // Keys every row of the tile sees.
        const int all_see = uni(seen_by(a, req, rt * R / a.G));

        const ConstInts table = (ConstInts)(a.table + b * a.table_stride);
        const int shift = a.c.page == 64 ? 0 : a.c.page == 128 ? 1 : 2;
        Codes<D> kc[4], vc[4];
        unsigned ks = 0, vs = 0;
        // (past the run: its last unit's page, read again and not used)
        auto page_of = [&](int c) { return table[min(c, c1 - 1) >> shift]; };
        const int off = i * (D / 2) + g * (D / 8);
        const int soff = i * (D / 8) + (D == 128 ? g : g >> 1) * 4;
        // The loads are unconditional, so that the compiler waits for them where they are
        // used: a page outside the cache reads page 0, and the unit's keys are masked.
        auto rows_at = [&](int c, int page) {
            const unsigned p = (unsigned)page < (unsigned)a.c.pages ? page : 0;
            return ((long long)p * a.c.Hkv + hk) * a.c.page + (c & ((1 << shift) - 1)) * 64;
        };
        auto fetch_k = [&](int c, int page) __attribute__((always_inline)) {
            const long long row = rows_at(c, page);
            const uint8_t* p = a.c.kc + row * (D / 2);
            ks = *reinterpret_cast<const unsigned*>(a.c.ks + row / 4 * (D / 8) + soff);
#pragma unroll
            for (int t = 0; t < 4; ++t) kc[t].load(p + (off + t * 8 * D));
        };
        auto fetch_v = [&](int c, int page) __attribute__((always_inline)) {
            const long long row = rows_at(c, page);
            const uint8_t* p = a.c.vc + row * (D / 2);
            vs = *reinterpret_cast<const unsigned*>(a.c.vs + row / 4 * (D / 8) + soff);
#pragma unroll
            for (int t = 0; t < 4; ++t) vc[t].load(p + (off + t * 8 * D));
        };
        char* const st = stage[wave];
        int c = c0 + wave, page = -1, next = -1;
        if (c < c1) {  // (a request without keys may have no table)
            page = page_of(c);
            next = page_of(c + NW);
            fetch_k(c, page);
            fetch_v(c, page);
        }
        for (; c < c1; c += NW) {
            const bool ok = (unsigned)page < (unsigned)a.c.pages;
            page = next;
            next = page_of(c + 2 * NW);
            f32x4 S[2][2][NB];
            float sc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                sc[t] = e8m0(ks >> (8 * t) & 255);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) S[t / 2][t % 2][nb] = f32x4{};
            }
#pragma unroll
            for (int n = 0; n < DW; ++n)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const x8 kf = expand<T>(kc[t].w[n], sc[t]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        S[t / 2][t % 2][nb] = Elem<T>::mma16(kf, w.qf[nb][n], S[t / 2][t % 2][nb]);
                }
            __builtin_amdgcn_sched_barrier(0);
            fetch_k(c + NW, page);
            const int key0 = c * 64;
            if (key0 + 64 > all_see || !ok) {
                int lim2[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) lim2[nb] = ok ? lim[nb] : 0;
#pragma unroll
                for (int half = 0; half < 2; ++half) w.mask(S[half], key0 + 32 * half, lim2, g);
                // Values behind the last token are nothing.
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (!ok || key0 + 16 * t + i >= req.keys) {
                        vs = (vs & ~(255u << (8 * t))) | 127u << (8 * t);
#pragma unroll
                        for (int n = 0; n < DW; ++n) vc[t].w[n] = 0;
                    }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                x8 P[NB];
                w.softmax(S[half], P, a.scale);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float sc = e8m0(vs >> (8 * (2 * half + t)) & 255);
                    const int row = 16 * t + i;
#pragma unroll
                    for (int n = 0; n < DW; ++n)
                        *reinterpret_cast<GFX906_LDS x8*>(
                            (GFX906_LDS char*)st + row * W::RB +
                            ((g * DW + n) ^ vswz<W::NU>(row)) * 16) =
                            expand<T>(vc[2 * half + t].w[n], sc);
                }
                __builtin_amdgcn_wave_barrier();
                if (half) {
                    __builtin_amdgcn_sched_barrier(0);
                    fetch_v(c + NW, page);
                }
                w.pv(st, P);
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        // Merge the waves: a common max, then sums of 16 rows at a time through LDS.
        float l[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            l[nb] = quad_sum(w.lacc[nb][0]);
            if (g == 0) {
                ml_s[wave][16 * nb + i][0] = w.m[nb];
                ml_s[wave][16 * nb + i][1] = l[nb];
            }
        }
        __syncthreads();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float mx = kNoMax;
#pragma unroll
            for (int x = 0; x < NW; ++x) mx = max2(mx, ml_s[x][16 * nb + i][0]);
            const float f = __builtin_amdgcn_exp2f(w.m[nb] - mx);
            auto* const buf = (GFX906_LDS float*)(GFX906_LDS char*)stage[wave];
#pragma unroll
            for (int ob = 0; ob < W::NO; ++ob)
                *reinterpret_cast<GFX906_LDS f32x4*>(buf + i * D + ((16 * ob + 4 * g) ^ (4 * i & (D - 4)))) =
                    w.oacc[ob][nb] * f;
            __syncthreads();
            for (int e = tid; e < 4 * D; e += NT) {  // 16 rows x D/4 quads
                const int r = e / (D / 4), d = (e - r * (D / 4)) * 4, x = d ^ (4 * r & (D - 4));
                f32x4 acc = {};
                float mr = kNoMax, lr = 0.f;
#pragma unroll
                for (int y = 0; y < NW; ++y) mr = max2(mr, ml_s[y][16 * nb + r][0]);
#pragma unroll
                for (int y = 0; y < NW; ++y) {
                    lr += ml_s[y][16 * nb + r][1] * __builtin_amdgcn_exp2f(ml_s[y][16 * nb + r][0] - mr);
                    acc += *reinterpret_cast<const GFX906_LDS f32x4*>(
                        (const GFX906_LDS float*)(const GFX906_LDS char*)stage[y] + r * D + x);
                }
                const int row = rt * R + 16 * nb + r;
                if (row >= rows) continue;
                if (whole) {
                    const int tok = row / a.G, h = hk * a.G + row - tok * a.G;
                    T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + d;
                    acc *= lr != 0.f ? 1.f / lr : 0.f;
                    const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
                    *reinterpret_cast<u32x2*>(o) =
                        u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
                } else {
                    *reinterpret_cast<f32x4*>(a.ws_o + (slot * R + 16 * nb + r) * D + d) = acc;
                    if (d == 0)
                        *reinterpret_cast<f32x2*>(a.ws_ml + (slot * R + 16 * nb + r) * 2) =
                            f32x2{mr, lr};
                }
            }
            __syncthreads();
        }
        if constexpr (DIRECT) {
            for (int r = wave; r < R && rt * R + r < rows; r += NW) {
                const int tok = (rt * R + r) / a.G, h = hk * a.G + rt * R + r - tok * a.G;
                if (may_spoil<D, T>(a, b, hk, seen_by(a, req, tok), req.keys))
                    attend_row<D, T>(a, (const T*)a.q + (req.first + tok) * a.qt + h * a.qh, hk, b, 0,
                                     seen_by(a, req, tok), (T*)a.o + (req.first + tok) * a.ot + h * a.oh);
            }
        }
    }
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// Merges the slots of a head that lies in several runs, writes the zeros of a request
// without tokens, and does a row again that a value it does not see may have spoilt: query row
// `row` of kv head hk of request b, by a workgroup of NT threads.
template <int D, class T, int NB, int NT>
__device__ __forceinline__ void few_combine(const AttnArgs& a, int b, int hk, int row) {
    constexpr int R = 16 * NB, DQ = D / 4, NG = NT / DQ, NW = NT / 64;
    __shared__ f32x4 acc_s[NW][DQ];
    __shared__ float ml_s[NW][2];
    const Request req = request(a, b);
    const long long rows = (long long)req.m * a.G;
    if (rows > a.few_rows || row >= rows) return;
    const int tok = row / a.G, h = hk * a.G + row - tok * a.G;
    const int grp = threadIdx.x / DQ, d = (threadIdx.x - grp * DQ) * 4;
    T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + d;
    const int chunks = (req.keys + 63) / 64, tiles = (int)((rows + R - 1) / R), rt = row / R;
    if (chunks == 0) {
        if (grp == 0) *reinterpret_cast<u32x2*>(o) = u32x2{};
        return;
    }
    if (may_spoil<D, T>(a, b, hk, seen_by(a, req, tok), req.keys)) {  // (the same for every wave)
        if (threadIdx.x < 64)
            attend_row<D, T>(a, (const T*)a.q + (req.first + tok) * a.qt + h * a.qh, hk, b, 0,
                             seen_by(a, req, tok), o - d);
        return;
    }
    const int per = a.starts[a.B];
    const int s = a.starts[b] + (hk * tiles + rt) * (chunks + a.start_units) + a.start_units;
    const int w0 = (int)((unsigned)s / (unsigned)per);
    const int w1 = (int)((unsigned)(s + chunks - 1) / (unsigned)per);
    if (w0 == w1) return;
    float m = kNoMax, l = 0.f;
    f32x4 acc = {};
    constexpr int U = 4;
    for (int x = w0 + grp; x <= w1; x += NG * U) {
        f32x2 ml[U];
        f32x4 p[U];
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int y = x + n * NG;
            ml[n] = f32x2{kNoMax, 0.f};
            p[n] = f32x4{};
            if (y <= w1) {
                const long long at = (2LL * y + (y == w0 ? 1 : 0)) * R + (row - rt * R);
                ml[n] = *reinterpret_cast<const f32x2*>(a.ws_ml + at * 2);
                p[n] = *reinterpret_cast<const f32x4*>(a.ws_o + at * D + d);
            }
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const float mn = max2(m, ml[n][0]);
            const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(ml[n][0] - mn);
            acc = acc * f + p[n] * e;
            l = l * f + ml[n][1] * e;
            m = mn;
        }
    }
    // The groups of a wave, then the waves. (All groups through LDS: 100000 tokens, one kv head of 64,
    // 16.3 us a call and not 14.0; 131072, 2 of 128, 32 rows, 22.5 and 22.1.)
#pragma unroll
    for (int step = DQ; step < 64; step <<= 1) {
        const float mo = __shfl_xor(m, step), lo = __shfl_xor(l, step), mn = max2(m, mo);
        const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(mo - mn);
        l = l * f + lo * e;
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n] = acc[n] * f + __shfl_xor(acc[n], step) * e;
        m = mn;
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < DQ) {
        acc_s[wave][d / 4] = acc;
        if (d == 0) {
            ml_s[wave][0] = m;
            ml_s[wave][1] = l;
        }
    }
    __syncthreads();
    if (grp) return;
    float mx = kNoMax;
#pragma unroll
    for (int n = 0; n < NW; ++n) mx = max2(mx, ml_s[n][0]);
    acc = f32x4{};
    l = 0.f;
#pragma unroll
    for (int n = 0; n < NW; ++n) {
        const float f = __builtin_amdgcn_exp2f(ml_s[n][0] - mx);
        acc += acc_s[n][d / 4] * f;
        l += ml_s[n][1] * f;
    }
    acc *= l != 0.f ? 1.f / l : 0.f;
    const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
    *reinterpret_cast<u32x2*>(o) =
        u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
}
#endif

// grid: requests x kv heads, query rows.
template <int D, class T, int NB, int NT>
__global__ void __launch_bounds__(NT) few_combine_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int b = blockIdx.x / a.c.Hkv;
    few_combine<D, T, NB, NT>(a, b, blockIdx.x - b * a.c.Hkv, blockIdx.y);
#endif
}

// -- prompts: requests of more than few_rows query rows a kv head -----------------------

// A run is at least kPromptRun units: two prompts of 200 queries behind 800 tokens, 16/4 heads, 30
// us in the prompt kernels with 5, 37 with 8, 53 with 16.
constexpr int kTileRows = 128, kPromptStart = 4;
constexpr long long kPromptRun = kPromptStart + 1;
constexpr int kSelfTiles = 1024, kSelfRequests = 256;  // SELF (attn_prompt_kernel)

#if defined(__HIP_DEVICE_COMPILE__)
// Row tiles of a request, and the 64-key chunks that tile rt reads.
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Request& r) {
    const long long rows = (long long)r.m * a.G;
    return rows > a.few_rows ? (int)((rows + kTileRows - 1) / kTileRows) : 0;
}
__device__ __forceinline__ int tile_end(const AttnArgs& a, const Request& r, int rt) {
    const long long last = min((long long)r.m * a.G, (rt + 1LL) * kTileRows) - 1;
    return seen_by(a, r, (int)(last / a.G));
}
__device__ __forceinline__ int tile_chunks(const AttnArgs& a, const Request& r, int rt) {
    return (tile_end(a, r, rt) + 63) / 64;
}
#endif

// Tiles of all requests and their units (chunks, and kPromptStart for the start and the
// merge of a tile that has any), summed up. One workgroup.
__global__ void __launch_bounds__(1024) prompt_plan_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ int first[kMaxRequests + 1];
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
    for (int b = b0; b < b1; ++b) n += tiles_of(a, request(a, b));
    n = scan(n) - n;
    for (int b = b0; b < b1; ++b) {
        first[b] = a.p_first[b] = cap(n);
        n += tiles_of(a, request(a, b));
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
            const int c = tile_chunks(a, r, i - first[x]);
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

// Attention of requests with many query rows, bound by the matrix rate.
//
// A tile is 128 query rows of a kv head (a token's G heads beside each other), 32 a wave;
// its keys come in chunks of 64. As in attn_few_kernel the tiles' chunks are laid end to
// end and every workgroup takes an equal run, since causal tiles differ in length and a
// chunk of a long context has too few tiles for the GPU; prompt_combine_kernel merges tiles
// that lie in several runs.
//
// A chunk's codes are loaded by all threads (32 values each of K and of V at D = 128),
// two chunks ahead, expanded to the element type on the way to LDS, and then used as
// attn_tile_kernel uses its tiles: the second product of one block of 32 keys and the first
// product of the next but one around the softmax of the block between, one barrier a chunk.
// K and V have two buffers each: after the barrier of chunk w those of K(w) and V(w-1) are
// free for K(w+2) and V(w+1).
//
// 3 prompts of 77 .. 2111 queries behind 300 .. 8192 tokens, 16/4 heads of 128: 175 us (173
// GFLOP: 990 TFLOP/s; a library product of 8192 reaches 1180), and 206 in the first calls of a
// process. No unit is full: the matrix pipe is busy for 44 % of the clocks (at 2.25 GHz), the vector
// unit for 42, LDS for 42, a quarter of that in bank conflicts, which the stores of expanded tiles
// have (the same reads in attn_tile_kernel have none). Small batches are bound by a run's start:
// two tiles' loads and merges, 20 us.
//
// SELF: few tiles. Every workgroup adds up the tiles itself, as in attn_few_kernel, instead
// of a kernel before this one.
template <int D, class T, bool SELF>
__global__ void __launch_bounds__(256, 2) attn_prompt_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using W = Tile<D, T>;
    using x8 = typename W::x8;
    constexpr int RB = W::RB, NU = W::NU, BYTES = 64 * RB, NB32 = D / 32;
    __shared__ __attribute__((aligned(1024))) char ka[BYTES];
    __shared__ __attribute__((aligned(1024))) char kb[BYTES];
    __shared__ __attribute__((aligned(1024))) char va[BYTES];
    __shared__ __attribute__((aligned(1024))) char vb[BYTES];
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

    __shared__ int first_s[SELF ? kSelfRequests + 1 : 1];
    __shared__ long long cost_s[SELF ? kSelfTiles + 1 : 1], sum_s[4];
    auto p_first = [&](int x) { return SELF ? first_s[x] : a.p_first[x]; };
    auto p_cost = [&](int x) { return SELF ? cost_s[x] : a.p_cost[x]; };
    if constexpr (SELF) {
        auto scan = [&](long long x) {  // inclusive, over the workgroup
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const long long y = __shfl_up(x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 63) sum_s[wave] = x;
            __syncthreads();
            for (int w = 0; w < wave; ++w) x += sum_s[w];
            return x;
        };
        const long long n = scan(tid < a.B ? tiles_of(a, request(a, tid)) : 0);
        first_s[tid + 1] = (int)min(n, (long long)a.p_tiles);
        if (tid == 0) first_s[0] = 0;
        __syncthreads();
        const int nt = first_s[a.B];
        constexpr int PER = kSelfTiles / 256;
        long long c[PER], sum = 0;
        int req[PER];
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int t = tid * PER + n;
            c[n] = req[n] = 0;
            if (t >= nt) continue;
            int lo = 0;
            for (int hi = a.B - 1; lo < hi;) {
                const int mid = (lo + hi + 1) / 2;
                if (first_s[mid] <= t)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            const int chunks = tile_chunks(a, request(a, lo), t - first_s[lo]);
            req[n] = lo;
            c[n] = chunks ? chunks + kPromptStart : 0;
            sum += c[n];
        }
        long long at = scan(sum) - sum;
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int t = tid * PER + n;
            if (t < nt) cost_s[t] = at;
            if (blockIdx.x == 0 && t < nt) {
                a.p_cost[t] = at;
                a.p_req[t] = req[n];
            }
            at += c[n];
        }
        if (tid == 255) cost_s[nt] = at;
        if (blockIdx.x == 0) {
            if (tid <= a.B) a.p_first[tid] = first_s[tid];
            if (tid == 0 && a.B == 256) a.p_first[256] = first_s[256];
            if (tid == 255) a.p_cost[nt] = at;
        }
        __syncthreads();
    }
    const int ntile = uni(p_first(a.B));
    const long long all = p_cost(ntile) * a.c.Hkv;
    const long long per = max(kPromptRun, (all + a.p_groups - 1) / a.p_groups);
    const int wg = (gridDim.x & 7) == 0 ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)
                                        : blockIdx.x;  // (consecutive runs on one XCD)
    long long u0 = wg * per;
    const long long hi = min(all, u0 + per);
    if (u0 >= hi) return;
    // The request, kv head and tile of unit u0.
    for (int x = tid; x < a.B; x += 256)
        if (p_cost(p_first(x)) * a.c.Hkv <= u0 && u0 < p_cost(p_first(x + 1)) * a.c.Hkv) found = x;
    __syncthreads();
    int b = uni(found);
    int t0 = uni(p_first(b)), t1 = uni(p_first(b + 1));
    long long base = p_cost(t0), each = p_cost(t1) - base;
    int hk = uni((int)((u0 - base * a.c.Hkv) / each));
    {
        const long long at = u0 - base * a.c.Hkv - hk * each;
        __syncthreads();
        for (int x = t0 + tid; x < t1; x += 256)
            if (p_cost(x) - base <= at && at < p_cost(x + 1) - base) found = x;
        __syncthreads();
    }
    int tile = uni(found);

    // Where this thread's values of a chunk lie: 16 bytes of codes and their scale.
    const bool d64v = D == 64 && tid >= 128;  // D = 64: half of the threads have K, half V
    const int part = D == 64 ? tid & 127 : tid;
    const int crow = part / NB32, cblk = part % NB32;
    const int coff = crow * (D / 2) + cblk * 16;
    const int csoff = (crow & 15) * (D / 8) + cblk * 4 + (crow >> 4);
    int kst[4], vst[4];  // their places in LDS
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        kst[n] = crow * RB + ((cblk * 4 + n) ^ kswz<NU>(crow & 31)) * 16;
        vst[n] = crow * RB + ((cblk * 4 + n) ^ vswz<NU>(crow & 31)) * 16;
    }

    while (u0 < hi) {
        while (u0 >= base * a.c.Hkv + hk * each + (p_cost(tile + 1) - base)) {
            if (++tile < t1) continue;  // (tiles without keys have no units)
            tile = t0;
            if (++hk < a.c.Hkv) continue;
            do {
                ++b;
                t0 = t1;
                t1 = uni(p_first(b + 1));
            } while (t0 == t1 || p_cost(t1) == p_cost(t0));
            base = p_cost(t0);
            each = p_cost(t1) - base;
            hk = 0;
            tile = t0;
        }
        const Request req = request(a, b);
        const int rt = tile - t0;
        const int end = uni(tile_end(a, req, rt)), chunks = (end + 63) / 64;
        const long long s = base * a.c.Hkv + hk * each + (p_cost(tile) - base);
        const int p0 = uni((int)(u0 - s)), p1 = uni((int)min((long long)chunks + kPromptStart, hi - s));
        u0 = s + p1;
        const int c0 = max(0, p0 - kPromptStart), c1 = p1 - kPromptStart;
        if (c1 <= 0) continue;
        const bool whole = c0 == 0 && c1 == chunks;
        const long long slot = 2LL * wg + (c0 == 0 ? 1 : 0);

        W w;
        w.init(lane);
        int lim[2];
        const long long rows = (long long)req.m * a.G;
        const unsigned neg = a.qsign < 0.f ? 0x80008000u : 0u;
        const long long row0 = (long long)rt * kTileRows + wave * 32;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const long long r = row0 + 16 * nb + i;
            const int tok = (int)(r / a.G), h = hk * a.G + (int)(r - (long long)tok * a.G);
            lim[nb] = r < rows ? seen_by(a, req, tok) : 0;
            const T* q = (const T*)a.q + (req.first + tok) * a.qt + h * a.qh + 8 * g;
#pragma unroll
            for (int n = 0; n < W::NQ; ++n) {
                u32x4 x = {};
                if (r < rows) x = *reinterpret_cast<const u32x4*>(q + 32 * n);
                w.qf[nb][n] = __builtin_bit_cast(x8, x ^ neg);
            }
        }
        const bool active = row0 < rows;  // (wave-uniform)
        const int all_see = active ? uni(seen_by(a, req, (int)(row0 / a.G))) : 0;

        const ConstInts table = (ConstInts)(a.table + b * a.table_stride);
        const int shift = a.c.page == 64 ? 0 : a.c.page == 128 ? 1 : 2;
        auto page_of = [&](int c) { return table[min(c, c1 - 1) >> shift]; };
        auto good = [&](int c, int page) { return c < c1 && (unsigned)page < (unsigned)a.c.pages; };
        auto row_of = [&](int c, int page) {
            const unsigned p = (unsigned)page < (unsigned)a.c.pages ? page : 0;
            return ((long long)p * a.c.Hkv + hk) * a.c.page + (min(c, c1 - 1) & ((1 << shift) - 1)) * 64;
        };
        // Codes of chunks kc (K) and vc (V), on their way to LDS.
        struct Raw {
            u32x4 kw, vw;
            unsigned ke, ve;
        };
        auto load = [&](int kc, int kpage, int vc, int vpage) __attribute__((always_inline)) {
            Raw r{};
            const long long kr = row_of(kc, kpage), vr = row_of(vc, vpage);
            if constexpr (D == 128) {
                r.kw = *reinterpret_cast<const u32x4*>(a.c.kc + kr * (D / 2) + coff);
                r.ke = a.c.ks[kr / 4 * (D / 8) + csoff];
                r.vw = *reinterpret_cast<const u32x4*>(a.c.vc + vr * (D / 2) + coff);
                r.ve = a.c.vs[vr / 4 * (D / 8) + csoff];
            } else {
                const long long row = d64v ? vr : kr;
                r.kw = *reinterpret_cast<const u32x4*>((d64v ? a.c.vc : a.c.kc) + row * (D / 2) + coff);
                r.ke = (d64v ? a.c.vs : a.c.ks)[row / 4 * (D / 8) + csoff];
            }
            return r;
        };
        auto put = [&](char* dst, const int (&at)[4], u32x4 x, unsigned e)
            __attribute__((always_inline)) {
            const float sc = e8m0(e);
#pragma unroll
            for (int n = 0; n < 4; ++n)
                *reinterpret_cast<GFX906_LDS x8*>((GFX906_LDS char*)dst + at[n]) = expand<T>(x[n], sc);
        };
        // V of chunk c is nothing behind the last key that the tile sees.
        auto clear = [&](u32x4& x, unsigned& e, int c, int page) __attribute__((always_inline)) {
            if (!good(c, page) || c * 64 + crow >= end) {
                x = u32x4{};
                e = 127;
            }
        };
        auto store = [&](char* kd, char* vd, int vc, int vpage, Raw& r) __attribute__((always_inline)) {
            if constexpr (D == 128) {
                put(kd, kst, r.kw, r.ke);
                clear(r.vw, r.ve, vc, vpage);
                put(vd, vst, r.vw, r.ve);
            } else if (!d64v) {
                put(kd, kst, r.kw, r.ke);
            } else {
                clear(r.kw, r.ke, vc, vpage);
                put(vd, vst, r.kw, r.ke);
            }
        };
        auto mask = [&](f32x4 (&S)[2][2], int c, int page, int half) __attribute__((always_inline)) {
            const int key0 = c * 64 + 32 * half;
            const bool ok = good(c, page);
            if (key0 + 32 <= all_see && ok) return;
            int lim2[2];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) lim2[nb] = ok ? lim[nb] : 0;
            w.mask(S, key0, lim2, g);
        };

        f32x4 Sa[2][2], Sb[2][2];
        x8 Pa[2], Pb[2];
        Pb[0] = x8{};
        Pb[1] = x8{};
        int g0 = page_of(c0), g1 = page_of(c0 + 1), g2 = page_of(c0 + 2), g3 = page_of(c0 + 3);
        __syncthreads();  // (the tile before: every wave is done with LDS)
        Raw raw0 = load(c0, g0, c0, g0), raw1 = load(c0 + 1, g1, c0, g0);
        Raw raw = load(c0 + 2, g2, c0 + 1, g1);
        store(ka, va, c0, g0, raw0);
        if (D == 128 || !d64v) put(kb, kst, raw1.kw, raw1.ke);
        for (int z = tid; z < BYTES / 16; z += 256) *reinterpret_cast<u32x4*>(vb + 16 * z) = u32x4{};
        __syncthreads();
        if (active) w.qk(ka, Sa);

        auto step = [&](int c, const char* vp, char* kc, char* vc, const char* kn)
            __attribute__((always_inline)) {
            if (active) {
                mask(Sa, c, g0, 0);
                w.turn(vp + 32 * RB, Pb, kc + 32 * RB, Sb, Sa, Pa, a.scale);
            }
            lds_barrier();
            // V(c+1) goes where V(c-1) was, K(c+2) where K(c) was.
            store(kc, const_cast<char*>(vp), c + 1, g1, raw);
            raw = load(c + 3, g3, c + 2, g2);
            if (active) {
                mask(Sb, c, g0, 1);
                w.turn(vc, Pa, kn, Sa, Sb, Pb, a.scale);
            }
            g0 = g1;
            g1 = g2;
            g2 = g3;
            g3 = page_of(c + 4);
        };
        int c = c0;
        for (; c < c1; c += 2) {
            step(c, vb, ka, va, kb);
            step(c + 1, va, kb, vb, ka);
        }
        if (active) w.pv(vb + 32 * RB, Pb);

#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const long long r = row0 + 16 * nb + i;
            const float l = quad_sum(w.lacc[nb][0]);
            if (r >= rows) continue;
            const long long at = slot * kTileRows + wave * 32 + 16 * nb + i;
            if (!whole) {
#pragma unroll
                for (int ob = 0; ob < W::NO; ++ob)
                    *reinterpret_cast<f32x4*>(a.p_o + at * D + 16 * ob + 4 * g) = w.oacc[ob][nb];
                if (g == 0) *reinterpret_cast<f32x2*>(a.p_ml + at * 2) = f32x2{w.m[nb], l};
                continue;
            }
            const int tok = (int)(r / a.G), h = hk * a.G + (int)(r - (long long)tok * a.G);
            T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + 4 * g;
            const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
            for (int ob = 0; ob < W::NO; ++ob) {
                const f32x4 x = w.oacc[ob][nb] * inv;
                const auto x0 = Elem<T>::cvt2(x[0], x[1]), x1 = Elem<T>::cvt2(x[2], x[3]);
                *reinterpret_cast<u32x2*>(o + 16 * ob) =
                    u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
            }
        }
    }
#endif
}

// Merges the runs of a tile, writes the zeros of tiles that see no key, and does rows
// again that a value they do not see may have spoilt. One workgroup per 16 rows
// of a tile and kv head; behind these one per request and query row of attn_few_kernel's. (4 requests
// of 1 .. 70 queries in 1000 .. 20000 tokens, 32/8 heads: 87 us, and 96 with two merges one after the
// other; 16 of 1 .. 300 in 300 .. 4000, 16/4 heads: 86 and 90.)
template <int D, class T>
__global__ void __launch_bounds__(256) prompt_combine_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int ROWS = 16;
    const int tile = blockIdx.x / (kTileRows / ROWS), hk = blockIdx.y, tid = threadIdx.x;
    if (tile >= a.p_tiles) {
        const int e = blockIdx.x - a.p_tiles * (kTileRows / ROWS), few = e / kFewRows;
        few_combine<D, T, 2, 256>(a, few, hk, e - few * kFewRows);
        return;
    }
    const int r0 = blockIdx.x % (kTileRows / ROWS) * ROWS;
    const int b = a.p_req[tile];
    if (tile >= a.p_first[a.B]) return;
    const int t0 = a.p_first[b], t1 = a.p_first[b + 1], rt = tile - t0;
    const Request req = request(a, b);
    const int rows = (int)min(r0 + (long long)ROWS, (long long)req.m * a.G - (long long)rt * kTileRows);
    if (r0 >= rows) return;
    auto tok_of = [&](int r) { return (int)(((long long)rt * kTileRows + r) / a.G); };
    auto head_of = [&](int r, int tok) {
        return hk * a.G + (int)((long long)rt * kTileRows + r - (long long)tok * a.G);
    };
    const int end = tile_end(a, req, rt), chunks = (end + 63) / 64;
    int w0 = 0, w1 = 0;
    if (chunks) {
        const long long all = a.p_cost[a.p_first[a.B]] * a.c.Hkv;
        const long long per = max(kPromptRun, (all + a.p_groups - 1) / a.p_groups);
        const long long base = a.p_cost[t0], each = a.p_cost[t1] - base;
        const long long s = base * a.c.Hkv + hk * each + (a.p_cost[tile] - base) + kPromptStart;
        w0 = (int)(s / per);
        w1 = (int)((s + chunks - 1) / per);
    }
    if (!chunks || w0 != w1) {
        for (int e = tid; e < (rows - r0) * (D / 4); e += 256) {
            const int r = r0 + e / (D / 4), d = e % (D / 4) * 4, tok = tok_of(r);
            float m = kNoMax, l = 0.f;
            f32x4 acc = {};
            constexpr int U = 4;
            for (int x = w0; chunks && x <= w1; x += U) {
                f32x2 ml[U];
                f32x4 p[U];
#pragma unroll
                for (int n = 0; n < U; ++n) {
                    const int y = min(x + n, w1);
                    const long long at = (2LL * y + (y == w0 ? 1 : 0)) * kTileRows + r;
                    ml[n] = *reinterpret_cast<const f32x2*>(a.p_ml + at * 2);
                    p[n] = *reinterpret_cast<const f32x4*>(a.p_o + at * D + d);
                }
#pragma unroll
                for (int n = 0; n < U; ++n) {
                    if (x + n > w1) continue;
                    const float mn = max2(m, ml[n][0]);
                    const float f = __builtin_amdgcn_exp2f(m - mn);
                    const float e = __builtin_amdgcn_exp2f(ml[n][0] - mn);
                    acc = acc * f + p[n] * e;
                    l = l * f + ml[n][1] * e;
                    m = mn;
                }
            }
            acc *= l != 0.f ? 1.f / l : 0.f;
            T* o = (T*)a.o + (req.first + tok) * a.ot + head_of(r, tok) * a.oh + d;
            const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
            *reinterpret_cast<u32x2*>(o) =
                u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
        }
    }
    const int see0 = seen_by(a, req, tok_of(r0));
    if (see0 < end && may_spoil<D, T>(a, b, hk, see0, end)) {  // (the same for every wave)
        __syncthreads();
        for (int r = r0 + (tid >> 6); r < rows; r += 4) {
            const int tok = tok_of(r), see = seen_by(a, req, tok), h = head_of(r, tok);
            if (may_spoil<D, T>(a, b, hk, see, end))
                attend_row<D, T>(a, (const T*)a.q + (req.first + tok) * a.qt + h * a.qh, hk, b, 0, see,
                                 (T*)a.o + (req.first + tok) * a.ot + h * a.oh);
        }
    }
#endif
}

// -- host -----------------------------------------------------------------------------

int check_cache(int Hkv, int D, int pages, int page, const void* kc, const void* ks,
                const void* vc, const void* vs, const char* who) {
    if (D != 64 && D != 128) return g_err.fail("%s: head dim must be 64 or 128", who);
    if (page != 64 && page != 128 && page != 256)
        return g_err.fail("%s: pages hold 64, 128 or 256 tokens", who);
    if (Hkv <= 0 || Hkv > 65535) return g_err.fail("%s: bad number of kv heads", who);
    if (pages < 0 || (long long)pages * page >= (1LL << 31))
        return g_err.fail("%s: the cache must hold fewer than 2^31 tokens", who);
    if (pages > 0 && (!kc || !ks || !vc || !vs)) return g_err.fail("%s: null cache", who);
    if (!aligned(kc, 16) || !aligned(vc, 16) || !aligned(ks, 4) || !aligned(vs, 4))
        return g_err.fail("%s: codes must be 16-byte and scales 4-byte aligned", who);
    return 0;
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
FewPlan few_plan(int B, int G, int Hkv, int D, int max_q, int max_len) {
    FewPlan p{};
    const long long rows = std::min<long long>((long long)max_q * G, kFewRows);
    p.nb = rows > 16 ? 2 : 1;
    p.tiles = (int)((rows + 16 * p.nb - 1) / (16 * p.nb));
    const long long segs = (long long)B * Hkv * p.tiles;
    // (a unit of 32 rows takes about as long as two of 16. 32 requests of 100 .. 16384 tokens,
    // one query each: 36.1 us with 8 units, 28.8 with 16, 30.5 with 24; 131072 tokens with 32
    // rows: 22.5 with 8, 24.0 with 16)
    p.start = p.nb == 1 ? 16 : 8;
    p.units = segs * ((std::max(max_len, 1) + 63LL) / 64 + p.start);
    p.direct = max_len <= (segs >= kDirectHeads ? 2 : 1) * kDirectTokens && segs < (1LL << 31);
    if (p.direct) return p;
    // A workgroup a CU, with a unit a wave at least. (Three of four waves, with 8 units for a
    // start: 32 ragged requests 29.3 us and not 28.8, 32 of 4000 tokens 33.5 and not 30.)
    p.groups = (int)std::max(1LL, std::min<long long>(kGroups, p.units / (kMinUnits + p.start) + 1));
    p.many = p.groups / segs >= 32;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.o_off = up((size_t)(B + 1) * sizeof(int));
    p.ml_off = p.o_off + (size_t)2 * p.groups * 16 * p.nb * D * sizeof(float);
    p.bytes = p.ml_off + (size_t)2 * p.groups * 16 * p.nb * 2 * sizeof(float);
    return p;
}

// How attn_prompt_kernel is launched, and its part of the workspace behind the few
// rows' one. tiles: the most there can be of T queries.
struct PromptPlan {
    bool used;
    int groups, tiles;
    bool self;
    size_t cost_off, req_off, o_off, ml_off, bytes;
};
PromptPlan prompt_plan(int T, int B, int G, int D, int max_q, size_t after) {
    PromptPlan p{};
    p.used = (long long)max_q * G > kFewRows;
    if (!p.used) return p;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.groups = 512;  // two a CU
    p.tiles = (int)std::min<long long>((long long)T * G / kTileRows + B, (1LL << 27));
    p.cost_off = up(after) + up((size_t)(B + 1) * sizeof(int));
    p.self = p.tiles <= kSelfTiles && B <= kSelfRequests;
    p.req_off = p.cost_off + up((size_t)(p.tiles + 1) * sizeof(long long));
    p.o_off = p.req_off + up((size_t)p.tiles * sizeof(int));
    p.ml_off = p.o_off + (size_t)2 * p.groups * kTileRows * D * sizeof(float);
    p.bytes = p.ml_off + (size_t)2 * p.groups * kTileRows * 2 * sizeof(float);
    return p;
}

}  // namespace

extern "C" const char* kv4_last_error(void) { return g_err.get(); }

extern "C" int kv4_plan_pages(const int* lens, const int* new_lens, int* table,
                              long long table_stride, int W, const int* free_pages, int n_free,
                              const int* used, int B, int page, int n_slots, int* slots,
                              int* cu_new, int* lens_out, int* used_out, int* missing,
                              hipStream_t stream) {
    g_err.text[0] = 0;
    if (page != 64 && page != 128 && page != 256)
        return g_err.fail("kv4_plan_pages: pages hold 64, 128 or 256 tokens");
    if (B < 0 || B > kMaxRequests)
        return g_err.fail("kv4_plan_pages: at most %d requests", kMaxRequests);
    if (W < 0 || n_free < 0 || n_slots < 0 || (B > 1 && table_stride < W))
        return g_err.fail("kv4_plan_pages: negative sizes or overlapping table rows");
    if ((B > 0 && (!lens || !new_lens || !lens_out)) || (B > 0 && W > 0 && !table) ||
        (n_free > 0 && !free_pages) || !used || (n_slots > 0 && !slots) || !cu_new || !used_out ||
        !missing)
        return g_err.fail("kv4_plan_pages: null argument");
    const PlanArgs a{lens,  new_lens, table,    table_stride, free_pages, used, slots, cu_new,
                     lens_out, used_out, missing, W, n_free, B, page, n_slots};
    const long long work = std::max<long long>(n_slots, (long long)B * 16);
    const int grid = (int)std::min<long long>(256, std::max<long long>(1, (work + 255) / 256));
    hipLaunchKernelGGL(plan_pages_kernel, dim3(grid), dim3(256), 0, stream, a);
    return g_err.launched("kv4_plan_pages", hipGetLastError());
}

extern "C" int kv4_store(const void* k, const void* v, const long long* k_strides,
                         const long long* v_strides, int dtype, int T, int Hkv, int D,
                         const int* slots, void* k_codes, void* k_scales, void* v_codes,
                         void* v_scales, int pages, int page, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, "kv4_store")) return 1;
    if (dtype != KV4_DTYPE_F16 && dtype != KV4_DTYPE_BF16) return g_err.fail("kv4_store: bad dtype");
    if (T < 0) return g_err.fail("kv4_store: negative token count");
    if (T == 0 || pages == 0) return 0;
    if (!k || !v || !slots || !k_strides || !v_strides)
        return g_err.fail("kv4_store: null argument");
    for (int i = 0; i < 2; ++i)
        if (k_strides[i] < 0 || v_strides[i] < 0 || k_strides[i] % 8 || v_strides[i] % 8)
            return g_err.fail("kv4_store: strides must be non-negative multiples of 8 elements");
    if (!aligned(k, 16) || !aligned(v, 16))
        return g_err.fail("kv4_store: k and v must be 16-byte aligned");
    RowArgs a{};
    a.k = k;
    a.v = v;
    a.kt = k_strides[0];
    a.kh = k_strides[1];
    a.vt = v_strides[0];
    a.vh = v_strides[1];
    a.slots = slots;
    a.c = Cache{(const uint8_t*)k_codes, (const uint8_t*)k_scales, (const uint8_t*)v_codes,
                (const uint8_t*)v_scales, pages, page, Hkv, D};
    const long long n = (long long)T * Hkv * (D / 32);
    if (n >= (1LL << 31)) return g_err.fail("kv4_store: too many rows");
    a.n = (unsigned)n;
    const dim3 grid((unsigned)((n + 255) / 256), 2);
    if (dtype == KV4_DTYPE_F16)
        hipLaunchKernelGGL(store_kernel<f16>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(store_kernel<bf16>, grid, dim3(256), 0, stream, a);
    return g_err.launched("kv4_store", hipGetLastError());
}

extern "C" int kv4_load(void* k, void* v, int dtype, int T, int Hkv, int D, const int* slots,
                        const void* k_codes, const void* k_scales, const void* v_codes,
                        const void* v_scales, int pages, int page, hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, "kv4_load")) return 1;
    if (dtype != KV4_DTYPE_F16 && dtype != KV4_DTYPE_BF16) return g_err.fail("kv4_load: bad dtype");
    if (T < 0) return g_err.fail("kv4_load: negative token count");
    if (T == 0) return 0;
    if (!k || !v || !slots) return g_err.fail("kv4_load: null argument");
    if (!aligned(k, 16) || !aligned(v, 16))
        return g_err.fail("kv4_load: k and v must be 16-byte aligned");
    RowArgs a{};
    a.ko = k;
    a.vo = v;
    a.slots = slots;
    a.c = Cache{(const uint8_t*)k_codes, (const uint8_t*)k_scales, (const uint8_t*)v_codes,
                (const uint8_t*)v_scales, pages, page, Hkv, D};
    const long long n = (long long)T * Hkv * (D / 8);
    if (n >= (1LL << 31)) return g_err.fail("kv4_load: too many rows");
    a.n = (unsigned)n;
    const dim3 grid((unsigned)((n + 255) / 256), 2);
    if (dtype == KV4_DTYPE_F16)
        hipLaunchKernelGGL(load_kernel<f16>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(load_kernel<bf16>, grid, dim3(256), 0, stream, a);
    return g_err.launched("kv4_load", hipGetLastError());
}

extern "C" size_t kv4_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int D, int max_q,
                                           int max_len) {
    if (T <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || D <= 0 || max_q <= 0) return 0;
    const size_t few = few_plan(B, Hq / Hkv, Hkv, D, std::min(max_q, T), max_len).bytes;
    const PromptPlan p = prompt_plan(T, B, Hq / Hkv, D, std::min(max_q, T), few);
    return p.used ? p.bytes : few;
}

extern "C" int kv4_attn(const void* q, void* o, const long long* q_strides,
                        const long long* o_strides, int dtype, int T, int B, int Hq, int Hkv, int D,
                        const void* k_codes, const void* k_scales, const void* v_codes,
                        const void* v_scales, int pages, int page, const int* table,
                        long long table_stride, int W, const int* lens, const int* cu_q, int max_q,
                        float scale, int causal, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
    g_err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, "kv4_attn")) return 1;
    if (dtype != KV4_DTYPE_F16 && dtype != KV4_DTYPE_BF16) return g_err.fail("kv4_attn: bad dtype");
    if (T < 0 || B < 0 || W < 0 || max_q < 0) return g_err.fail("kv4_attn: negative sizes");
    if (B > kMaxRequests) return g_err.fail("kv4_attn: at most %d requests", kMaxRequests);
    if (Hq <= 0 || Hq % Hkv || Hq > 65535)
        return g_err.fail("kv4_attn: query heads must be a multiple of kv heads");
    if (!cu_q && T != B) return g_err.fail("kv4_attn: without cu_q, one query a request");
    if (T == 0 || B == 0 || max_q == 0) return 0;
    if (!q || !o || !q_strides || !o_strides || !lens || (W > 0 && !table))
        return g_err.fail("kv4_attn: null argument");
    if ((long long)W * page >= (1LL << 31) || table_stride < 0)
        return g_err.fail("kv4_attn: table too wide or a negative stride");
    for (int i = 0; i < 2; ++i)
        if (q_strides[i] < 0 || q_strides[i] % 8 || o_strides[i] < 0 || o_strides[i] % 4)
            return g_err.fail("kv4_attn: q strides must be non-negative multiples of 8, "
                              "o strides of 4");
    if (!aligned(q, 16) || !aligned(o, 8))
        return g_err.fail("kv4_attn: q must be 16-byte and o 8-byte aligned");
    if (q == o) return g_err.fail("kv4_attn: o must not be q");
    const long long oe[2] = {T, Hq};
    if (!rows_apart(o_strides, oe, 2, D)) return g_err.fail("kv4_attn: o's rows overlap");
    if (!good_scale(scale)) return g_err.fail("kv4_attn: scale must be finite, and below 2.3e38");
    const FewPlan plan = few_plan(B, Hq / Hkv, Hkv, D, cu_q ? std::min(max_q, T) : 1, W * page);
    if (plan.units >= (1LL << 30)) return g_err.fail("kv4_attn: table too wide for so many heads");
    const PromptPlan pp = prompt_plan(T, B, Hq / Hkv, D, cu_q ? std::min(max_q, T) : 1, plan.bytes);
    const size_t need = pp.used ? pp.bytes : plan.bytes;
    const long long heads = (long long)B * Hkv;
    const long long combines = pp.tiles * (long long)(kTileRows / 16) +
                               (plan.direct ? 0 : (long long)B * kFewRows);
    if (!(plan.direct ? launchable(heads * plan.tiles, 512)
                      : launchable(heads, plan.many ? 1024 : 256)) ||
        (pp.used && !launchable(combines, 256)))
        return g_err.fail("kv4_attn: too many requests, heads or query rows for one call");
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return g_err.fail("kv4_attn: workspace misaligned or smaller than "
                          "kv4_attn_workspace_bytes()");
    AttnArgs a{};
    a.q = q;
    a.o = o;
    a.qt = q_strides[0];
    a.qh = q_strides[1];
    a.ot = o_strides[0];
    a.oh = o_strides[1];
    a.c = Cache{(const uint8_t*)k_codes, (const uint8_t*)k_scales, (const uint8_t*)v_codes,
                (const uint8_t*)v_scales, pages, page, Hkv, D};
    a.table = table;
    a.table_stride = table_stride;
    a.lens = lens;
    a.cu = cu_q;
    a.W = W;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.G = Hq / Hkv;
    a.max_q = cu_q ? std::min(max_q, T) : 1;
    a.causal = causal;
    a.scale = log2_scale(scale);
    a.qsign = scale < 0.f ? -1.f : 1.f;
    a.few_rows = kFewRows;
    a.groups = plan.groups;
    a.min_units = kMinUnits + plan.start;
    a.start_units = plan.start;
    a.tiles = plan.tiles;
    a.starts = (int*)workspace;
    a.ws_o = (float*)((char*)workspace + plan.o_off);
    a.ws_ml = (float*)((char*)workspace + plan.ml_off);
    if (pp.used) {
        char* ws = (char*)workspace;
        a.p_groups = pp.groups;
        a.p_tiles = pp.tiles;
        a.p_first = (int*)(ws + ((plan.bytes + 255) & ~(size_t)255));
        a.p_cost = (long long*)(ws + pp.cost_off);
        a.p_req = (int*)(ws + pp.req_off);
        a.p_o = (float*)(ws + pp.o_off);
        a.p_ml = (float*)(ws + pp.ml_off);
    }
    const long long rows = (long long)a.max_q * a.G;
    const dim3 cgrid((unsigned)heads, (unsigned)std::min<long long>(rows, kFewRows));
    auto go = [&](auto d, auto t) {
        constexpr int kD = decltype(d)::value;
        using E = decltype(t);
        auto direct = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)(heads * plan.tiles)), dim3(512), 0, stream, a);
        };
        auto runs = [&](auto kernel, auto combine, auto combine_many) {
            hipLaunchKernelGGL(kernel, dim3(a.groups), dim3(512), 0, stream, a);
            if (pp.used) return;  // (prompt_combine_kernel merges)
            if (plan.many)
                hipLaunchKernelGGL(combine_many, cgrid, dim3(1024), 0, stream, a);
            else
                hipLaunchKernelGGL(combine, cgrid, dim3(256), 0, stream, a);
        };
        if (plan.direct && plan.nb == 1)
            direct(attn_few_kernel<kD, E, 1, true>);
        else if (plan.direct)
            direct(attn_few_kernel<kD, E, 2, true>);
        else if (plan.nb == 1)
            runs(attn_few_kernel<kD, E, 1, false>, few_combine_kernel<kD, E, 1, 256>,
                 few_combine_kernel<kD, E, 1, 1024>);
        else
            runs(attn_few_kernel<kD, E, 2, false>, few_combine_kernel<kD, E, 2, 256>,
                 few_combine_kernel<kD, E, 2, 1024>);
        if (pp.used) {
            if (pp.self) {
                hipLaunchKernelGGL((attn_prompt_kernel<kD, E, true>), dim3(pp.groups), dim3(256), 0,
                                   stream, a);
            } else {
                hipLaunchKernelGGL(prompt_plan_kernel, dim3(1), dim3(1024), 0, stream, a);
                hipLaunchKernelGGL((attn_prompt_kernel<kD, E, false>), dim3(pp.groups), dim3(256), 0,
                                   stream, a);
            }
            hipLaunchKernelGGL((prompt_combine_kernel<kD, E>), dim3((unsigned)combines, Hkv),
                               dim3(256), 0, stream, a);
        }
    };
    if (dtype == KV4_DTYPE_F16)
        D == 64 ? go(std::integral_constant<int, 64>{}, f16{})
                : go(std::integral_constant<int, 128>{}, f16{});
    else
        D == 64 ? go(std::integral_constant<int, 64>{}, bf16{})
                : go(std::integral_constant<int, 128>{}, bf16{});
    return g_err.launched("kv4_attn", hipGetLastError());
}
