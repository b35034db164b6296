// Key/value cache in 8 bits for AMD MI355X (gfx950): storing and reading rows, the attention
// weights of its blocks and eviction by them. The format and the entry points are
// described in gfx906_amd_attn.h; the attention is in kv8_attn_kernel.hip.
//
// gfx950 converts between pairs of E4M3 codes and fp16, bf16 or fp32 with a power-of-two
// scale in one instruction (v_cvt_scalef32_*), rounding to nearest even.
#include "kv8.h"

#include <algorithm>
#include <type_traits>

#include "longctx_tile.h"
#include "paged.h"

namespace gfx906_amd {
namespace kv8 {
LastError& last_error() {
    static thread_local LastError e;
    return e;
}
}  // namespace kv8
}  // namespace gfx906_amd

namespace {

using namespace gfx906_amd::kv8;

#if defined(__HIP_DEVICE_COMPILE__)
// Exponents of scales.
constexpr int kLow = -15, kHigh = 7;
__device__ __forceinline__ float scale_of(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// Exponent of the least scale for rows whose largest |x| has the bits `top` (of fp32): 448 is
// 1.75 * 2^8, so mantissas past 0.75 take the next one.
__device__ __forceinline__ int exponent_for(unsigned top) {
    return min(kHigh, max(kLow, (int)((top + 0x1fffffu) >> 23) - 135));
}

// A pair of numbers as E4M3 codes in the low or high half of w.
template <class T, bool HIGH>
__device__ __forceinline__ unsigned pack2(unsigned w, unsigned pair, float s) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const s16x2 old = __builtin_bit_cast(s16x2, w);
    if constexpr (__is_same(T, f16))
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(
                                                old, __builtin_bit_cast(f16x2, pair), s, HIGH));
    else
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
                                                old, __builtin_bit_cast(bf16x2, pair), s, HIGH));
}
template <class T>
__device__ __forceinline__ unsigned pack4(unsigned a, unsigned b, float s) {
    return pack2<T, true>(pack2<T, false>(0, a, s), b, s);
}
// Four codes at scale `from` as codes at scale `to`: exact, but where they become subnormal.
__device__ __forceinline__ unsigned rescale(unsigned w, float from, float to) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, from, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, from, true);
    s16x2 r = {};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a[0], a[1], to, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, b[0], b[1], to, true);
    return __builtin_bit_cast(unsigned, r);
}

// Patterns of the element type: infinity, NaN, and 57344, the largest number held.
template <class T>
constexpr unsigned kInf16 = __is_same(T, f16) ? 0x7c00u : 0x7f80u;
template <class T>
constexpr unsigned kNan16 = __is_same(T, f16) ? 0x7e00u : 0x7fc0u;
template <class T>
constexpr unsigned kMax16 = __is_same(T, f16) ? 0x7b00u : 0x4760u;

// Larger |x| of both numbers of each dword, patterns compared as integers.
__device__ __forceinline__ unsigned top2(unsigned m, unsigned w) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned,
                              __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                        __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
__device__ __forceinline__ unsigned wave_top(unsigned m) {
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
    return m;
}
// Infinite and NaN numbers as NaN, others at most 57344 in size; m: the larger of m and the
// finite ones.
template <class T>
__device__ __forceinline__ unsigned tame(unsigned w, unsigned& m) {
    unsigned out = 0, mags = 0;
#pragma unroll
    for (int sh = 0; sh < 32; sh += 16) {
        const unsigned x = w >> sh & 0xffffu, a = x & 0x7fffu;
        const bool bad = a >= kInf16<T>;
        const unsigned b = bad ? kNan16<T> : min(a, kMax16<T>);
        out |= ((x & 0x8000u) | b) << sh;
        mags |= (bad ? 0u : b) << sh;
    }
    m = top2(m, mags);
    return out;
}
template <class T>
__device__ __forceinline__ unsigned f32_bits(unsigned x16) {
    if constexpr (__is_same(T, f16))
        return __float_as_uint((float)__builtin_bit_cast(f16, (unsigned short)x16));
    else
        return x16 << 16;
}
#endif

// -- storing and reading rows ---------------------------------------------------------

struct StoreArgs {
    const void* k;
    const void* v;
    long long kt, kh, vt, vh;  // strides: token, head
    Cache c;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* cu;
    float* weights;
    int W, T, B, max_q, causal;
    unsigned tasks;  // blocks that may be written, of one head
};

// A wave has a block of a request that gets rows, of one kv head, of K or V: it is the only
// one to touch it, so the block's maximum, its scale and its older codes need no exchange
// between waves. Request b's blocks have the numbers from cu[b] / 64 + 2b on (n rows touch at
// most n / 64 + 2 blocks), where a wave finds its request by two steps of 64.
//
// A lane has 8 dims of every row group's tokens (D / 8 of them): the 16 or 8 tokens whose codes lie
// side by side in V, so that V is written in 16 or 8 bytes without an exchange. Up to four rows
// (a decoding step) are written as they are where the scale stays, a dword of dims a lane.
//
// Bound by bytes: 8 prompts of 500 .. 4096 rows, 16 heads of 128, 36 us (4.9 TB/s; some 8 more without the
// loads past the caches).
template <class T, int D>
__global__ void __launch_bounds__(256) store_kernel(const StoreArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int DL = D / 8, NT = D / 8;  // lanes a row; tokens a lane
    const int lane = threadIdx.x & 63;
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const unsigned id = uni(blockIdx.x * 4 + (threadIdx.x >> 6));
    const bool is_v = id & 1;
    const unsigned task = (id >> 1) / (unsigned)a.c.Hkv;
    const int h = uni((int)((id >> 1) - task * a.c.Hkv));
    if (task >= a.tasks) return;
    // The last request whose first number is at most `task`: one load of each lane's request up to 64
    // of them, else two steps of 64.
    auto first_of = [&](int x) { return (unsigned)((cu_at(a, x) >> 6) + 2 * x); };
    Request r;
    unsigned first;
    int b;
    if (a.B <= 64) {
        Request mine{};
        first = ~0u;
        if (lane < a.B) {
            mine = request(a, lane);
            first = (unsigned)((mine.first >> 6) + 2 * lane);
        }
        b = uni(max(0, __popcll(__ballot(first <= task)) - 1));
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, b); };
        r.first = of(mine.first);
        r.n = of(mine.n);
        r.len = of((int)mine.len);  // (an int is where it comes from)
        first = (unsigned)of((int)first);
    } else {
        auto starts = [&](int x) { return x < a.B && first_of(x) <= task; };
        const int step = (a.B + 63) / 64;
        b = uni(max(0, __popcll(__ballot(starts(lane * step))) - 1)) * step;
        b += uni(max(0, __popcll(__ballot(lane < step && starts(b + lane))) - 1));
        r = request(a, b);
        first = first_of(b);
    }
    const long long old = r.len - r.n;  // tokens before the new ones (negative: rows too many)
    const long long j = max(0LL, old) / kBlock + (task - first);
    const long long p0 = max(old, j * kBlock), p1 = min(r.len, (j + 1) * kBlock);
    if (p0 >= p1 || j * kBlock >= (long long)a.W * a.c.page) return;
    const int before = uni((int)(p0 - j * kBlock)), count = uni((int)(p1 - p0));
    const long long row0 = r.first + (p0 - old) - before;  // row of the block's token 0
    const T* src = is_v ? (const T*)a.v + h * a.vh : (const T*)a.k + h * a.kh;
    const long long st = is_v ? a.vt : a.kt;
    constexpr int FEW = 4;
    unsigned few[FEW] = {};  // (on their way while the page is looked up)
    if (count <= FEW) {
#pragma unroll
        for (int n = 0; n < FEW; ++n)
            if (n < count && 2 * lane < D)
                few[n] = *reinterpret_cast<const unsigned*>(src + (row0 + before + n) * st + 2 * lane);
    }
    const int page = ((ConstInts)(a.table + b * a.table_stride))[j * kBlock / a.c.page];
    if ((unsigned)page >= (unsigned)a.c.pages) return;
    const long long blk = block_at(a.c, page, h, (int)(j % (a.c.page / kBlock)));
    uint8_t* codes = const_cast<uint8_t*>(is_v ? a.c.vc : a.c.kc) + blk * (kBlock * D);
    float* scale = const_cast<float*>(is_v ? a.c.vs : a.c.ks) + blk;
    const int old_e =
        before ? min(kHigh, max(kLow, (int)(__float_as_uint(*scale) >> 23 & 255) - 127)) : kLow;
    if (!is_v && a.weights && before == 0 && lane == 0) a.weights[blk] = 0.f;

    if (count <= FEW) {
        unsigned m = 0;
#pragma unroll
        for (int n = 0; n < FEW; ++n) m = top2(m, few[n]);
        m = wave_top(m);
        if (m > kMax16<T>) {
            m = 0;
#pragma unroll
            for (int n = 0; n < FEW; ++n) few[n] = tame<T>(few[n], m);
            m = wave_top(m);
        }
        const int e = max(old_e, exponent_for(f32_bits<T>(m)));
        if (before == 0 || e == old_e) {
            const float s = scale_of(e);
            if (before == 0 && lane == 0) *scale = s;
#pragma unroll
            for (int n = 0; n < FEW; ++n) {
                if (n >= count || 2 * lane >= D) continue;
                const unsigned w = pack2<T, false>(0, few[n], s);
                const int t = before + n;
                if (is_v) {
                    codes[2 * lane * kBlock + place(t)] = (uint8_t)w;
                    codes[(2 * lane + 1) * kBlock + place(t)] = (uint8_t)(w >> 8);
                } else {
                    *reinterpret_cast<unsigned short*>(codes + t * D + 2 * lane) = (unsigned short)w;
                }
            }
            return;
        }
    }

    const int dl = lane % DL, sub = lane / DL;
    auto token = [&](int n) {
        return D == 128 ? 16 * (n >> 2) + 4 * sub + (n & 3)
                        : 32 * (sub >> 2) + 16 * (n >> 2) + 4 * (sub & 3) + (n & 3);
    };
    auto is_new = [&](int t) { return t >= before && t < before + count; };
    u32x4 x[NT];
    unsigned m = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int t = token(n);
        x[n] = u32x4{};
        // (read once: past the lines that the codes are written to)
        if (is_new(t))
            x[n] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4*>(src + (row0 + t) * st + 8 * dl));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = top2(m, x[n][i]);
    m = wave_top(m);
    if (m > kMax16<T>) {
        m = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n][i] = tame<T>(x[n][i], m);
        m = wave_top(m);
    }
    const int e = max(old_e, exponent_for(f32_bits<T>(m)));
    const float s = scale_of(e), old_s = scale_of(old_e);
    const bool grown = before && e > old_e;
    if ((grown || !before) && lane == 0) *scale = s;
    if (!is_v) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int t = token(n);
            u32x2* dst = reinterpret_cast<u32x2*>(codes + t * D + 8 * dl);
            if (is_new(t)) {
                *dst = u32x2{pack4<T>(x[n][0], x[n][1], s), pack4<T>(x[n][2], x[n][3], s)};
            } else if (grown && t < before) {
                const u32x2 w = *dst;
                *dst = u32x2{rescale(w[0], old_s, s), rescale(w[1], old_s, s)};
            }
        }
        return;
    }
    unsigned mask[NT / 4];  // bytes of new tokens
#pragma unroll
    for (int q = 0; q < NT / 4; ++q) {
        mask[q] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mask[q] |= is_new(token(4 * q + i)) ? 255u << (8 * i) : 0u;
    }
    uint8_t* row = codes + 8 * dl * kBlock + place(token(0));
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        unsigned w[NT / 4];
#pragma unroll
        for (int q = 0; q < NT / 4; ++q) {
            // dim d of four tokens, two and two
            auto pair = [&](int n) {
                return __builtin_amdgcn_perm(x[n + 1][d / 2], x[n][d / 2],
                                             d & 1 ? 0x07060302u : 0x05040100u);
            };
            w[q] = pack4<T>(pair(4 * q), pair(4 * q + 2), s);
        }
        if (before) {
#pragma unroll
            for (int q = 0; q < NT / 4; ++q) {
                unsigned o = *reinterpret_cast<const unsigned*>(row + d * kBlock + 4 * q);
                if (grown) o = rescale(o, old_s, s);
                w[q] = (o & ~mask[q]) | (w[q] & mask[q]);
            }
        }
        if constexpr (NT == 16)
            *reinterpret_cast<u32x4*>(row + d * kBlock) = u32x4{w[0], w[1], w[2], w[3]};
        else
            *reinterpret_cast<u32x2*>(row + d * kBlock) = u32x2{w[0], w[1]};
    }
#endif
}

struct LoadArgs {
    void* k;
    void* v;
    const int* slots;
    Cache c;
    int T;
};

// 64 rows of a head a workgroup, 8 dims a lane. Of V a row is D bytes in as many lines, so the
// blocks that the rows lie in are read whole, one after the other, and the rows picked from
// LDS. 15081 rows of 16 heads of 128, 36 to 40 us (73 with a byte of V a load). grid: rows / 64, heads x (K, V).
template <class T, int D>
__global__ void __launch_bounds__(256) load_kernel(const LoadArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using x8 = typename Elem<T>::x8;
    constexpr int DL = D / 8, RW = 256 / DL, PITCH = kBlock + 4;
    __shared__ __attribute__((aligned(16))) unsigned char vb[D * PITCH];  // (written as dwords)
    const int h = blockIdx.y >> 1, dl = threadIdx.x % DL, lane = threadIdx.x & 63;
    const bool is_v = blockIdx.y & 1;
    const long long t0 = blockIdx.x * 64LL;
    x8* const out = reinterpret_cast<x8*>(is_v ? a.v : a.k);
    const int mine = t0 + lane < a.T ? a.slots[t0 + lane] : -1;  // (every wave has all 64)
    const int part = a.c.page / kBlock;
    // Number of the row's block among those of a head, -1 outside the cache.
    const int block = mine >= 0 && mine < a.c.pages * (long long)a.c.page ? mine / kBlock : -1;
    auto where = [&](int blk) { return block_at(a.c, blk / part, h, blk % part); };
    auto put = [&](long long t, unsigned lo, unsigned hi, float s) {
        out[(t * a.c.Hkv + h) * DL + dl] = expand<T>(lo, hi, s);
    };
#pragma unroll
    for (int n = 0; n < 64 / RW; ++n) {
        const int r = n * RW + threadIdx.x / DL, blk = __shfl(block, r), slot = __shfl(mine, r);
        if (t0 + r >= a.T) continue;
        if (blk < 0) {
            put(t0 + r, 0, 0, 1.f);
        } else if (!is_v) {
            const long long at = where(blk);
            const u32x2 x = *reinterpret_cast<const u32x2*>(a.c.kc + at * (kBlock * D) +
                                                            slot % kBlock * D + 8 * dl);
            put(t0 + r, x[0], x[1], a.c.ks[at]);
        }
    }
    if (!is_v) return;
    // (the next block's codes are on their way while rows are picked from one)
    unsigned long long left = __ballot(block >= 0);
    if (!left) return;
    u32x4 x[D / 64];
    float s = 0.f;
    int blk = 0;
    auto fetch = [&] {
        blk = __builtin_amdgcn_readfirstlane(__shfl(block, (int)__ffsll(left) - 1));
        const long long at = where(blk);
        s = a.c.vs[at];
#pragma unroll
        for (int n = 0; n < D / 64; ++n)
            x[n] = *reinterpret_cast<const u32x4*>(a.c.vc + at * (kBlock * D) + 4096 * n + 16 * threadIdx.x);
    };
    fetch();
    while (true) {
        const unsigned long long same = __ballot(block == blk);
        const float unit = s;
        left &= ~same;
        lds_barrier();  // (the block before has been read)
#pragma unroll
        for (int n = 0; n < D / 64; ++n) {
            unsigned* p = reinterpret_cast<unsigned*>(vb + (64 * n + threadIdx.x / 4) * PITCH +
                                                      16 * (threadIdx.x & 3));
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = x[n][e];
        }
        if (left) fetch();
        lds_barrier();
#pragma unroll
        for (int n = 0; n < 64 / RW; ++n) {
            const int r = n * RW + threadIdx.x / DL, slot = __shfl(mine, r);
            if (!(same >> r & 1)) continue;
            const unsigned char* p = vb + 8 * dl * PITCH + place(slot % kBlock);
            unsigned w[2] = {};
#pragma unroll
            for (int d = 0; d < 8; ++d) w[d / 4] |= (unsigned)p[d * PITCH] << (8 * (d & 3));
            put(t0 + r, w[0], w[1], unit);
        }
        if (!left) return;
    }
#endif
}

// -- attention weights of blocks ------------------------------------------------------

struct WeighArgs {
    float* weights;
    const void* q;
    const float* lse;
    long long qt, qh;  // strides: token, head
    Cache c;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* cu;
    int W, T, B, Hq, G, max_q, causal;
    float scale, qsign;  // log2_scale(); a negative scale negates q
    int groups, split_rows, parts;  // of WeighPlan
    float* sums;                    // [request][kv head][part][block]
};

#if defined(__HIP_DEVICE_COMPILE__)
// Keys of a block as the matrix operand: keys 16 t + i, dims 64 j + 16 g + 8 n .. + 7 at step 2 j + n;
// their codes first, and the operand of them.
template <int D>
struct Keys {
    u32x4 raw[4][D / 64];
    float s;
    __device__ __forceinline__ void load(const Cache& c, long long blk, int i, int g) {
        s = ((ConstFloats)c.ks)[blk];
        const uint8_t* kp = c.kc + blk * (kBlock * D) + i * D + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
                raw[t][j] = *reinterpret_cast<const u32x4*>(kp + t * 16 * D + 64 * j);
    }
    template <class T>
    __device__ __forceinline__ typename Elem<T>::x8 step(int t, int n) const {
        return expand<T>(raw[t][n / 2][2 * (n % 2)], raw[t][n / 2][2 * (n % 2) + 1], s);
    }
};
// exp2 of 16 rows' scores with a block's keys less m (a lane's row), added to acc: those of keys below
// lim, where not every row sees every key.
template <int D, class T>
__device__ __forceinline__ void add_weights(const typename Elem<T>::x8 (&kf)[4][D / 32],
                                            const typename Elem<T>::x8 (&qf)[D / 32], float scale,
                                            float m, bool all, int lim, int key0, int g,
                                            float (&acc)[4]) {
    f32x4 S[4] = {};
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int t = 0; t < 4; ++t) S[t] = Elem<T>::mma16(kf[t][n], qf[n], S[t]);
    if (all) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += __builtin_amdgcn_exp2f(fmaf(S[t][e], scale, -m));
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(S[t][e], scale, -m));
                acc[e] += key0 + 16 * t + 4 * g + e < lim ? p : 0.f;
            }
    }
}
// What exp2 takes off: the lse in log2 units; infinity for a row of lse -inf (it sees nothing, or is
// behind the last), which then weighs 0.
__device__ __forceinline__ float shift_of(float lse) {
    return lse == -INFINITY ? INFINITY : lse * kLog2e;
}
#endif

// Few query rows (single tokens, drafts): a block of 64 keys a wave, the rows (a token's G heads beside
// each other) in tiles of 16. Bound by the bytes of the keys: codes are expanded 16 keys at a time, so
// that the registers are few and enough waves have theirs in flight. (A wave that goes over several
// blocks, with the next one's codes on their way, has half as many waves beside it: 39 us and not 29
// for 32 requests of 100 .. 16384 tokens.)
//
// grid: blocks of the table, kv heads, requests; one wave each, as ragged requests then fill the GPU best (four
// to a workgroup: 29.5 us and not 27.4).
template <int D, class T>
__global__ void __launch_bounds__(64, D == 64 ? 8 : 4) weigh_few_kernel(const WeighArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using x8 = typename Elem<T>::x8;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int hk = blockIdx.y, b = blockIdx.z;
    const Request req = request(a, b);
    const long long chunk = blockIdx.x;
    if (chunk * kBlock >= req.keys) return;
    const int page = ((ConstInts)(a.table + b * a.table_stride))[chunk * kBlock / a.c.page];
    if ((unsigned)page >= (unsigned)a.c.pages) return;
    const int key0 = (int)chunk * kBlock, rows = req.m * a.G;
    const long long blk = block_at(a.c, page, hk, (int)(chunk % (a.c.page / kBlock)));
    Keys<D> k;
    k.load(a.c, blk, i, g);
    const unsigned neg = a.qsign < 0.f ? 0x80008000u : 0u;
    float acc[4] = {};
    for (int r0 = 0; r0 < rows; r0 += 16) {
        const int r = r0 + i, tok = (int)((unsigned)r / (unsigned)a.G), h = hk * a.G + r - tok * a.G;
        const bool ok = r < rows;
        const T* q = (const T*)a.q + (req.first + tok) * a.qt + h * a.qh + 16 * g;
        x8 qf[D / 32];
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            u32x4 x = {};
            if (ok) x = *reinterpret_cast<const u32x4*>(q + 64 * (n / 2) + 8 * (n % 2));
            qf[n] = __builtin_bit_cast(x8, x ^ neg);
        }
        const float lse = ok ? a.lse[(long long)(req.first + tok) * a.Hq + h] : -INFINITY;
        const float m = shift_of(lse);
        const int lim = lse == -INFINITY ? 0 : seen_by(a, req, tok);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 S = {};
#pragma unroll
            for (int n = 0; n < D / 32; ++n)
                S = Elem<T>::mma16(k.template step<T>(t, n), qf[n], S);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(S[e], a.scale, -m));
                acc[e] += key0 + 16 * t + 4 * g + e < lim ? p : 0.f;
            }
        }
    }
    const float sum = wave_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    // (once a block and call, so that its order is set; requests that share a page add in any)
    if (lane == 0) atomicAdd(a.weights + blk, sum);
#endif
}

// Prompts: a workgroup has four blocks of 64 keys, one a wave in registers as above, and a part of the
// query rows (a.split_rows), which go by through LDS 64 at a time, operand by operand (frag_slot()), the
// next ones on their way while the four waves use them. Bound by neither unit alone: a tile's products are
// issued before its exponentials, so that a wave's matrix and vector work follow each other, and other waves
// hardly fill the gaps: the vector unit is busy for 63 % of the clocks, the matrix pipe for 34, 97 in all.
// Parts' sums go to the workspace, which weigh_join_kernel adds up, so that the
// order of a sum is set. 3 prompts of 77 .. 2111 queries behind 300 .. 8192 tokens, 16/4 heads of 128: 101 to
// 104 us (86 GFLOP) and 5 for the sums; 275 with every wave reading its rows from memory.
//
// grid: parts x groups of four blocks, kv heads, requests.
template <int D, class T>
__global__ void __launch_bounds__(256, 3) weigh_prompt_kernel(const WeighArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using x8 = typename Elem<T>::x8;
    constexpr int NS = D / 32, UN = D / 8, RW = 256 / UN, PER = 64 / RW;  // steps; 16-byte units a row;
                                                                          // rows a load; loads a stage
    __shared__ __attribute__((aligned(1024))) char qs[2][64 * 2 * D];
    __shared__ float ms[2][64];
    __shared__ int lims[2][64];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int wave = uni(tid >> 6), hk = blockIdx.y, b = blockIdx.z, G = a.G;
    const int part = uni((int)(blockIdx.x / (unsigned)a.groups));
    const long long group = blockIdx.x - (long long)part * a.groups;
    const Request req = request(a, b);
    const int rows = req.m * G;  // (the host has checked that it fits)
    if (group * (4 * kBlock) >= req.keys || (long long)part * a.split_rows >= rows) return;
    const long long chunk = group * 4 + wave;
    const int key0 = (int)(chunk * kBlock);
    int page = -1;
    if (key0 < req.keys) page = uni(a.table[b * a.table_stride + key0 / a.c.page]);
    const bool have = (unsigned)page < (unsigned)a.c.pages;
    const long long blk = have ? block_at(a.c, page, hk, (int)(chunk % (a.c.page / kBlock))) : 0;
    x8 kf[4][NS] = {};
    if (have) {
        Keys<D> k;
        k.load(a.c, blk, i, g);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < NS; ++n) kf[t][n] = k.template step<T>(t, n);
    }

    // The part's rows; from the first query on that sees the group's first key.
    const long long q0 = a.causal ? max(0LL, group * (4 * kBlock) - (req.len - req.n)) : 0;
    const int end = min(rows, (part + 1) * a.split_rows);
    int r0 = max(part * a.split_rows, (int)min(q0 * G, (long long)end) & ~63);
    // This thread's rows of the stages are r0 + lr, RW further on with every load: its head of the kv
    // head's and its place in q (a step of 64-bit places, another where a token's heads end); of the
    // first wave's lanes also row r0 + lane, 64 further on with every stage, and its token and lse.
    const int lr = tid / UN, u = tid % UN;
    struct Step {
        int tok, h;
        long long far, wrap;
    };
    auto step_of = [&](int n, long long per_tok, long long per_head) {
        const int t = uni((int)((unsigned)n / (unsigned)G)), h = n - t * G;
        return Step{t, h, t * per_tok + h * per_head, per_tok - G * per_head};
    };
    const Step qstep = step_of(RW, a.qt, a.qh), lstep = step_of(64, a.Hq, 1);
    int h = (int)((unsigned)(r0 + lr) % (unsigned)G), row = r0 + lr;
    const T* q = (const T*)a.q + (req.first + (row - h) / G) * a.qt + (hk * G + h) * a.qh + 8 * u;
    int ltok = (int)((unsigned)(r0 + lane) / (unsigned)G), lh = r0 + lane - ltok * G;
    const float* lse = a.lse + (long long)(req.first + ltok) * a.Hq + hk * G + lh;
    // Unit u is dims 8 u ..: step 2 j + n and lane group of u = 8 j + 2 g + n.
    const int at = (2 * (u >> 3) + (u & 1)) * 1024 + 16 * frag_slot(lr & 15, u >> 1 & 3, u & 1) +
                   (lr >> 4) * (NS * 1024);
    const unsigned neg = a.qsign < 0.f ? 0x80008000u : 0u;
    u32x4 x[PER];
    float m = 0.f;
    int lim = 0;
    auto fetch = [&] {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            x[n] = u32x4{};
            if (row < end) x[n] = *reinterpret_cast<const u32x4*>(q);
            row += RW;
            h += qstep.h;
            q += qstep.far;
            if (h >= G) {
                h -= G;
                q += qstep.wrap;
            }
        }
        if (wave == 0) {
            const bool ok = r0 + lane < end;
            m = ok ? *lse : -INFINITY;
            lim = m == -INFINITY ? 0 : seen_by(a, req, ltok);
            ltok += lstep.tok;
            lh += lstep.h;
            lse += lstep.far;
            if (lh >= G) {
                lh -= G;
                ++ltok;
                lse += lstep.wrap;
            }
        }
    };
    float acc[4] = {};
    fetch();
    for (int buf = 0; r0 < end; buf ^= 1) {
#pragma unroll
        for (int n = 0; n < PER; ++n)
            *reinterpret_cast<GFX906_LDS u32x4*>((GFX906_LDS char*)qs[buf] + at +
                                                 n * (RW / 16) * (NS * 1024)) = x[n] ^ neg;
        if (wave == 0) {
            ms[buf][lane] = shift_of(m);
            lims[buf][lane] = lim;
        }
        r0 += 64;
        if (r0 < end) fetch();
        lds_barrier();
        if (!have) continue;
        auto rows_of = [&](int t, x8 (&qf)[NS]) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
                qf[n] = lds_read16<T>(qs[buf], (t * NS + n) * 1024 + 16 * frag_slot(i, g, n & 1));
        };
        const int least = lims[buf][lane];
        if (!__any(least < key0 + kBlock)) {  // every row sees every key: the common case, without a branch
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                x8 qf[NS];
                rows_of(t, qf);
                add_weights<D, T>(kf, qf, a.scale, ms[buf][16 * t + i], true, 0, key0, g, acc);
            }
        } else if (__any(least > key0)) {
#pragma unroll 1
            for (int t = 0; t < 4; ++t) {
                x8 qf[NS];
                rows_of(t, qf);
                add_weights<D, T>(kf, qf, a.scale, ms[buf][16 * t + i], false, lims[buf][16 * t + i], key0,
                                  g, acc);
            }
        }
    }
    if (!have) return;
    const float sum = wave_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (lane) return;
    if (a.parts == 1)
        atomicAdd(a.weights + blk, sum);
    else
        a.sums[(((long long)b * a.c.Hkv + hk) * a.parts + part) * (4LL * a.groups) + chunk] = sum;
#endif
}

// Adds up the parts of every block. grid: blocks of the table / 256, kv heads, requests.
__global__ void __launch_bounds__(256) weigh_join_kernel(const WeighArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const long long chunk = blockIdx.x * 256LL + threadIdx.x;
    const int hk = blockIdx.y, b = blockIdx.z;
    const Request req = request(a, b);
    if (chunk * kBlock >= req.keys) return;
    const int page = a.table[b * a.table_stride + chunk * kBlock / a.c.page];
    if ((unsigned)page >= (unsigned)a.c.pages) return;
    const int parts = min(a.parts, (req.m * a.G + a.split_rows - 1) / a.split_rows);
    float sum = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p)
        sum += a.sums[(((long long)b * a.c.Hkv + hk) * a.parts + p) * (4LL * a.groups) + chunk];
    atomicAdd(a.weights + block_at(a.c, page, hk, (int)(chunk % (a.c.page / kBlock))), sum);
#endif
}

// How a call is launched: the rows of a part, so that there are up to 32 parts and workgroups for the
// GPU, and what the parts' sums take.
struct WeighPlan {
    long long blocks, groups;  // of the table: blocks of 64 keys, groups of four
    int split_rows, parts;
    size_t bytes;
};
// Query rows of a kv head that go to weigh_few_kernel. 32 requests of 100 .. 16384 tokens, 32/8 heads, us
// there / in weigh_prompt_kernel: 4 rows 27.3 / 45.8, 32 rows 34.8 / 46.4, 64 rows 47.0 / 44.2; one of
// 131000, 16/2 heads, 64 rows 17.5 / 15.5.
constexpr int kWeighFew = 32;
WeighPlan weigh_plan(int B, int G, int Hkv, int W, int page, int max_q) {
    WeighPlan p{};
    p.blocks = (long long)W * (page / kBlock);
    p.groups = (p.blocks + 3) / 4;
    const long long rows = (long long)max_q * G;
    if (rows <= kWeighFew) return p;
    const long long room = std::max(1LL, (1LL << 24) / std::max(1LL, 4 * p.groups * Hkv * B));
    const long long most = std::min({32LL, room, (rows + 511) / 512});
    p.split_rows = (int)(((rows + most - 1) / most + 63) / 64 * 64);
    p.parts = (int)((rows + p.split_rows - 1) / p.split_rows);
    if (p.parts > 1) p.bytes = (size_t)(4 * p.groups * Hkv * B * p.parts) * sizeof(float);
    return p;
}

// -- eviction -------------------------------------------------------------------------

struct EvictArgs {
    const float* weights;
    int pages, Hkv, page, W, B, first, recent, n_free;
    int* table;
    long long table_stride;
    const int* lens;
    const int* keep;
    int* free_pages;
    const int* used;
    int *lens_out, *used_out, *lost;
    unsigned long long* keys;  // [B][W], for wide tables
};

// Columns of a table whose keys fit LDS, and up to which a thread has one.
constexpr int kEvictLds = 4096, kEvictNarrow = 512;

#if defined(__HIP_DEVICE_COMPILE__)
// Pages of a request, how many entries of its row go, and which may: columns c0 .. c1 - 1.
struct Surplus {
    int n, gone, c0, c1;
};
__device__ __forceinline__ Surplus surplus(const EvictArgs& a, int len, int keep) {
    const long long n = min(((long long)max(0, len) + a.page - 1) / a.page, (long long)a.W);
    Surplus s;
    s.n = (int)n;
    s.gone = (int)max(0LL, min(n - keep, n - a.recent - a.first));
    s.c0 = s.gone ? a.first : 0;
    s.c1 = s.gone ? s.n - a.recent : 0;
    return s;
}
// Of the entries that go, those that name a page: entries that name none go before all others.
__device__ __forceinline__ int given_back(int gone, int bad) { return gone - min(gone, bad); }
#endif

// Before several requests' rows close up: how many entries a row loses follows from its length and
// budget, but which of them name a page only from the table, whose rows a workgroup each rewrites. So
// the pages that every request gives back are counted first, into lens_out, a wave a request. 64 requests of
// up to 512 pages 3.0 us.
__global__ void __launch_bounds__(256) evict_count_kernel(const EvictArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int lane = threadIdx.x & 63;
    if (b >= a.B) return;
    const Surplus s = surplus(a, ((ConstInts)a.lens)[b], ((ConstInts)a.keep)[b]);
    const int* const row = a.table + b * a.table_stride;
    int bad = 0;
    for (int base = s.c0 + lane; base < s.c1; base += 8 * 64) {
        int page[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) page[u] = row[min(base + 64 * u, s.c1 - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            bad += base + 64 * u < s.c1 && (unsigned)page[u] >= (unsigned)a.pages;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) bad += __shfl_xor(bad, o);
    if (lane == 0) a.lens_out[b] = given_back(s.gone, bad);
#endif
}

// Then added up: lens_out becomes the pages that the requests in front of each give back, and the free
// list's new end is set. One workgroup; 64 requests 2.5 us. (Counting in this one too: 64 requests of 512
// pages 15.6 us a call and not 14.1, 1000 of 64 pages 79 and not 18.)
__global__ void __launch_bounds__(1024) evict_place_kernel(const EvictArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ long long part[16];
    constexpr int PER = kMaxRequests / 1024;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int used = min(max(0, ((ConstInts)a.used)[0]), a.n_free);
    int given[PER];
    long long sum = 0;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        const int b = t * PER + n;
        given[n] = b < a.B ? a.lens_out[b] : 0;
        sum += given[n];
    }
    long long upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += part[w];
    long long at = upto - sum;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        const int b = t * PER + n;
        // (places past the free list are not written)
        if (b < a.B) a.lens_out[b] = (int)min(at, 0x7fffffffLL);
        at += given[n];
    }
    if (t == 1023) {
        a.used_out[0] = (int)max(0LL, used - upto);
        a.lost[0] = (int)min(max(0LL, upto - used), 0x7fffffffLL);
    }
#endif
}

// A workgroup a request. Which entries go: the `gone`-th smallest of the pages' weights, as 64-bit keys
// that order alike (0 for an entry that names no page, which is not given back), by
// histograms of 8 bits from the highest one in which they differ; mostly two or three
// passes until a bin is taken whole. Then the row closes up, NT columns at a time. Where a request's
// pages go in the free list evict_place_kernel has written, but for a single request. Bound by
// latency (dependent steps in one workgroup): 64 requests of up to 512 pages 8.4 us, one of 2048 14.6.
//
// LDS: whether the keys are kept there or in the workspace.
template <int NT, bool LDS>
__global__ void __launch_bounds__(NT) evict_kernel(const EvictArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef unsigned long long u64;
    constexpr int NW = NT / 64;
    __shared__ u64 keys_s[LDS ? kEvictLds : 1];
    __shared__ u64 red[3][NW];
    __shared__ int hist[256];
    __shared__ int wave_n[2][NW];
    __shared__ int chosen[3];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b = blockIdx.x;
    // (what needs no other value is loaded first)
    const int len = b < a.B ? ((ConstInts)a.lens)[b] : 0, keep = b < a.B ? ((ConstInts)a.keep)[b] : 0;
    const int had = ((ConstInts)a.used)[0];
    const bool alone = a.B <= 1;
    const int before = alone ? 0 : a.lens_out[b];
    const Surplus s = surplus(a, len, keep);
    const int n = s.n, gone = s.gone, c0 = s.c0, c1 = s.c1;
    int* const row = a.table + b * a.table_stride;
    u64* const keys = LDS ? keys_s : a.keys + (long long)b * a.W;
    const int per = a.Hkv * (a.page / kBlock);
    int bad = 0;  // entries that name no page
    u64 any = 0, each = ~0ull;
    // (two columns a thread at a time, the weights of both in flight)
    for (int base = c0 + t; base < c1; base += 2 * NT) {
        int page[2];
        double sum[2] = {};
#pragma unroll
        for (int u = 0; u < 2; ++u) page[u] = base + u * NT < c1 ? row[base + u * NT] : -1;
        const float* w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            w[u] = a.weights + ((unsigned)page[u] < (unsigned)a.pages ? (long long)page[u] * per : 0);
        if (a.pages) {
            for (int x = 0; x < per; x += 8) {
                float f[2][8];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < 8; ++n) f[u][n] = w[u][min(x + n, per - 1)];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < 8; ++n) sum[u] += x + n < per ? (double)f[u][n] : 0.0;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (base + u * NT >= c1) continue;
            u64 key = 0;
            if ((unsigned)page[u] >= (unsigned)a.pages) {
                ++bad;
            } else {
                const u64 v = (u64)__double_as_longlong(sum[u] + 0.0);
                key = sum[u] != sum[u] ? ~0ull : v >> 63 ? ~v : v | 1ull << 63;
            }
            keys[base + u * NT] = key;
            any |= key;
            each &= key;
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        bad += __shfl_xor(bad, o);
        any |= __shfl_xor(any, o);
        each &= __shfl_xor(each, o);
    }
    if (lane == 0) {
        red[0][wave] = (u64)bad;
        red[1][wave] = any;
        red[2][wave] = each;
    }
    for (int x = t; x < 256; x += NT) hist[x] = 0;
    __syncthreads();
    {
        // (a lane a wave's numbers, over the 16 or 8 lanes)
        const int w = lane % NW;
        bad = (int)red[0][w];
        any = red[1][w];
        each = red[2][w];
#pragma unroll
        for (int o = NW / 2; o; o >>= 1) {
            bad += __shfl_xor(bad, o);
            any |= __shfl_xor(any, o);
            each &= __shfl_xor(each, o);
        }
    }
    const int used = min(max(0, had), a.n_free), given = given_back(gone, bad);
    const int back = alone ? max(0, used - given) : a.used_out[0];
    if (t == 0) {
        if (alone) {
            a.used_out[0] = back;
            a.lost[0] = max(0, given - used);
        }
        if (b < a.B) a.lens_out[b] = len - gone * a.page;
    }
    if (gone == 0) return;
    // Of the keys whose bits from `hi` up are those of `limit`, the least `rem` go, and all below.
    u64 limit = each;
    int rem = gone, hi = any == each ? 0 : 64 - __clzll((long long)(any ^ each));
    bool whole = false;  // the keys up to `limit` go, else those below and the first `rem` equal ones
    while (hi > 0) {
        const int lo = max(0, hi - 8);
        limit = hi < 64 ? limit & ~0ull << hi : 0;
        for (int c = c0 + t; c < c1; c += NT) {
            const u64 k = keys[c];
            if (hi == 64 || k >> hi == limit >> hi)
                atomicAdd(&hist[(int)(k >> lo) & ((1 << (hi - lo)) - 1)], 1);
        }
        __syncthreads();
        if (wave == 0) {
            int x[4], sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                x[q] = hist[4 * lane + q];
                sum += x[q];
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(upto, o);
                if (lane >= o) upto += y;
            }
            int at = upto - sum;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (at < rem && rem <= at + x[q]) {
                    chosen[0] = 4 * lane + q;
                    chosen[1] = rem - at;
                    chosen[2] = x[q];
                }
                at += x[q];
            }
        }
        __syncthreads();
        const int bin = chosen[0], held = chosen[2];
        rem = chosen[1];
        limit |= (u64)bin << lo;
        hi = lo;
        if (rem == held) {
            limit |= (1ull << lo) - 1;
            whole = true;
            break;
        }
        for (int x = t; x < 256; x += NT) hist[x] = 0;
        __syncthreads();
    }

    // The row closes up. Entries are read before the barriers behind which others are written
    // to their places or in front of them.
    int turn = 0;
    auto scan = [&](bool x, int& total) {  // how many before this thread have x
        const u64 m = __ballot(x);
        turn ^= 1;  // (who still reads the counts of one scan has not reached the barrier of the next)
        if (lane == 0) wave_n[turn][wave] = __popcll(m);
        __syncthreads();
        int at = __popcll(m & ((1ull << lane) - 1));
        total = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const int c = wave_n[turn][w];
            at += w < wave ? c : 0;
            total += c;
        }
        return at;
    };
    int equal0 = 0, gone0 = 0, given0 = 0;
    for (int base = 0; base < n; base += NT) {
        const int c = base + t;
        const int page = c < n ? row[c] : -1;
        const bool may = c >= c0 && c < c1;
        const u64 key = may ? keys[c] : 0;
        bool out = may && (whole ? key <= limit : key < limit);
        int total;
        if (!whole) {
            const bool equal = may && key == limit;
            const int at = equal0 + scan(equal, total);
            equal0 += total;
            out |= equal && at < rem;
        }
        const int at = gone0 + scan(out, total);
        gone0 += total;
        const bool named = (unsigned)page < (unsigned)a.pages;
        int place = at;
        if (bad) {
            place = given0 + scan(out && named, total);
            given0 += total;
        }
        if (out) {
            const long long f = (long long)back + before + place;
            if (named && f < used) a.free_pages[f] = page;
        } else if (c < n) {
            row[c - at] = page;
        }
    }
    __syncthreads();
    for (int c = n - gone + t; c < n; c += NT) row[c] = -1;
#endif
}

template <class F>
void for_types(int dtype, int D, F go) {
    if (dtype == KV8_DTYPE_F16)
        D == 64 ? go(std::integral_constant<int, 64>{}, f16{})
                : go(std::integral_constant<int, 128>{}, f16{});
    else
        D == 64 ? go(std::integral_constant<int, 64>{}, bf16{})
                : go(std::integral_constant<int, 128>{}, bf16{});
}

int check_table(const int* table, long long stride, int B, int W, int page, const char* who) {
    if (W < 0 || (B > 0 && W > 0 && !table)) return last_error().fail("%s: null table or negative width", who);
    if ((long long)W * page >= (1LL << 31) || stride < 0)
        return last_error().fail("%s: table too wide or a negative stride", who);
    return 0;
}

}  // namespace

extern "C" const char* kv8_last_error(void) { return last_error().get(); }

extern "C" int kv8_store(const void* k, const void* v, const long long* k_strides,
                         const long long* v_strides, int dtype, int T, int B, int Hkv, int D,
                         void* k_codes, float* k_scales, void* v_codes, float* v_scales, int pages,
                         int page, const int* table, long long table_stride, int W, const int* lens,
                         const int* cu_new, float* weights, hipStream_t stream) {
    const char* who = "kv8_store";
    LastError& err = last_error();
    err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, who)) return 1;
    if (dtype != KV8_DTYPE_F16 && dtype != KV8_DTYPE_BF16) return err.fail("%s: bad dtype", who);
    if (T < 0 || B < 0) return err.fail("%s: negative sizes", who);
    if (B > kMaxRequests) return err.fail("%s: at most %d requests", who, kMaxRequests);
    if (!cu_new && T != B) return err.fail("%s: without cu_new, one row a request", who);
    if (check_table(table, table_stride, B, W, page, who)) return 1;
    if (T == 0 || B == 0 || pages == 0 || W == 0) return 0;
    if (!k || !v || !lens || !k_strides || !v_strides) return err.fail("%s: null argument", who);
    for (int i = 0; i < 2; ++i)
        if (k_strides[i] < 0 || v_strides[i] < 0 || k_strides[i] % 8 || v_strides[i] % 8)
            return err.fail("%s: strides must be non-negative multiples of 8 elements", who);
    if (!aligned(k, 16) || !aligned(v, 16))
        return err.fail("%s: k and v must be 16-byte aligned", who);
    StoreArgs a{};
    a.k = k;
    a.v = v;
    a.kt = k_strides[0];
    a.kh = k_strides[1];
    a.vt = v_strides[0];
    a.vh = v_strides[1];
    a.c = Cache{(const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                pages, page, Hkv, D};
    a.table = table;
    a.table_stride = table_stride;
    a.lens = lens;
    a.cu = cu_new;
    a.weights = weights;
    a.W = W;
    a.T = T;
    a.B = B;
    a.max_q = T;
    a.tasks = (unsigned)(T / kBlock) + 2u * B;
    const long long waves = (long long)a.tasks * Hkv * 2, grid = (waves + 3) / 4;
    if (!launchable(grid, 256) || waves >= (1LL << 32))
        return err.fail("%s: too many rows for one call", who);
    for_types(dtype, D, [&](auto d, auto t) {
        hipLaunchKernelGGL((store_kernel<decltype(t), decltype(d)::value>), dim3((unsigned)grid),
                           dim3(256), 0, stream, a);
    });
    return err.launched(who, hipGetLastError());
}

extern "C" int kv8_load(void* k, void* v, int dtype, int T, int Hkv, int D, const int* slots,
                        const void* k_codes, const float* k_scales, const void* v_codes,
                        const float* v_scales, int pages, int page, hipStream_t stream) {
    const char* who = "kv8_load";
    LastError& err = last_error();
    err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, who)) return 1;
    if (dtype != KV8_DTYPE_F16 && dtype != KV8_DTYPE_BF16) return err.fail("%s: bad dtype", who);
    if (T < 0) return err.fail("%s: negative token count", who);
    if (T == 0) return 0;
    if (!k || !v || !slots) return err.fail("%s: null argument", who);
    if (!aligned(k, 16) || !aligned(v, 16))
        return err.fail("%s: k and v must be 16-byte aligned", who);
    if (Hkv > 32767 || !launchable((T + 63LL) / 64 * Hkv * 2, 256))
        return err.fail("%s: too many rows or heads for one call", who);
    const LoadArgs a{k, v, slots,
                     Cache{(const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                           pages, page, Hkv, D},
                     T};
    for_types(dtype, D, [&](auto d, auto t) {
        hipLaunchKernelGGL((load_kernel<decltype(t), decltype(d)::value>),
                           dim3((unsigned)((T + 63LL) / 64), (unsigned)Hkv * 2), dim3(256), 0, stream,
                           a);
    });
    return err.launched(who, hipGetLastError());
}

extern "C" size_t kv8_weigh_workspace_bytes(int T, int B, int Hq, int Hkv, int max_q, int W, int page) {
    if (T <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || max_q <= 0 || W <= 0 || page <= 0) return 0;
    return weigh_plan(B, Hq / Hkv, Hkv, W, page, std::min(max_q, T)).bytes;
}

extern "C" int kv8_weigh(float* weights, const void* q, const long long* q_strides, int dtype,
                         const float* lse, int T, int B, int Hq, int Hkv, int D,
                         const void* k_codes, const float* k_scales, int pages, int page,
                         const int* table, long long table_stride, int W, const int* lens,
                         const int* cu_q, int max_q, float scale, int causal, void* workspace,
                         size_t workspace_bytes, hipStream_t stream) {
    const char* who = "kv8_weigh";
    LastError& err = last_error();
    err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, k_codes, k_scales, who)) return 1;
    if (dtype != KV8_DTYPE_F16 && dtype != KV8_DTYPE_BF16) return err.fail("%s: bad dtype", who);
    if (T < 0 || B < 0 || max_q < 0) return err.fail("%s: negative sizes", who);
    if (B > kMaxRequests) return err.fail("%s: at most %d requests", who, kMaxRequests);
    if (Hq <= 0 || Hq % Hkv || Hq > 65535)
        return err.fail("%s: query heads must be a multiple of kv heads", who);
    if (!cu_q && T != B) return err.fail("%s: without cu_q, one query a request", who);
    if (check_table(table, table_stride, B, W, page, who)) return 1;
    if (!good_scale(scale)) return err.fail("%s: scale must be finite, and below 2.3e38", who);
    if (T == 0 || B == 0 || max_q == 0 || pages == 0 || W == 0) return 0;
    if (!weights || !q || !q_strides || !lse || !lens) return err.fail("%s: null argument", who);
    for (int i = 0; i < 2; ++i)
        if (q_strides[i] < 0 || q_strides[i] % 8)
            return err.fail("%s: strides must be non-negative multiples of 8 elements", who);
    if (!aligned(q, 16) || !aligned(weights, 4) || !aligned(lse, 4))
        return err.fail("%s: q must be 16-byte, weights and lse 4-byte aligned", who);
    WeighArgs a{};
    a.weights = weights;
    a.q = q;
    a.lse = lse;
    a.qt = q_strides[0];
    a.qh = q_strides[1];
    a.c = Cache{(const uint8_t*)k_codes, k_scales, nullptr, nullptr, pages, page, Hkv, D};
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
    if ((long long)a.max_q * a.G >= (1LL << 30)) return err.fail("%s: too many query rows", who);
    const WeighPlan p = weigh_plan(B, a.G, Hkv, W, page, a.max_q);
    if (B > 65535 || !launchable((p.parts ? p.parts * p.groups : p.groups) * Hkv * B, 256) ||
        p.parts * p.groups >= (1LL << 31))
        return err.fail("%s: table too wide for so many heads", who);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 4)))
        return err.fail("%s: workspace misaligned or smaller than kv8_weigh_workspace_bytes()", who);
    a.groups = (int)p.groups;
    a.split_rows = p.split_rows;
    a.parts = p.parts;
    a.sums = (float*)workspace;
    for_types(dtype, D, [&](auto d, auto t) {
        constexpr int kD = decltype(d)::value;
        if (!p.parts)
            hipLaunchKernelGGL((weigh_few_kernel<kD, decltype(t)>),
                               dim3((unsigned)p.blocks, (unsigned)Hkv, (unsigned)B), dim3(64), 0, stream,
                               a);
        else
            hipLaunchKernelGGL((weigh_prompt_kernel<kD, decltype(t)>),
                               dim3((unsigned)(p.parts * p.groups), (unsigned)Hkv, (unsigned)B),
                               dim3(256), 0, stream, a);
    });
    if (p.parts > 1)
        hipLaunchKernelGGL(weigh_join_kernel,
                           dim3((unsigned)((p.blocks + 255) / 256), (unsigned)Hkv, (unsigned)B),
                           dim3(256), 0, stream, a);
    return err.launched(who, hipGetLastError());
}

extern "C" size_t kv8_evict_workspace_bytes(int B, int W) {
    return B > 0 && W > kEvictLds ? (size_t)B * W * sizeof(unsigned long long) : 0;
}

extern "C" int kv8_evict(const float* weights, int pages, int Hkv, int page, int* table,
                         long long table_stride, int W, const int* lens, const int* keep, int B,
                         int first, int recent, int* free_pages, int n_free, const int* used,
                         int* lens_out, int* used_out, int* lost, void* workspace,
                         size_t workspace_bytes, hipStream_t stream) {
    const char* who = "kv8_evict";
    LastError& err = last_error();
    err.text[0] = 0;
    if (page != 64 && page != 128 && page != 256)
        return err.fail("%s: pages hold 64, 128 or 256 tokens", who);
    if (Hkv <= 0 || Hkv > 65535) return err.fail("%s: bad number of kv heads", who);
    if (pages < 0 || (long long)pages * page >= (1LL << 31))
        return err.fail("%s: the cache must hold fewer than 2^31 tokens", who);
    if (B < 0 || B > kMaxRequests) return err.fail("%s: at most %d requests", who, kMaxRequests);
    if (n_free < 0) return err.fail("%s: negative sizes", who);
    if (first < 0 || recent < 1)
        return err.fail("%s: first must be at least 0 and recent at least 1", who);
    if (check_table(table, table_stride, B, W, page, who)) return 1;
    if (B > 1 && table_stride < W) return err.fail("%s: overlapping table rows", who);
    if (!used || !used_out || !lost || (n_free > 0 && !free_pages) ||
        (B > 0 && (!lens || !keep || !lens_out)) || (pages > 0 && !weights))
        return err.fail("%s: null argument", who);
    const size_t need = kv8_evict_workspace_bytes(B, W);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 8)))
        return err.fail("%s: workspace misaligned or smaller than kv8_evict_workspace_bytes()", who);
    // Every workgroup reads inputs that others' results would overwrite.
    struct Ints {
        const int* at;
        long long n;
    };
    const Ints outs[3] = {{lens_out, B}, {used_out, 1}, {lost, 1}};
    const Ints ins[4] = {{lens, B}, {keep, B}, {used, 1}, {free_pages, n_free}};
    auto apart = [](const Ints& x, const Ints& y) {
        const uintptr_t p = (uintptr_t)x.at, q = (uintptr_t)y.at;
        return !x.n || !y.n || p + 4 * x.n <= q || q + 4 * y.n <= p;
    };
    for (int i = 0; i < 3; ++i) {
        for (const Ints& in : ins)
            if (!apart(outs[i], in)) return err.fail("%s: results overlap the arguments", who);
        for (int j = 0; j < i; ++j)
            if (!apart(outs[i], outs[j])) return err.fail("%s: results overlap each other", who);
    }
    // (more of them than a row has columns are as many as it has, and columns past the first ones
    // then fit an int)
    first = std::min(first, W);
    recent = std::min(recent, std::max(W, 1));
    const EvictArgs a{weights, pages, Hkv,  page,       W,    B,        first,    recent,
                      n_free,  table, table_stride, lens, keep, free_pages, used, lens_out,
                      used_out, lost, (unsigned long long*)workspace};
    const dim3 grid((unsigned)std::max(B, 1));
    if (B > 1) {
        hipLaunchKernelGGL(evict_count_kernel, dim3((unsigned)(B + 3) / 4), dim3(256), 0, stream, a);
        hipLaunchKernelGGL(evict_place_kernel, dim3(1), dim3(1024), 0, stream, a);
    }
    if (W <= kEvictNarrow)
        hipLaunchKernelGGL((evict_kernel<512, true>), grid, dim3(512), 0, stream, a);
    else if (W <= kEvictLds)
        hipLaunchKernelGGL((evict_kernel<1024, true>), grid, dim3(1024), 0, stream, a);
    else
        hipLaunchKernelGGL((evict_kernel<1024, false>), grid, dim3(1024), 0, stream, a);
    return err.launched(who, hipGetLastError());
}
