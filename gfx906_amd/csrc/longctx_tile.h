// One wave's work on blocks of 32 keys, for 16 or 32 query rows and head dims of 64
// or 128: the matrix products, the softmax and the tile layout in LDS that the sparse
// and the 4-bit cache's prompt kernels share. The scheme is that of attn_fwd_pipe
// (attn_kernel.hip):
//
//  * S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32; a lane holds, for
//    query 16 nb + l%16, the scores of keys 16 kb + 4 (l/16) + 0..3, and the same
//    registers rounded to the element type are the second product's operand.
//  * P = exp2(s c - m) is computed with a running max m that may be stale; when some
//    rounded p passes 2^15 the block's exact max is taken and O, l and P follow.
//  * l is summed on the matrix pipe from the rounded P, so numerator and
//    denominator see the same weights.
//
// Tiles of 32 rows lie in LDS in the element type, 16-byte units XOR-swizzled so
// that the reads of K (16 rows x one unit) and the transposed reads of V (4 rows x
// 2 units) are free of bank conflicts.
#pragma once

#include "longctx.h"

#if defined(__HIP_DEVICE_COMPILE__)

namespace gfx906_amd {
namespace longctx {

#define GFX906_LDS __attribute__((address_space(3)))

typedef __fp16 fp16x4_t __attribute__((ext_vector_type(4)));

constexpr float kPLimit = 32768.0f;
// A buffer offset past every descriptor's range: loads zeros.
constexpr unsigned kOutOfRange = 0x80000000u;

// This wave's LDS accesses are done, then the workgroup's barrier; loads into LDS
// stay in flight (waited for by count).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ float max2(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
}
__device__ __forceinline__ float max3(float a, float b, float c) { return max2(max2(a, b), c); }

// Sum / max over lanes i, i+16, i+32, i+48.
__device__ __forceinline__ float quad_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned y = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float quad_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned y = __float_as_uint(max2(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <class T>
__device__ __forceinline__ typename Elem<T>::x8 lds_read16(const char* base, int off) {
    return *(const GFX906_LDS typename Elem<T>::x8*)((const GFX906_LDS char*)base + off);
}
// Two transposed 8-byte reads (ds_read_b64_tr_b16) joined into one operand.
template <class T>
__device__ __forceinline__ typename Elem<T>::x8 lds_read_tr2(const char* base, int lo, int hi) {
    const fp16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
        (GFX906_LDS fp16x4_t*)((GFX906_LDS char*)base + lo));
    const fp16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
        (GFX906_LDS fp16x4_t*)((GFX906_LDS char*)base + hi));
    const u32x2 l = __builtin_bit_cast(u32x2, a), h = __builtin_bit_cast(u32x2, b);
    return __builtin_bit_cast(typename Elem<T>::x8, u32x4{l[0], l[1], h[0], h[1]});
}

// Swizzles of the 16-byte unit index within row r of a K or V tile, NU units a row.
template <int NU>
__device__ __forceinline__ int kswz(int r) { return NU >= 16 ? (r & 15) : ((r >> 1) & 7); }
template <int NU>
__device__ __forceinline__ int vswz(int r) { return NU >= 16 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }

// Whether some element of P (non-negative) exceeds kPLimit or is NaN, in any lane.
// bf16 goes through the same packed fp16 maxima: patterns of non-negative values
// order alike, and kPLimit's bf16 pattern read as fp16 is 7.0.
template <class T, int NB>
__device__ __forceinline__ bool p_above(const typename Elem<T>::x8 (&P)[NB]) {
    auto h = [](unsigned u) { return __builtin_bit_cast(f16x2, u); };
    auto mx = [](f16x2 x, f16x2 y) { return __builtin_elementwise_maximum(x, y); };
    const u32x4 a = __builtin_bit_cast(u32x4, P[0]);
    f16x2 r;
    if constexpr (NB == 2) {
        const u32x4 b = __builtin_bit_cast(u32x4, P[1]);
        const f16x2 x = mx(mx(h(a[0]), h(a[1])), h(a[2])), y = mx(mx(h(a[3]), h(b[0])), h(b[1]));
        r = mx(y, mx(mx(h(b[2]), h(b[3])), x));
    } else {
        r = mx(mx(mx(h(a[0]), h(a[1])), h(a[2])), h(a[3]));
    }
    const f16 lim = __is_same(T, f16) ? (f16)kPLimit : __builtin_bit_cast(f16, (bf16)kPLimit);
    return __builtin_amdgcn_ballot_w64(!(r[0] <= lim) || !(r[1] <= lim)) != 0;
}

// NB: column blocks of 16 query rows.
template <int D, class T, int NB = 2>
struct Tile {
    using E = Elem<T>;
    using x8 = typename E::x8;
    static constexpr int NU = D / 8, RB = 2 * D, BYTES = 32 * RB;  // one tile
    static constexpr int NQ = D / 32, NO = D / 16;

    x8 qf[NB][NQ];  // query 16 nb + l%16, dims 32 s + 8 (l/16)..+7
    f32x4 oacc[NO][NB];
    f32x4 lacc[NB];
    float m[NB];  // running max in log2 units
    bool far;    // (wave-uniform) some |m| is past 2^16: exact maxima from there on
    x8 one;
    int kaddr[NQ], vaddr[NO];

    __device__ __forceinline__ void init(int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int ob = 0; ob < NO; ++ob) oacc[ob][nb] = f32x4{};
            lacc[nb] = f32x4{};
            m[nb] = kNoMax;
        }
        far = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) one[e] = (T)(i == 0 ? 1.0f : 0.0f);
#pragma unroll
        for (int s = 0; s < NQ; ++s) kaddr[s] = i * RB + ((4 * s + g) ^ kswz<NU>(i)) * 16;
        const int vrow = 4 * g + (i >> 2), vx = vswz<NU>(vrow) >> 1;
#pragma unroll
        for (int ob = 0; ob < NO; ++ob) vaddr[ob] = vrow * RB + (ob ^ vx) * 32 + (i & 3) * 8;
    }

    // S of the K tile kt.
    __device__ __forceinline__ void qk(const char* kt, f32x4 (&S)[2][NB]) const {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) S[kb][nb] = f32x4{};
#pragma unroll
        for (int s = 0; s < NQ; ++s)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const x8 kf = lds_read16<T>(kt, kaddr[s] + 16 * kb * RB);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) S[kb][nb] = E::mma16(kf, qf[nb][s], S[kb][nb]);
            }
        // K reads a few fragments ahead of the products (as attn_fwd_pipe's order).
        constexpr int A = D == 64 ? 3 : 2;
        __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
        for (int n = 0; n < 2 * NQ - A; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NB * A, 0);
    }

    // O^T += V^T P^T of the V tile vt.
    __device__ __forceinline__ void pv(const char* vt, const x8 (&P)[NB]) {
#pragma unroll
        for (int ob = 0; ob < NO; ++ob) {
            const x8 vf = lds_read_tr2<T>(vt, vaddr[ob], vaddr[ob] + 16 * RB);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) oacc[ob][nb] = E::mma16(vf, P[nb], oacc[ob][nb]);
        }
        constexpr int A = D == 128 ? 4 : 3;
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * A, 0);
#pragma unroll
        for (int n = 0; n < NO - A; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NB * A, 0);
    }

    // Scores of keys key0 + 0..31 at or past lim[nb] to -inf.
    __device__ __forceinline__ void mask(f32x4 (&S)[2][NB], int key0, const int (&lim)[NB],
                                         int g) const {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key0 + 16 * kb + 4 * g + r >= lim[nb]) S[kb][nb][r] = -INFINITY;
    }

    // P of column block nb. FAR: from the rounded product s c, as m is, so that a score
    // equal to the max gives exactly 1 and none gives more. Below |m| = 2^16 the fma's
    // unrounded product differs from that by less than 2^-8 in the exponent, which is
    // within what an fp32 sum of that size may be off by; at 2^33 it would be 2^9 and
    // overflow.
    template <bool FAR>
    __device__ __forceinline__ void weights(const f32x4 (&S)[2][NB], x8 (&P)[NB], float c,
                                            int nb) const {
#pragma clang fp contract(off)
        auto p = [&](float s) __attribute__((always_inline)) {
#pragma clang fp contract(off)
            const float sc = s * c;
            return __builtin_amdgcn_exp2f(FAR ? sc - m[nb] : fmaf(s, c, -m[nb]));
        };
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const f32x4& s = e < 4 ? S[0][nb] : S[1][nb];
            const typename E::x2 h = E::cvt2(p(s[e & 3]), p(s[(e & 3) + 1]));
            P[nb][e] = h[0];
            P[nb][e + 1] = h[1];
        }
    }

    __device__ __forceinline__ void softmax(const f32x4 (&S)[2][NB], x8 (&P)[NB], float c) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) weights<false>(S, P, c, nb);
        settle(S, P, c);
    }

    // One step of the pipeline: the second product of one block (vt, Pp), the first of
    // another (kt, Sn), and P of the block S between them, in the order written: behind every
    // fragment's products the read of the fragment AV (V) or AK (K) further on, and a share
    // of the softmax, so that a wave's own instructions fill the matrix pipe's time. (The
    // compiler's order has all products before all exponentials: the call of 16 heads of 16384
    // tokens, 32 blocks of 64, 300 us and 284 this way; a 4-bit cache's prompts 218 and 201.)
    __device__ __forceinline__ void turn(const char* vt, const x8 (&Pp)[NB], const char* kt,
                                         f32x4 (&Sn)[2][NB], const f32x4 (&S)[2][NB], x8 (&P)[NB],
                                         float c) {
        constexpr int AV = 2, AK = 2, NK = 2 * NQ, EPS = 8 * NB / (NO + NK);
        x8 vf[NO], kf[NK];
        float p[8 * NB];
        auto vread = [&](int n) __attribute__((always_inline)) {
            vf[n] = lds_read_tr2<T>(vt, vaddr[n], vaddr[n] + 16 * RB);
        };
        auto kread = [&](int n) __attribute__((always_inline)) {
            kf[n] = lds_read16<T>(kt, kaddr[n / 2] + 16 * (n % 2) * RB);
        };
        auto share = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
            for (int q = slot * EPS; q < (slot + 1) * EPS; ++q) {
                const int nb = q / 8, e = q % 8;
                p[q] = __builtin_amdgcn_exp2f(fmaf(S[e / 4][nb][e & 3], c, -m[nb]));
                if (e & 1) {
                    const typename E::x2 h = E::cvt2(p[q - 1], p[q]);
                    P[nb][e - 1] = h[0];
                    P[nb][e] = h[1];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int n = 0; n < AV; ++n) vread(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NO; ++n) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) oacc[n][nb] = E::mma16(vf[n], Pp[nb], oacc[n][nb]);
            if (n + AV < NO) vread(n + AV);
            if (n >= NO - AK) kread(n - (NO - AK));
            share(n);
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) Sn[kb][nb] = f32x4{};
#pragma unroll
        for (int n = 0; n < NK; ++n) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                Sn[n % 2][nb] = E::mma16(kf[n], qf[nb][n / 2], Sn[n % 2][nb]);
            if (n + AK < NK) kread(n + AK);
            share(NO + n);
        }
        settle(S, P, c);
    }

    // Where some p passed the limit: the exact maximum of the block, and O, l and P after
    // it. Then the row sums.
    __device__ __forceinline__ void settle(const f32x4 (&S)[2][NB], x8 (&P)[NB], float c) {
        if (__builtin_expect(p_above<T, NB>(P) || far, 0)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float a = max3(S[0][nb][0], S[0][nb][1], S[0][nb][2]);
                const float b = max3(S[0][nb][3], S[1][nb][0], S[1][nb][1]);
                const float mx = max3(a, b, max2(S[1][nb][2], S[1][nb][3]));
                const float mn = max2(m[nb], quad_max(mx) * c);
                const float w = __builtin_amdgcn_exp2f(m[nb] - mn);
#pragma unroll
                for (int ob = 0; ob < NO; ++ob) oacc[ob][nb] *= w;
                lacc[nb] *= w;
                m[nb] = mn;
                weights<true>(S, P, c, nb);
            }
            auto big = [](float x) { return fabsf(x) > 65536.f && x != kNoMax; };
            far = __builtin_amdgcn_ballot_w64(big(m[0]) || big(m[NB - 1])) != 0;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) lacc[nb] = E::mma16(one, P[nb], lacc[nb]);
    }
};

// Whether a tile of V in LDS holds an infinity or NaN in its first `rows` rows.
template <int D, class T>
__device__ __forceinline__ bool not_finite(const char* vt, int lane) {
    constexpr unsigned kExp = __is_same(T, f16) ? 0x7c00u : 0x7f80u;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < Tile<D, T>::BYTES / 1024; ++u) {
        const u32x4 x = *(const GFX906_LDS u32x4*)((const GFX906_LDS char*)vt + u * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            bad |= (x[e] & kExp) == kExp || (x[e] >> 16 & kExp) == kExp;
    }
    return __any(bad);
}

}  // namespace longctx
}  // namespace gfx906_amd

#endif
