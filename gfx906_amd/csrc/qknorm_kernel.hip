// Norms of queries and keys for each head with the position rotation in the same
// pass, for AMD MI355X (gfx950). The entry point is described in
// gfx906_amd_attn.h.
//
//   y = x / sqrt(mean(x^2) + eps) * w        over the D dims of a head
//   (y_i, y_j) <- (c y_i - s y_j, s y_i + c y_j)   for the pairs of the first R dims
//
// in fp32, rounded once. Bound by bytes: every row is read and written once, and a
// token's angles are kept in registers while a wave goes over its heads. 2 x 8192 tokens, 24
// heads of 64 each in q and k, 36 us in the kernel and 40 a call: 5.1 TB/s. 32 tokens, 32 and 8 heads of
// 128: 5.4, a launch and three loads that wait for each other.
#include "longctx.h"

#include <algorithm>
#include <type_traits>

#include "gfx906_amd_attn.h"

namespace {

using namespace gfx906_amd::longctx;

thread_local LastError g_err;

constexpr int kUnroll = 4;  // rows in flight a lane

struct Rows {
    const void* x;
    void* y;
    const void* w;
    long long xb, xs, xh, yb, ys, yh;  // strides: batch, token, head
    int H, chunks;                     // heads; chunks of them a wave takes
};
struct RotateArgs {
    Rows part[2];  // q, k
    const float* cos;
    const float* sin;
    const int* pos;
    long long ab, pb, ps;  // strides of a row of angles, of pos: batch, token
    unsigned B, S, N, groups;  // groups: of tokens
    int D, R, w32, heads;  // w32: weights are fp32; heads a wave goes over
    int tok_step, head_step, head_next;  // of a row group; from one round of a wave to the next
    float eps, inv_d;
};

// A row is 8 dims a lane in L = 2^k lanes (some idle where D is not 8 L), a wave 64 / L rows: of one
// head's tokens, or of one token's heads (tok_step, head_step). The wave goes over `heads` heads with
// the same tokens' angles; kUnroll rows a lane are in flight, of as many heads or, where there are too few
// heads, of TS tokens.
//
// NEAR: pairs are neighbours (2i, 2i+1) and lie in one lane; else halves
// (i, i + R/2), whose other number another lane holds.
template <class T, int L, bool NEAR, int TS>
__global__ void __launch_bounds__(256) norm_rotate_kernel(const RotateArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using x8 = typename Elem<T>::x8;
    constexpr int RG = 64 / L, HS = kUnroll / TS, NA = NEAR ? 4 : 8;
    const int lane = threadIdx.x & 63, l = lane % L, grp = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned task = blockIdx.x * 4 + wave;
    const unsigned per = a.part[0].chunks + a.part[1].chunks;
    const unsigned tg = task / per;
    if (tg >= a.groups) return;
    int chunk = task - tg * per;
    const bool is_k = chunk >= a.part[0].chunks;
    if (is_k) chunk -= a.part[0].chunks;
    const Rows& p = a.part[is_k];
    int h = chunk * a.heads + grp * a.head_step;
    const int h1 = min(p.H, (chunk + 1) * a.heads);
    // The lane's tokens, counted over batches, and where their rows and angles lie.
    const bool turn = 8 * l < a.R;
    const int half = a.R / 16;  // lanes between the numbers of a pair
    bool live[TS];
    const T* x[TS];
    T* y[TS];
    long long at[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        const unsigned t = a.tok_step ? (tg * TS + i) * RG + grp : tg, last = a.B * a.S - 1;
        live[i] = t <= last && 8 * l < a.D;
        const unsigned b = min(t, last) / a.S, s = min(t, last) - b * a.S;
        x[i] = (const T*)p.x + b * p.xb + s * p.xs + 8 * l;
        y[i] = (T*)p.y + b * p.yb + s * p.ys + 8 * l;
        at[i] = s;
        if (turn && a.pos) at[i] = a.pos[b * a.pb + s * a.ps];
    }
    u32x4 raw[kUnroll];
    auto fetch = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            raw[u] = u32x4{};
            const int hh = from + u % HS * a.head_next;
            if (live[u / HS] && hh < h1)
                raw[u] = *reinterpret_cast<const u32x4*>(x[u / HS] + hh * p.xh);
        }
    };
    // (the positions' loads and the first rows' are on their way together; angles and weights follow)
    fetch(h);
    float w[8], c[TS][NA], n[TS][NA];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
    if (p.w && 8 * l < a.D) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            w[e] = a.w32 ? ((const float*)p.w)[8 * l + e] : (float)((const T*)p.w)[8 * l + e];
    }
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        if (turn) {
            const bool ok = (unsigned long long)at[i] < a.N;
            const long long off = (ok ? at[i] : 0) * a.ab + (NEAR ? 4 * l : 8 * (l < half ? l : l - half));
            const float sign = NEAR || l >= half ? 1.f : -1.f;
#pragma unroll
            for (int e = 0; e < NA; e += 4) {
                const f32x4 cc = *reinterpret_cast<const f32x4*>(a.cos + off + e);
                const f32x4 ss = *reinterpret_cast<const f32x4*>(a.sin + off + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    c[i][e + k] = ok ? cc[k] : NAN;
                    n[i][e + k] = ok ? sign * ss[k] : NAN;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < NA; ++e) c[i][e] = 1.f, n[i][e] = 0.f;
        }
    }
    const int other = grp * L + (l < half ? l + half : l - half);

    while (true) {
        u32x4 now[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) now[u] = raw[u];
        const int next = h + HS * a.head_next;
        const bool more = __any(next < h1);
        if (more) fetch(next);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const x8 in = __builtin_bit_cast(x8, now[u]);
            float v[8], sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = (float)in[e];
                sum = fmaf(v[e], v[e], sum);
            }
#pragma unroll
            for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o);
            float mean = sum * a.inv_d + a.eps, r = __builtin_amdgcn_rsqf(mean);
            const bool big = !(mean < INFINITY), off = big || mean < 0x1p-100f;
            if (__builtin_expect(__any(off), 0)) {
                // Squares past fp32 or below its range (bf16 rows): the row times 2^-80 or 2^80, and eps
                // with its square, in two steps, as 2^160 is no fp32 number. (The wave's other rows
                // keep what they have.)
                const float f = big ? 0x1p-80f : off ? 0x1p80f : 1.f;
                sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] *= f;
                    sum = fmaf(v[e], v[e], sum);
                }
#pragma unroll
                for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o);
                if (off) r = 1.0f / sqrtf(sum * a.inv_d + a.eps * f * f);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * r * w[e];
            if (a.R) {
                float z[8];
                if constexpr (NEAR) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        z[e] = v[e] * c[u / HS][e / 2] - v[e + 1] * n[u / HS][e / 2];
                        z[e + 1] = v[e] * n[u / HS][e / 2] + v[e + 1] * c[u / HS][e / 2];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        z[e] = v[e] * c[u / HS][e] + __shfl(v[e], other) * n[u / HS][e];
                }
                if (turn) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = z[e];
                }
            }
            const int hh = h + u % HS * a.head_next;
            if (live[u / HS] && hh < h1) {
                u32x4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out[e] = __builtin_bit_cast(unsigned, Elem<T>::cvt2(v[2 * e], v[2 * e + 1]));
                *reinterpret_cast<u32x4*>(y[u / HS] + hh * p.yh) = out;
            }
        }
        if (!more) break;
        h = next;
    }
#endif
}

}  // namespace

extern "C" const char* qk_norm_rotate_last_error(void) { return g_err.get(); }

extern "C" int qk_norm_rotate(const void* q, const void* k, void* q_out, void* k_out,
                              const long long* q_strides, const long long* k_strides,
                              const long long* q_out_strides, const long long* k_out_strides,
                              int dtype, int B, int S, int Hq, int Hk, int D, const void* q_weight,
                              const void* k_weight, int weight_f32, float eps, const float* cos,
                              const float* sin, long long angle_stride, int N, int R,
                              int neighbours, const int* positions, const long long* p_strides,
                              hipStream_t stream) {
    g_err.text[0] = 0;
    const char* who = "qk_norm_rotate";
    if (dtype != KV8_DTYPE_F16 && dtype != KV8_DTYPE_BF16) return g_err.fail("%s: bad dtype", who);
    if (D <= 0 || D > 512 || D % 8)
        return g_err.fail("%s: head dim must be a multiple of 8 up to 512", who);
    if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || Hq > 65535 || Hk > 65535)
        return g_err.fail("%s: bad number of tokens or heads", who);
    if ((long long)B * S >= (1LL << 31)) return g_err.fail("%s: too many tokens", who);
    if (R < 0 || R > D || R % (neighbours ? 8 : 16))
        return g_err.fail("%s: rotated dims must be a multiple of %d up to the head dim", who,
                          neighbours ? 8 : 16);
    if (!(eps >= 0.f) || !(eps < INFINITY))
        return g_err.fail("%s: eps must be finite and not negative", who);
    if (B == 0 || S == 0 || Hq + Hk == 0) return 0;
    if ((Hq && (!q || !q_out || !q_strides || !q_out_strides)) ||
        (Hk && (!k || !k_out || !k_strides || !k_out_strides)) || (R && (!cos || !sin)) ||
        (positions && !p_strides))
        return g_err.fail("%s: null argument", who);
    if (R && (N <= 0 || angle_stride < 0 || angle_stride % 4 || !aligned(cos, 16) || !aligned(sin, 16)))
        return g_err.fail("%s: angles need rows, 16-byte aligned ones", who);
    if (R && !positions && N < S) return g_err.fail("%s: fewer rows of angles than tokens", who);
    const void* ptrs[4] = {q, k, q_out, k_out};
    const long long* strides[4] = {q_strides, k_strides, q_out_strides, k_out_strides};
    for (int i = 0; i < 4; ++i) {
        const int H = i % 2 ? Hk : Hq;
        if (!H) continue;
        if (!aligned(ptrs[i], 16)) return g_err.fail("%s: rows must be 16-byte aligned", who);
        for (int j = 0; j < 3; ++j)
            if (strides[i][j] < 0 || strides[i][j] % 8)
                return g_err.fail("%s: strides must be non-negative multiples of 8 elements", who);
        const long long e[3] = {B, S, H};
        if (i >= 2 && !rows_apart(strides[i], e, 3, D))
            return g_err.fail("%s: rows of the results overlap", who);
    }
    int L = 1;
    while (8 * L < D) L *= 2;
    RotateArgs a{};
    const int rg = 64 / L;
    // Rows of a wave are a token's heads, or a head's tokens where those lie closer or where heads would
    // leave places empty, in the wave or in what is in flight. [B, S, H, D] of 40 M numbers, heads
    // against tokens: D 64, 16 and 4 heads 60 us, 34, 32 and 8 heads 42 us, 33; D 128, 16 and 4 heads
    // 48 us, 38, 32 and 8 heads 33 us, 36. One head: 334 us against 96, and 55 with four tokens in flight.
    const long long* st = Hq ? q_strides : k_strides;
    const long long tokens = (long long)B * S;
    auto filled = [&](int H) {
        return !H || (H >= std::max(2 * rg, kUnroll) && 8 * H >= 7 * ((H + rg - 1) / rg * rg));
    };
    const bool by_token = tokens >= rg && (st[1] < st[2] || !filled(Hq) || !filled(Hk));
    // Four tokens a lane in flight, where there is one head a token, of which one round is too little, and
    // tokens enough for as many waves. 40 M numbers, us so / with one token, neighbours and halves, in a projection
    // with far positions: D 40, 1 head of q and k each 62 75 / 84 94, D 128 46 55 / 58 65, 2 heads each 55 62 /
    // 50 55, 39 46 / 37 41, 3 heads 63 64 / 41 44, 37 43 / 33 33, 4 and 1 57 65 / 44 49, 38 47 / 34 38. One head
    // of 128, 15625 tokens 8.1 / 11.8, 7812 tokens 6.1 / 6.7.
    const int most_heads = std::max(Hq, Hk);
    const bool four = by_token && most_heads == 1 && tokens >= 1024LL * rg;
    a.tok_step = by_token;
    a.head_step = by_token ? 0 : 1;
    a.head_next = by_token ? 1 : rg;
    const int set = by_token ? (four ? 4 : 1) * rg : 1;  // tokens of a wave
    a.groups = (unsigned)((tokens + set - 1) / set);
    // Rounds of a wave: as many as keep 4096 waves (16 a CU) busy, what is in flight at once at least.
    const int most = (most_heads + a.head_next - 1) / a.head_next, once = four ? 1 : kUnroll;
    const long long rounds_all = a.groups * (long long)((Hq + Hk + a.head_next - 1) / a.head_next);
    const int rounds = (int)std::min<long long>(
        most, rounds_all < 4096 ? 1 : std::max<long long>(once, rounds_all / 4096 / once * once));
    a.heads = rounds * a.head_next;
    a.part[0] = Rows{q, q_out, q_weight, 0, 0, 0, 0, 0, 0, Hq, (Hq + a.heads - 1) / a.heads};
    a.part[1] = Rows{k, k_out, k_weight, 0, 0, 0, 0, 0, 0, Hk, (Hk + a.heads - 1) / a.heads};
    for (int i = 0; i < 2; ++i) {
        if (!a.part[i].H) continue;
        a.part[i].xb = strides[i][0], a.part[i].xs = strides[i][1], a.part[i].xh = strides[i][2];
        a.part[i].yb = strides[i + 2][0], a.part[i].ys = strides[i + 2][1];
        a.part[i].yh = strides[i + 2][2];
    }
    a.cos = cos;
    a.sin = sin;
    a.ab = angle_stride;
    a.pos = R ? positions : nullptr;
    if (a.pos) a.pb = p_strides[0], a.ps = p_strides[1];
    a.B = (unsigned)B;
    a.S = (unsigned)S;
    a.N = (unsigned)std::max(N, 0);
    a.D = D;
    a.R = R;
    a.w32 = weight_f32;
    a.eps = eps;
    a.inv_d = 1.f / D;
    const long long tasks = a.groups * (long long)(a.part[0].chunks + a.part[1].chunks);
    const long long grid = (tasks + 3) / 4;
    if (!launchable(grid, 256)) return g_err.fail("%s: too many rows for one call", who);
    auto go = [&](auto t) {
        using T = decltype(t);
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, stream, a);
        };
        auto pick = [&](auto lanes) {
            constexpr int l = decltype(lanes)::value;
            if (four)
                neighbours ? run(norm_rotate_kernel<T, l, true, 4>) : run(norm_rotate_kernel<T, l, false, 4>);
            else
                neighbours ? run(norm_rotate_kernel<T, l, true, 1>) : run(norm_rotate_kernel<T, l, false, 1>);
        };
        switch (L) {
            case 1: return pick(std::integral_constant<int, 1>{});
            case 2: return pick(std::integral_constant<int, 2>{});
            case 4: return pick(std::integral_constant<int, 4>{});
            case 8: return pick(std::integral_constant<int, 8>{});
            case 16: return pick(std::integral_constant<int, 16>{});
            case 32: return pick(std::integral_constant<int, 32>{});
            default: return pick(std::integral_constant<int, 64>{});
        }
    };
    dtype == KV8_DTYPE_F16 ? go(f16{}) : go(bf16{});
    return g_err.launched(who, hipGetLastError());
}
