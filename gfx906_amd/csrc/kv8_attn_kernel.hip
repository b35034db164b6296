// Attention over the 8-bit cache (gfx906_amd_attn.h) for AMD MI355X (gfx950).
//
// How the work is dealt out is that of the 4-bit cache (kv4_kernel.hip, paged.h): few query
// rows in equal runs of 64-token units, prompts in tiles of 256 rows, short ones of 128. The codes are laid
// out for the matrix products: 16 bytes of a key are 16 dims, 16 bytes of V are 16 tokens of a
// dim, in the order that both products have them in, so that the few-row kernel's operands
// come straight from memory, and the prompt kernel stores its tiles operand by operand.
//
// The softmax weights are rounded to the element type, as the second product's instructions take them (fp32
// ones run at a sixteenth of the rate), and the sum that a result is divided by is that of the rounded ones:
// results are 1.17 to 1.33 times as far from 64 bits as with fp32 weights (norms of whole results, whose own
// rounding is most of both). The lse is summed from unrounded weights.
#include "kv8.h"

#include <algorithm>
#include <type_traits>

#include "longctx_tile.h"
#include "paged.h"

namespace {

using namespace gfx906_amd::kv8;
static_assert(kMaxRequests == kPagedRequests);

struct AttnArgs {
    const void* q;
    void* o;
    float* lse;  // [T][Hq] or NULL
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
    float* ws_ml;       // [slot][row][4]: max, sum of rounded and of unrounded weights
    // The same of attn_prompt_kernel, and its plan.
    int p_groups, p_tiles;  // p_tiles: room for so many tiles
    int* p_first;         // [B + 1]: first tile of every request
    long long* p_cost;    // [tiles + 1]: units before a tile, of one kv head
    int* p_req;           // [tiles]: request of a tile
    float* p_o;
    float* p_ml;
};

#if defined(__HIP_DEVICE_COMPILE__)
// Natural logarithm of the sum of a row's weights: max m in log2 units, sum l relative to it.
__device__ __forceinline__ float lse_of(float m, float l) {
    return l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// V codes of a block of which some rows do not see all keys: a weight of 0 would not keep a NaN out
// of the sum of a row that does not see it. NaN codes become 0; whether there were any (in the wave).
template <int D>
__device__ __forceinline__ bool strip_nans(u32x4 (&vc)[D / 16]) {
    unsigned any = 0;
#pragma unroll
    for (int ob = 0; ob < D / 16; ++ob)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned n = nan_bytes(vc[ob][e]);
            any |= n;
            vc[ob][e] &= ~((n >> 7) * 255u);
        }
    return __any(any);
}

// Afterwards: the sums of the rows that see a NaN of the block (its codes at vp, of this lane) become
// NaN. Which do is a product too, of who sees what with what is NaN.
template <int D, class T, int NB>
__device__ __forceinline__ void give_nans(const uint8_t* vp, f32x4 (&oacc)[D / 16][NB], int key0,
                                          const int (&lim)[NB], int g) {
    using x8 = typename Elem<T>::x8;
    x8 sees[2][NB];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sees[half][nb][e] =
                    (T)(key0 + 32 * half + 16 * (e / 4) + 4 * g + (e & 3) < lim[nb] ? 1.f : 0.f);
#pragma unroll
    for (int ob = 0; ob < D / 16; ++ob) {
        u32x4 x = *reinterpret_cast<const u32x4*>(vp + ob * 16 * kBlock);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (nan_bytes(x[e]) >> 7) * 0x38u;  // 1.0
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            f32x4 count = {};
#pragma unroll
            for (int half = 0; half < 2; ++half)
                count = Elem<T>::mma16(expand<T>(x[2 * half], x[2 * half + 1], 1.f), sees[half][nb],
                                       count);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (count[e] > 0.f) oacc[ob][nb][e] = NAN;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
#endif

// Attention of requests with few query rows (single tokens, drafts), bound by the bytes of the
// cache.
//
// Work is counted in units of 64 tokens of one kv head of one request (and of one tile of 16 NB
// query rows), laid end to end over the requests; every workgroup takes an equal run, its eight
// waves every eighth unit of a head, merged through LDS. A head that lies in one run is finished
// there; of others each run writes unnormalised O and its statistics to a slot of the workspace
// (2 w + 1 of workgroup w for the run that begins the head, 2 w for the others), which
// few_combine_kernel merges. DIRECT: short tables. One workgroup a head, no runs, no second kernel.
//
// A wave reads a unit's keys as 16 bytes a lane: those of lane group g are dims 64 j + 16 g .. of
// key l%16, two steps' operands once they are expanded (Q has the same dims in the same steps).
// V's 16 bytes are tokens of dim l%16 of 16, which is where the first product leaves their weights.
// The next unit's K codes are loaded once the scores of one are done, its V codes at the end.
//
// 32 requests of 100 .. 16384 tokens, 8 kv heads of 128, one query each: 36.8 us (193 MB: 5.3 TB/s) and 4.6
// for the merge; 131072 tokens, 2 kv heads, 32 rows: 18.9 and 5.0, of which the bytes take 11, a run's start
// 4 and the waves' merge 2; 1024 tokens, 16 heads of 64, in DIRECT: 6.2.
template <int D, class T, int NB, bool DIRECT, bool LSE>
__global__ void __launch_bounds__(512, D == 64 && NB == 1 ? 4 : 2) attn_few_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using W = Tile<D, T, NB, false, LSE>;
    using x8 = typename W::x8;
    constexpr int R = 16 * NB, NJ = D / 64, NW = 8, NT = 64 * NW;
    __shared__ __attribute__((aligned(1024))) float stage[NW][R * D];
    __shared__ float ml_s[NW][R][3];
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
    // Up to 64 requests every lane keeps one, and no wave waits for another to find its run.
    const bool few = a.B <= 64;
    Request mine{};
    auto get = [&](int x) __attribute__((always_inline)) {
        if (!few) return request(a, x);
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, x); };
        Request r;
        r.first = of(mine.first);
        r.n = of(mine.n);
        r.m = of(mine.m);
        r.len = of((int)mine.len);  // (an int is where it comes from)
        r.keys = of(mine.keys);
        return r;
    };
    if constexpr (!DIRECT) {
        auto upto = [&](int sum) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(sum, o);
                if (lane >= o) sum += x;
            }
            return sum;
        };
        auto run = [&](int all) {
            const int per =
                max(a.min_units, uni((int)((unsigned)(all + a.groups - 1) / (unsigned)a.groups)));
            // (the last run may end past 2^31 before it is cut)
            const long long lo = (long long)blockIdx.x * per;
            u0 = (int)min(lo, (long long)all);
            hi = (int)min((long long)all, lo + per);
            return per;
        };
        if (few) {
            int n = 0;
            if (lane < a.B) {
                mine = request(a, lane);
                n = count(units_of(mine));
            }
            const int sum = upto(n), per = run(uni(__shfl(sum, 63)));
            if (blockIdx.x == 0 && wave == 0) {
                if (lane < a.B) a.starts[lane] = sum - n;
                if (lane == 0) a.starts[a.B] = per;
            }
            if (u0 >= hi) return;
            b = uni((int)__ffsll(__ballot(sum > u0)) - 1);
            start = __builtin_amdgcn_readlane(sum - n, b);
        } else {
            const int per_run = (a.B + NT - 1) / NT;
            int n = 0;
            for (int x = tid * per_run; x < min(a.B, (tid + 1) * per_run); ++x)
                n += count(units_of(request(a, x)));
            int sum = upto(n);
            if (lane == 63) ml_s[wave][0][0] = __int_as_float(sum);
            __syncthreads();
            for (int w = 0; w < wave; ++w) sum += __float_as_int(ml_s[w][0][0]);
            run0[tid + 1] = sum;
            if (tid == 0) run0[0] = 0;
            __syncthreads();
            const int per = run(run0[NT]);
            if (blockIdx.x == 0) {
                n = run0[tid];
                for (int x = tid * per_run; x < min(a.B, (tid + 1) * per_run); ++x) {
                    a.starts[x] = n;
                    n += count(units_of(request(a, x)));
                }
                if (tid == 0) a.starts[a.B] = per;
            }
            if (u0 >= hi) return;
            if (run0[tid] <= u0 && u0 < run0[tid + 1]) found = tid;
            __syncthreads();
            b = uni(found) * per_run;
            start = uni(run0[uni(found)]);
        }
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
            req = get(b);
            Units un = units_of(req);
            while (start + count(un) <= u0) {
                start += count(un);
                req = get(++b);
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
            const T* q = (const T*)a.q + (req.first + tok) * a.qt + h * a.qh + 16 * g;
#pragma unroll
            for (int n = 0; n < W::NQ; ++n) {
                u32x4 x = {};
                if (ok) x = *reinterpret_cast<const u32x4*>(q + 64 * (n / 2) + 8 * (n % 2));
                w.qf[nb][n] = __builtin_bit_cast(x8, x ^ neg);
            }
        }
        // Keys every row of the tile sees.
        const int all_see = uni(seen_by(a, req, rt * R / a.G));

        const ConstInts table = (ConstInts)(a.table + b * a.table_stride);
        const int shift = a.c.page == 64 ? 0 : a.c.page == 128 ? 1 : 2;
        // (past the run: its last unit's page, which is not used)
        auto page_of = [&](int c) { return table[min(c, c1 - 1) >> shift]; };
        // (a page outside the cache reads page 0, and the unit's keys are masked)
        auto block_of = [&](int c, int page) {
            const unsigned p = (unsigned)page < (unsigned)a.c.pages ? page : 0;
            return block_at(a.c, p, hk, c & ((1 << shift) - 1));
        };
        // Up to 16 rows read the cache once, past the caches' lines in use (32 requests of 100 .. 16384
        // tokens 40.9 us and not 44.1); more rows are several tiles, which find it there.
        auto codes = [](const uint8_t* p) __attribute__((always_inline)) {
            const u32x4* q = reinterpret_cast<const u32x4*>(p);
            return NB == 1 ? __builtin_nontemporal_load(q) : *q;
        };
        u32x4 kc[4][NJ], vc[W::NO];
        float ks = 0.f, vs = 0.f;
        const int koff = i * D + 16 * g, voff = i * kBlock + 16 * g;
        auto fetch_k = [&](int c, int page) __attribute__((always_inline)) {
            const long long blk = block_of(c, page);
            ks = ((ConstFloats)a.c.ks)[blk];
            const uint8_t* p = a.c.kc + blk * (kBlock * D);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    kc[t][j] = codes(p + (koff + t * 16 * D + 64 * j));
        };
        auto fetch_v = [&](int c, int page) __attribute__((always_inline)) {
            const long long blk = block_of(c, page);
            vs = ((ConstFloats)a.c.vs)[blk];
            const uint8_t* p = a.c.vc + blk * (kBlock * D);
#pragma unroll
            for (int ob = 0; ob < W::NO; ++ob)
                vc[ob] = codes(p + (voff + ob * 16 * kBlock));
        };
        int c = c0 + wave, page = -1, next = -1;
        bool nans = false;
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
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) S[t / 2][t % 2][nb] = f32x4{};
#pragma unroll
            for (int n = 0; n < W::NQ; ++n)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const u32x4 x = kc[t][n / 2];
                    const x8 kf = expand<T>(x[2 * (n % 2)], x[2 * (n % 2) + 1], ks);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        S[t / 2][t % 2][nb] = Elem<T>::mma16(kf, w.qf[nb][n], S[t / 2][t % 2][nb]);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (c + NW < c1) fetch_k(c + NW, page);
            const int key0 = c * 64;
            if (key0 + 64 > all_see || !ok) {
                int lim2[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) lim2[nb] = ok ? lim[nb] : 0;
#pragma unroll
                for (int half = 0; half < 2; ++half) w.mask(S[half], key0 + 32 * half, lim2, g);
                nans |= strip_nans<D>(vc) && ok;
            }
            const float s = ok ? vs : 1.f;  // (a scale that is NaN would reach every row)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                x8 P[NB];
                w.softmax(S[half], P, a.scale);
#pragma unroll
                for (int ob = 0; ob < W::NO; ++ob) {
                    const x8 vf = expand<T>(vc[ob][2 * half], vc[ob][2 * half + 1], s);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        w.oacc[ob][nb] = Elem<T>::mma16(vf, P[nb], w.oacc[ob][nb]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (c + NW < c1) fetch_v(c + NW, page);
        }
        if (__builtin_expect(nans, 0)) {
            for (c = c0 + wave; c < c1; c += NW) {
                const int page = page_of(c);
                if (c * 64 + 64 <= all_see || (unsigned)page >= (unsigned)a.c.pages) continue;
                give_nans<D, T, NB>(a.c.vc + block_of(c, page) * (kBlock * D) + voff, w.oacc, c * 64, lim,
                                    g);
            }
        }

        // Merge the waves: all rows through LDS, each wave's relative to its own max. (Barriers wait for
        // LDS accesses only, not for the stores of partial results.)
        auto* const buf = (GFX906_LDS float*)stage[wave];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float l = quad_sum(w.lacc[nb][0]);
            float lu = l;
            if constexpr (LSE) lu = quad_sum(w.lsum[nb]);
            if (g == 0) {
                ml_s[wave][16 * nb + i][0] = w.m[nb];
                ml_s[wave][16 * nb + i][1] = l;
                ml_s[wave][16 * nb + i][2] = lu;
            }
#pragma unroll
            for (int ob = 0; ob < W::NO; ++ob)
                *reinterpret_cast<GFX906_LDS f32x4*>(buf + (16 * nb + i) * D +
                                                     ((16 * ob + 4 * g) ^ (4 * i & (D - 4)))) =
                    w.oacc[ob][nb];
        }
        lds_barrier();
        const int n_rows = min(R, rows - rt * R);
#pragma unroll 1
        for (int e = tid; e < n_rows * (D / 4); e += NT) {
            const int r = e / (D / 4), d = (e - r * (D / 4)) * 4, x = d ^ (4 * (r & 15) & (D - 4));
            f32x4 acc = {};
            float mr = kNoMax, lr = 0.f, lu = 0.f;
#pragma unroll
            for (int y = 0; y < NW; ++y) mr = max2(mr, ml_s[y][r][0]);
#pragma unroll
            for (int y = 0; y < NW; ++y) {
                const float f = __builtin_amdgcn_exp2f(ml_s[y][r][0] - mr);
                lr += ml_s[y][r][1] * f;
                lu += ml_s[y][r][2] * f;
                acc += *reinterpret_cast<const GFX906_LDS f32x4*>((const GFX906_LDS float*)stage[y] +
                                                                  r * D + x) * f;
            }
            if (whole) {
                const int row = rt * R + r, tok = row / a.G, h = hk * a.G + row - tok * a.G;
                T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + d;
                acc *= lr != 0.f ? 1.f / lr : 0.f;
                const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
                *reinterpret_cast<u32x2*>(o) =
                    u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
                if (LSE && d == 0) a.lse[(long long)(req.first + tok) * a.Hq + h] = lse_of(mr, lu);
            } else {
                *reinterpret_cast<f32x4*>(a.ws_o + (slot * R + r) * D + d) = acc;
                if (d == 0)
                    *reinterpret_cast<f32x4*>(a.ws_ml + (slot * R + r) * 4) = f32x4{mr, lr, lu, 0.f};
            }
        }
        lds_barrier();
    }
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// Merges the slots of a head that lies in several runs, and writes the zeros of a request
// without tokens: query row `row` of kv head hk of request b, by a workgroup of NT threads.
template <int D, class T, int NB, int NT, bool LSE>
__device__ __forceinline__ void few_combine(const AttnArgs& a, int b, int hk, int row) {
    constexpr int R = 16 * NB, DQ = D / 4, NG = NT / DQ, NW = NT / 64;
    __shared__ f32x4 acc_s[NW][DQ];
    __shared__ float ml_s[NW][3];
    const Request req = request(a, b);
    const long long rows = (long long)req.m * a.G;
    if (rows > a.few_rows || row >= rows) return;
    const int tok = row / a.G, h = hk * a.G + row - tok * a.G;
    const int grp = threadIdx.x / DQ, d = (threadIdx.x - grp * DQ) * 4;
    T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + d;
    const int chunks = (req.keys + 63) / 64, tiles = (int)((rows + R - 1) / R), rt = row / R;
    float* const lse = LSE ? a.lse + (long long)(req.first + tok) * a.Hq + h : nullptr;
    if (chunks == 0) {
        if (grp == 0) *reinterpret_cast<u32x2*>(o) = u32x2{};
        if (LSE && threadIdx.x == 0) *lse = -INFINITY;
        return;
    }
    const int per = a.starts[a.B];
    const int s = a.starts[b] + (hk * tiles + rt) * (chunks + a.start_units) + a.start_units;
    const int w0 = (int)((unsigned)s / (unsigned)per);
    const int w1 = (int)((unsigned)(s + chunks - 1) / (unsigned)per);
    if (w0 == w1) return;
    float m = kNoMax, l = 0.f, lu = 0.f;
    f32x4 acc = {};
    constexpr int U = 4;
    for (int x = w0 + grp; x <= w1; x += NG * U) {
        f32x4 ml[U];
        f32x4 p[U];
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int y = x + n * NG;
            ml[n] = f32x4{kNoMax, 0.f, 0.f, 0.f};
            p[n] = f32x4{};
            if (y <= w1) {
                const long long at = (2LL * y + (y == w0 ? 1 : 0)) * R + (row - rt * R);
                ml[n] = *reinterpret_cast<const f32x4*>(a.ws_ml + at * 4);
                p[n] = *reinterpret_cast<const f32x4*>(a.ws_o + at * D + d);
            }
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const float mn = max2(m, ml[n][0]);
            const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(ml[n][0] - mn);
            acc = acc * f + p[n] * e;
            l = l * f + ml[n][1] * e;
            lu = lu * f + ml[n][2] * e;
            m = mn;
        }
    }
    // The groups of a wave, then the waves.
#pragma unroll
    for (int step = DQ; step < 64; step <<= 1) {
        const float mo = __shfl_xor(m, step), lo = __shfl_xor(l, step), mn = max2(m, mo);
        const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(mo - mn);
        l = l * f + lo * e;
        if constexpr (LSE) lu = lu * f + __shfl_xor(lu, step) * e;
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
            ml_s[wave][2] = lu;
        }
    }
    __syncthreads();
    if (grp) return;
    float mx = kNoMax;
#pragma unroll
    for (int n = 0; n < NW; ++n) mx = max2(mx, ml_s[n][0]);
    acc = f32x4{};
    l = lu = 0.f;
#pragma unroll
    for (int n = 0; n < NW; ++n) {
        const float f = __builtin_amdgcn_exp2f(ml_s[n][0] - mx);
        acc += acc_s[n][d / 4] * f;
        l += ml_s[n][1] * f;
        lu += ml_s[n][2] * f;
    }
    acc *= l != 0.f ? 1.f / l : 0.f;
    const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
    *reinterpret_cast<u32x2*>(o) =
        u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
    if (LSE && d == 0) *lse = lse_of(mx, lu);
}
#endif

// grid: requests x kv heads, query rows.
template <int D, class T, int NB, int NT, bool LSE>
__global__ void __launch_bounds__(NT) few_combine_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int b = blockIdx.x / a.c.Hkv;
    few_combine<D, T, NB, NT, LSE>(a, b, blockIdx.x - b * a.c.Hkv, blockIdx.y);
#endif
}

// Attention of requests with many query rows, bound by the matrix rate.
//
// A tile is 32 NW query rows of a kv head (a token's G heads beside each other), 32 a wave; its keys
// come in chunks of 64. The tiles' chunks are laid end to end and every workgroup takes an equal run;
// prompt_combine_kernel merges tiles that lie in several runs. A chunk's codes are loaded by all
// threads two chunks ahead, expanded on the way to LDS into the operands of both products, and then
// used as attn_prompt_kernel of the 4-bit cache does: the second product of one block of 32 keys and
// the first product of the next but one around the softmax of the block between, one barrier a chunk.
//
// 3 prompts of 77 .. 2111 queries behind 300 .. 8192 tokens, 16/4 heads of 128: 166 us (173 GFLOP: 1044
// TFLOP/s; a library product of 8192 reaches 1240). The matrix pipe is busy for 44 % of the clocks, the
// vector unit for 38, LDS for 36, without bank conflicts.
//
// SELF: few tiles. Every workgroup adds up the tiles itself instead of a kernel before this one.
template <int D, class T, int NW, bool SELF, bool LSE>
__global__ void __launch_bounds__(64 * NW, 2) attn_prompt_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using W = Tile<D, T, 2, true, LSE>;
    using x8 = typename W::x8;
    constexpr int BYTES = 64 * W::RB, HALF = BYTES / 2, NT = 64 * NW, ROWS = 32 * NW;
    // 16 bytes of codes a thread of K and of V, NX times; where there are threads enough (ALONE), of
    // one of them.
    constexpr int LOADS = 2 * 64 * D / 16;  // of a chunk
    constexpr bool ALONE = LOADS <= NT;
    constexpr int NX = ALONE ? 1 : LOADS / (2 * NT), FAR = 16 * NT;
    __shared__ __attribute__((aligned(1024))) char ka[BYTES];
    __shared__ __attribute__((aligned(1024))) char kb[BYTES];
    __shared__ __attribute__((aligned(1024))) char va[BYTES];
    __shared__ __attribute__((aligned(1024))) char vb[BYTES];
    __shared__ int found, nans;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

    __shared__ int first_s[SELF ? kSelfRequests + 1 : 1];
    __shared__ long long cost_s[SELF ? kSelfTiles + 1 : 1], sum_s[NW];
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
        const long long n = scan(tid < a.B ? tiles_of<ROWS>(a, request(a, tid)) : 0);
        if (tid < kSelfRequests) first_s[tid + 1] = (int)min(n, (long long)a.p_tiles);
        if (tid == 0) first_s[0] = 0;
        __syncthreads();
        const int nt = first_s[a.B];
        constexpr int PER = kSelfTiles / NT;
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
            const int chunks = tile_chunks<ROWS>(a, request(a, lo), t - first_s[lo]);
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
        if (tid == NT - 1) cost_s[nt] = at;
        if (blockIdx.x == 0) {
            for (int x = tid; x <= a.B; x += NT) a.p_first[x] = first_s[x];
            if (tid == NT - 1) a.p_cost[nt] = at;
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
    for (int x = tid; x < a.B; x += NT)
        if (p_cost(p_first(x)) * a.c.Hkv <= u0 && u0 < p_cost(p_first(x + 1)) * a.c.Hkv) found = x;
    __syncthreads();
    int b = uni(found);
    int t0 = uni(p_first(b)), t1 = uni(p_first(b + 1));
    long long base = p_cost(t0), each = p_cost(t1) - base;
    int hk = uni((int)((u0 - base * a.c.Hkv) / each));
    {
        const long long at = u0 - base * a.c.Hkv - hk * each;
        __syncthreads();
        for (int x = t0 + tid; x < t1; x += NT)
            if (p_cost(x) - base <= at && at < p_cost(x + 1) - base) found = x;
        __syncthreads();
    }
    int tile = uni(found);

    // Where this thread's codes of a chunk go in LDS: of K 16 dims of a key, of V 16 tokens of a dim,
    // which are two operands'; the next ones lie FAR bytes further on.
    const bool has_v = !ALONE || tid >= NT / 2, has_k = !ALONE || !has_v;
    const int slot16 = ALONE ? tid & (NT / 2 - 1) : tid;
    auto kst = [&](int x) {
        const int u = slot16 + x * NT, key = u / (D / 16), unit = u % (D / 16);
        return (key / 32) * HALF + (4 * (unit >> 2) + (key >> 4 & 1)) * 1024 +
               16 * frag_slot(key & 15, unit & 3, unit >> 2);
    };
    auto vst = [&](int x) {
        const int u = slot16 + x * NT;
        return (u / 64) * 1024 + 16 * frag_slot(u / 4 & 15, u & 3, 0);
    };

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
        const int end = uni(tile_end<ROWS>(a, req, rt)), chunks = (end + 63) / 64;
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
        const long long row0 = (long long)rt * ROWS + wave * 32;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const long long r = row0 + 16 * nb + i;
            const int tok = (int)(r / a.G), h = hk * a.G + (int)(r - (long long)tok * a.G);
            lim[nb] = r < rows ? seen_by(a, req, tok) : 0;
            const T* q = (const T*)a.q + (req.first + tok) * a.qt + h * a.qh + 16 * g;
#pragma unroll
            for (int n = 0; n < W::NQ; ++n) {
                u32x4 x = {};
                if (r < rows) x = *reinterpret_cast<const u32x4*>(q + 64 * (n / 2) + 8 * (n % 2));
                w.qf[nb][n] = __builtin_bit_cast(x8, x ^ neg);
            }
        }
        const bool active = row0 < rows;  // (wave-uniform)
        const int all_see = active ? uni(seen_by(a, req, (int)(row0 / a.G))) : 0;
        // (of the tile: every row sees the chunks in front of it)
        const int tile_see = uni(seen_by(a, req, (int)((long long)rt * ROWS / a.G)));

        const ConstInts table = (ConstInts)(a.table + b * a.table_stride);
        const int shift = a.c.page == 64 ? 0 : a.c.page == 128 ? 1 : 2;
        auto page_of = [&](int c) { return table[min(c, c1 - 1) >> shift]; };
        auto good = [&](int c, int page) { return c < c1 && (unsigned)page < (unsigned)a.c.pages; };
        auto block_of = [&](int c, int page) {
            const unsigned p = (unsigned)page < (unsigned)a.c.pages ? page : 0;
            return block_at(a.c, p, hk, min(c, c1 - 1) & ((1 << shift) - 1));
        };
        // Codes of chunks kc (K) and vc (V), on their way to LDS.
        struct Raw {
            u32x4 kw[NX], vw[ALONE ? 1 : NX];  // (ALONE: kw is the one or the other)
            float ks, vs;
        };
        auto load = [&](int kc, int kpage, int vc, int vpage) __attribute__((always_inline)) {
            Raw r;
            const long long kb = block_of(kc, kpage), vb = block_of(vc, vpage);
            r.ks = ((ConstFloats)a.c.ks)[kb];
            r.vs = ((ConstFloats)a.c.vs)[vb];
            const uint8_t* kp = a.c.kc + kb * (kBlock * D) + 16 * slot16;
            const uint8_t* vp = a.c.vc + vb * (kBlock * D) + 16 * slot16;
            if constexpr (ALONE) {
                r.kw[0] = *reinterpret_cast<const u32x4*>(has_v ? vp : kp);
            } else {
#pragma unroll
                for (int x = 0; x < NX; ++x) {
                    r.kw[x] = *reinterpret_cast<const u32x4*>(kp + FAR * x);
                    r.vw[x] = *reinterpret_cast<const u32x4*>(vp + FAR * x);
                }
            }
            return r;
        };
        auto put = [&](char* dst, unsigned lo, unsigned hi, float s) __attribute__((always_inline)) {
            *reinterpret_cast<GFX906_LDS x8*>((GFX906_LDS char*)dst) = expand<T>(lo, hi, s);
        };
        auto put_k = [&](char* kd, const Raw& r) __attribute__((always_inline)) {
            if (!has_k) return;
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                put(kd + kst(x), r.kw[x][0], r.kw[x][1], r.ks);
                put(kd + kst(x) + 2048, r.kw[x][2], r.kw[x][3], r.ks);
            }
        };
        // V of chunk c. Where some row does not see all of it, NaN is 0 for now.
        auto put_v = [&](char* vd, int c, int page, Raw& r) __attribute__((always_inline)) {
            if (!has_v) return;
            u32x4(&vw)[NX] = ALONE ? r.kw : reinterpret_cast<u32x4(&)[NX]>(r.vw);
            if (c * 64 + 64 > tile_see || !good(c, page)) {
                unsigned any = 0;
#pragma unroll
                for (int x = 0; x < NX; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned n = nan_bytes(vw[x][e]);
                        any |= n;
                        vw[x][e] &= ~((n >> 7) * 255u);
                    }
                if (any && good(c, page)) nans = 1;
                if (!good(c, page)) r.vs = 1.f;  // (a scale that is NaN would reach every row)
            }
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                put(vd + vst(x), vw[x][0], vw[x][1], r.vs);
                put(vd + vst(x) + HALF, vw[x][2], vw[x][3], r.vs);
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
        if (tid == 0) nans = 0;
        __syncthreads();
        Raw raw0 = load(c0, g0, c0, g0), raw1 = load(c0 + 1, g1, c0, g0);
        Raw raw = load(c0 + 2, g2, c0 + 1, g1);
        put_k(ka, raw0);
        put_v(va, c0, g0, raw0);
        put_k(kb, raw1);
        for (int z = tid; z < BYTES / 16; z += NT) *reinterpret_cast<u32x4*>(vb + 16 * z) = u32x4{};
        __syncthreads();
        if (active) w.qk(ka, Sa);

        auto step = [&](int c, const char* vp, char* kc, char* vc, const char* kn)
            __attribute__((always_inline)) {
            if (active) {
                mask(Sa, c, g0, 0);
                w.turn(vp + HALF, Pb, kc + HALF, Sb, Sa, Pa, a.scale);
            }
            lds_barrier();
            // V(c+1) goes where V(c-1) was, K(c+2) where K(c) was.
            put_k(kc, raw);
            put_v(const_cast<char*>(vp), c + 1, g1, raw);
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
        if (active) w.pv(vb + HALF, Pb);
        __syncthreads();
        if (__builtin_expect(nans, 0)) {  // which rows see them
            for (int x = max(c0, tile_see / 64); x < c1; ++x) {
                const int page = page_of(x);
                if (!good(x, page)) continue;
                give_nans<D, T, 2>(a.c.vc + block_of(x, page) * (kBlock * D) + i * kBlock + 16 * g,
                                   w.oacc, x * 64, lim, g);
            }
        }

#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const long long r = row0 + 16 * nb + i;
            const float l = quad_sum(w.lacc[nb][0]);
            float lu = l;
            if constexpr (LSE) lu = quad_sum(w.lsum[nb]);
            if (r >= rows) continue;
            const long long at = slot * ROWS + wave * 32 + 16 * nb + i;
            if (!whole) {
#pragma unroll
                for (int ob = 0; ob < W::NO; ++ob)
                    *reinterpret_cast<f32x4*>(a.p_o + at * D + 16 * ob + 4 * g) = w.oacc[ob][nb];
                if (g == 0) *reinterpret_cast<f32x4*>(a.p_ml + at * 4) = f32x4{w.m[nb], l, lu, 0.f};
                continue;
            }
            const int tok = (int)(r / a.G), h = hk * a.G + (int)(r - (long long)tok * a.G);
            T* o = (T*)a.o + (req.first + tok) * a.ot + h * a.oh + 4 * g;
            if (LSE && g == 0) a.lse[(long long)(req.first + tok) * a.Hq + h] = lse_of(w.m[nb], lu);
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

// Merges the runs of a tile and writes the zeros of tiles that see no key. One workgroup per 16
// rows of a tile and kv head; behind these one per request and query row of attn_few_kernel's.
template <int D, class T, int TILE, bool LSE>
__global__ void __launch_bounds__(256) prompt_combine_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int ROWS = 16;
    const int tile = blockIdx.x / (TILE / ROWS), hk = blockIdx.y, tid = threadIdx.x;
    if (tile >= a.p_tiles) {
        const int e = blockIdx.x - a.p_tiles * (TILE / ROWS), few = e / kFewRows;
        few_combine<D, T, 2, 256, LSE>(a, few, hk, e - few * kFewRows);
        return;
    }
    const int r0 = blockIdx.x % (TILE / ROWS) * ROWS;
    const int b = a.p_req[tile];
    if (tile >= a.p_first[a.B]) return;
    const int t0 = a.p_first[b], t1 = a.p_first[b + 1], rt = tile - t0;
    const Request req = request(a, b);
    const int rows = (int)min(r0 + (long long)ROWS, (long long)req.m * a.G - (long long)rt * TILE);
    if (r0 >= rows) return;
    auto tok_of = [&](int r) { return (int)(((long long)rt * TILE + r) / a.G); };
    auto head_of = [&](int r, int tok) {
        return hk * a.G + (int)((long long)rt * TILE + r - (long long)tok * a.G);
    };
    const int end = tile_end<TILE>(a, req, rt), chunks = (end + 63) / 64;
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
            float m = kNoMax, l = 0.f, lu = 0.f;
            f32x4 acc = {};
            constexpr int U = 4;
            for (int x = w0; chunks && x <= w1; x += U) {
                f32x4 ml[U];
                f32x4 p[U];
#pragma unroll
                for (int n = 0; n < U; ++n) {
                    const int y = min(x + n, w1);
                    const long long at = (2LL * y + (y == w0 ? 1 : 0)) * TILE + r;
                    ml[n] = *reinterpret_cast<const f32x4*>(a.p_ml + at * 4);
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
                    lu = lu * f + ml[n][2] * e;
                    m = mn;
                }
            }
            acc *= l != 0.f ? 1.f / l : 0.f;
            T* o = (T*)a.o + (req.first + tok) * a.ot + head_of(r, tok) * a.oh + d;
            if (LSE && d == 0)
                a.lse[(long long)(req.first + tok) * a.Hq + head_of(r, tok)] = lse_of(m, lu);
            const auto x0 = Elem<T>::cvt2(acc[0], acc[1]), x1 = Elem<T>::cvt2(acc[2], acc[3]);
            *reinterpret_cast<u32x2*>(o) =
                u32x2{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1)};
        }
    }
#endif
}

// Units of a head's start: fewer than for the 4-bit cache, whose units are half as many bytes. us with 4 /
// 6 / 8 / 16 (codes loaded through the caches): 32 requests of 100 .. 16384 tokens, 32/8 heads of 128, 50.6 /
// 45.0 / 44.3 / 45.7; 64 of 100 .. 8000 52.2 / 46.8 / 45.5 / 49.3; 16 of 1000 .. 4000, three queries each,
// 16/4 heads, 17.5 / 17.4 / 17.2 / 19.1.
constexpr int kStart = 8;
// DIRECT reaches tables of 2048 tokens, no further with many heads: us there / in runs, 32 requests, 32/8
// heads of 128: of 4000 tokens each 49.0 / 53.0, of 100 .. 4000 26.6 / 21.6; one request of 2000 14.8 / 15.0,
// of 3000 19.8 / 15.1.
constexpr int kFar = 1;
// Waves of a prompt's tile, of 32 rows each: the more, the fewer times a chunk is expanded; but short
// prompts fill large tiles badly. us with eight / four: 3 prompts of 77 .. 2111 queries behind 300 ..
// 8192 tokens, 16/4 heads of 128, 192 / 207; one of 512 behind 16000, 8/2 heads, 64.4 / 67.9; 4 of 90 ..
// 300 behind 100 .. 1000, 8/2 heads, 37.8 / 38.7; one of 150, 4/2 heads (300 rows), 25.6 / 24.6; one of
// 300, 4/4 heads of 64, 26.9 / 22.1.
constexpr int kWaves = 8, kWavesShort = 4;
constexpr long long kLongRows = 512;
int prompt_waves(int max_q, int G) {
    return (long long)max_q * G >= kLongRows ? kWaves : kWavesShort;
}
// (eight waves a CU, as their registers allow)
PromptPlan prompt_plan8(int T, int B, int G, int D, int max_q, size_t after) {
    const int waves = prompt_waves(max_q, G);
    return prompt_plan(T, B, G, D, max_q, after, 4, 32 * waves, 256 * 8 / waves);
}

}  // namespace

extern "C" size_t kv8_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int D, int max_q,
                                           int max_len) {
    if (T <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || D <= 0 || max_q <= 0) return 0;
    const size_t few = few_plan(B, Hq / Hkv, Hkv, D, std::min(max_q, T), max_len, 4, kStart, kFar).bytes;
    const PromptPlan p = prompt_plan8(T, B, Hq / Hkv, D, std::min(max_q, T), few);
    return p.used ? p.bytes : few;
}

extern "C" int kv8_attn(const void* q, void* o, float* lse, const long long* q_strides,
                        const long long* o_strides, int dtype, int T, int B, int Hq, int Hkv, int D,
                        const void* k_codes, const float* k_scales, const void* v_codes,
                        const float* v_scales, int pages, int page, const int* table,
                        long long table_stride, int W, const int* lens, const int* cu_q, int max_q,
                        float scale, int causal, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
    LastError& err = last_error();
    err.text[0] = 0;
    if (check_cache(Hkv, D, pages, page, k_codes, k_scales, v_codes, v_scales, "kv8_attn")) return 1;
    if (dtype != KV8_DTYPE_F16 && dtype != KV8_DTYPE_BF16) return err.fail("kv8_attn: bad dtype");
    if (T < 0 || B < 0 || W < 0 || max_q < 0) return err.fail("kv8_attn: negative sizes");
    if (B > kMaxRequests) return err.fail("kv8_attn: at most %d requests", kMaxRequests);
    if (Hq <= 0 || Hq % Hkv || Hq > 65535)
        return err.fail("kv8_attn: query heads must be a multiple of kv heads");
    if (!cu_q && T != B) return err.fail("kv8_attn: without cu_q, one query a request");
    if (T == 0 || B == 0 || max_q == 0) return 0;
    if (!q || !o || !q_strides || !o_strides || !lens || (W > 0 && !table))
        return err.fail("kv8_attn: null argument");
    if ((long long)W * page >= (1LL << 31) || table_stride < 0)
        return err.fail("kv8_attn: table too wide or a negative stride");
    for (int i = 0; i < 2; ++i)
        if (q_strides[i] < 0 || q_strides[i] % 8 || o_strides[i] < 0 || o_strides[i] % 4)
            return err.fail("kv8_attn: q strides must be non-negative multiples of 8, "
                              "o strides of 4");
    if (!aligned(q, 16) || !aligned(o, 8) || !aligned(lse, 4))
        return err.fail("kv8_attn: q must be 16-byte, o 8-byte and lse 4-byte aligned");
    if (q == o) return err.fail("kv8_attn: o must not be q");
    const long long oe[2] = {T, Hq};
    if (!rows_apart(o_strides, oe, 2, D)) return err.fail("kv8_attn: o's rows overlap");
    if (!good_scale(scale)) return err.fail("kv8_attn: scale must be finite, and below 2.3e38");
    const FewPlan plan = few_plan(B, Hq / Hkv, Hkv, D, cu_q ? std::min(max_q, T) : 1, W * page, 4,
                                  kStart, kFar);
    if (plan.units >= (1LL << 30)) return err.fail("kv8_attn: table too wide for so many heads");
    const PromptPlan pp = prompt_plan8(T, B, Hq / Hkv, D, cu_q ? std::min(max_q, T) : 1, plan.bytes);
    const size_t need = pp.used ? pp.bytes : plan.bytes;
    const long long heads = (long long)B * Hkv;
    const int waves = prompt_waves(cu_q ? std::min(max_q, T) : 1, Hq / Hkv);
    const long long combines = pp.tiles * (long long)(2 * waves) +
                               (plan.direct ? 0 : (long long)B * kFewRows);
    if (!(plan.direct ? launchable(heads * plan.tiles, 512)
                      : launchable(heads, plan.many ? 1024 : 256)) ||
        (pp.used && !launchable(combines, 256)))
        return err.fail("kv8_attn: too many requests, heads or query rows for one call");
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return err.fail("kv8_attn: workspace misaligned or smaller than "
                          "kv8_attn_workspace_bytes()");
    AttnArgs a{};
    a.q = q;
    a.o = o;
    a.lse = lse;
    a.qt = q_strides[0];
    a.qh = q_strides[1];
    a.ot = o_strides[0];
    a.oh = o_strides[1];
    a.c = Cache{(const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                pages, page, Hkv, D};
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
    auto go = [&](auto d, auto t, auto with_lse) {
        constexpr int kD = decltype(d)::value;
        constexpr bool L = decltype(with_lse)::value;
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
            direct(attn_few_kernel<kD, E, 1, true, L>);
        else if (plan.direct)
            direct(attn_few_kernel<kD, E, 2, true, L>);
        else if (plan.nb == 1)
            runs(attn_few_kernel<kD, E, 1, false, L>, few_combine_kernel<kD, E, 1, 256, L>,
                 few_combine_kernel<kD, E, 1, 1024, L>);
        else
            runs(attn_few_kernel<kD, E, 2, false, L>, few_combine_kernel<kD, E, 2, 256, L>,
                 few_combine_kernel<kD, E, 2, 1024, L>);
        auto prompts = [&](auto waves) {
            constexpr int kW = decltype(waves)::value, kRows = 32 * kW;
            if (pp.self) {
                hipLaunchKernelGGL((attn_prompt_kernel<kD, E, kW, true, L>), dim3(pp.groups),
                                   dim3(64 * kW), 0, stream, a);
            } else {
                hipLaunchKernelGGL((prompt_plan_kernel<kRows, AttnArgs>), dim3(1), dim3(1024), 0, stream,
                                   a);
                hipLaunchKernelGGL((attn_prompt_kernel<kD, E, kW, false, L>), dim3(pp.groups),
                                   dim3(64 * kW), 0, stream, a);
            }
            hipLaunchKernelGGL((prompt_combine_kernel<kD, E, kRows, L>), dim3((unsigned)combines, Hkv),
                               dim3(256), 0, stream, a);
        };
        if (!pp.used) return;
        waves == kWaves ? prompts(std::integral_constant<int, kWaves>{})
                        : prompts(std::integral_constant<int, kWavesShort>{});
    };
    auto by_dim = [&](auto t, auto with_lse) {
        D == 64 ? go(std::integral_constant<int, 64>{}, t, with_lse)
                : go(std::integral_constant<int, 128>{}, t, with_lse);
    };
    auto by_type = [&](auto with_lse) {
        dtype == KV8_DTYPE_F16 ? by_dim(f16{}, with_lse) : by_dim(bf16{}, with_lse);
    };
    lse ? by_type(std::true_type{}) : by_type(std::false_type{});
    return err.launched("kv8_attn", hipGetLastError());
}
