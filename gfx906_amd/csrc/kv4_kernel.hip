// Key/value cache in 4 bits for AMD MI355X (gfx950): pages and slots from
// request lengths, storing and reading rows, attention over the cache. The
// format and the entry points are described in gfx906_amd_kv4.h.
//
// gfx950 converts between E2M1 pairs with an E8M0 scale and fp16, bf16 or fp32
// in one instruction (v_cvt_scalef32_*), rounding to nearest even and
// saturating, so the format costs half an instruction a value to read.
#include "longctx.h"

#include <algorithm>

#include "gfx906_amd_kv4.h"

namespace {

using namespace gfx906_amd::longctx;

thread_local LastError g_err;

constexpr int kMaxRequests = KV4_MAX_REQUESTS;

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

// Every workgroup adds up all requests (each of the 256 threads a run of them,
// then a scan over the threads) and serves its share of the slots and of the
// requests' table rows. Entries that are read (held pages) and written (new
// ones) are different, so workgroups need no order.
__global__ void __launch_bounds__(256) plan_pages_kernel(const PlanArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ long long tok0[kMaxRequests + 1];  // first slot of a request
    __shared__ long long pg0[kMaxRequests + 1];   // pages taken before a request
    __shared__ long long part[2][256];
    const int t = threadIdx.x, B = a.B, P = a.page;
    const int per = (B + 255) / 256, b0 = min(B, t * per), b1 = min(B, b0 + per);
    auto held = [&](int b) { return ((long long)max(0, a.lens[b]) + P - 1) / P; };
    auto total = [&](int b) {
        return ((long long)max(0, a.lens[b]) + max(0, a.new_lens[b]) + P - 1) / P;
    };
    long long n = 0, p = 0;
    for (int b = b0; b < b1; ++b) {
        n += max(0, a.new_lens[b]);
        p += total(b) - held(b);
    }
    part[0][t] = n;
    part[1][t] = p;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
        const long long x = t >= o ? part[0][t - o] : 0, y = t >= o ? part[1][t - o] : 0;
        __syncthreads();
        part[0][t] += x;
        part[1][t] += y;
        __syncthreads();
    }
    n = part[0][t] - n;
    p = part[1][t] - p;
    for (int b = b0; b < b1; ++b) {
        tok0[b] = n;
        pg0[b] = p;
        n += max(0, a.new_lens[b]);
        p += total(b) - held(b);
    }
    if (t == 255) {
        tok0[B] = part[0][255];
        pg0[B] = part[1][255];
    }
    __syncthreads();

    const long long used = max(0, a.used[0]);
    // Page of place k of request b's row, or -1.
    auto fresh = [&](int b, long long k) -> int {
        const long long f = used + pg0[b] + (k - held(b));
        return k < a.W && f < a.n_free ? a.free_pages[f] : -1;
    };
    const int stride = gridDim.x * 256, gt = blockIdx.x * 256 + t;
    for (int s = gt; s < a.n_slots; s += stride) {
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
            const long long pos = (long long)max(0, a.lens[lo]) + (s - tok0[lo]), k = pos / P;
            const int page = k >= held(lo) ? fresh(lo, k)
                             : k < a.W     ? a.table[lo * a.table_stride + k]
                                           : -1;
            const long long at = (long long)page * P + pos % P;
            if (page >= 0 && at < (1LL << 31)) slot = (int)at;
        }
        a.slots[s] = slot;
    }
    const long long cap = 0x7fffffff;
    for (int b = gt; b <= B; b += stride) {
        a.cu_new[b] = (int)min(cap, tok0[b]);
        if (b == B) break;
        a.lens_out[b] = (int)min(cap, (long long)max(0, a.lens[b]) + max(0, a.new_lens[b]));
    }
    for (int b = gt / 64; b < B; b += stride / 64) {
        const long long last = min(total(b), (long long)a.W);
        for (long long k = held(b) + (t & 63); k < last; k += 64)
            a.table[b * a.table_stride + k] = fresh(b, k);
    }
    if (blockIdx.x == 0) {
        // Pages of columns behind the table take their place in the free list too
        // (the pages are counted as missing, and left out of *used only at its end).
        long long lost = 0;
        for (int b = b0; b < b1; ++b) {
            const long long first = used + pg0[b], need = total(b) - held(b);
            const long long in_row = max(0LL, min(need, a.W - held(b)));
            lost += need - max(0LL, min(in_row, (long long)a.n_free - first));
        }
        __syncthreads();
        part[0][t] = lost;
        __syncthreads();
        if (t == 0) {
            long long m = 0;
            for (int i = 0; i < 256; ++i) m += part[0][i];
            a.missing[0] = (int)min(cap, m);
            a.used_out[0] = (int)min(cap, max(used, min(used + pg0[B], (long long)a.n_free)));
        }
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
    long long n;  // blocks of 32 values in k (and in v)
};

// One lane per block of 32 values of k or v.
template <class T>
__global__ void __launch_bounds__(256) store_kernel(const RowArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const bool is_v = id >= a.n;
    const long long blk = is_v ? id - a.n : id;
    if (blk >= a.n) return;
    const int nb = a.c.D / 32, j = (int)(blk % nb);
    const int h = (int)(blk / nb % a.c.Hkv);
    const long long t = blk / nb / a.c.Hkv;
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.c.pages * (long long)a.c.page) return;
    const T* src = is_v ? (const T*)a.v + t * a.vt + h * a.vh : (const T*)a.k + t * a.kt + h * a.kh;
    float x[32];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        x[i] = (float)src[32 * j + i];
        top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    const unsigned e = top >> 23, byte = e == 255 ? 255 : (unsigned)max(1, (int)e - 2);
    const float s = e8m0(byte);
    unsigned w[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i], x[8 * i + 1], s, 0);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 2], x[8 * i + 3], s, 1);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 4], x[8 * i + 5], s, 2);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 6], x[8 * i + 7], s, 3);
    }
    const int page = slot / a.c.page, tok = slot % a.c.page;
    uint8_t* codes = const_cast<uint8_t*>(is_v ? a.c.vc : a.c.kc);
    uint8_t* scales = const_cast<uint8_t*>(is_v ? a.c.vs : a.c.ks);
    *reinterpret_cast<u32x4*>(codes + code_at(a.c, page, h, tok) + 16 * j) =
        u32x4{w[0], w[1], w[2], w[3]};
    scales[scale_at(a.c, page, h, tok) + 4 * j] = (uint8_t)byte;
#endif
}

template <class T>
__global__ void __launch_bounds__(256) load_kernel(const RowArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const bool is_v = id >= a.n;
    const long long blk = is_v ? id - a.n : id;
    if (blk >= a.n) return;
    const int nb = a.c.D / 32, j = (int)(blk % nb);
    const int h = (int)(blk / nb % a.c.Hkv);
    const long long t = blk / nb / a.c.Hkv;
    const int slot = a.slots[t];
    T* dst = (T*)(is_v ? a.vo : a.ko) + blk * 32;
    u32x4 w = {};
    float s = 1.f;
    if (slot >= 0 && slot < a.c.pages * (long long)a.c.page) {
        const int page = slot / a.c.page, tok = slot % a.c.page;
        w = *reinterpret_cast<const u32x4*>((is_v ? a.c.vc : a.c.kc) +
                                            code_at(a.c, page, h, tok) + 16 * j);
        s = e8m0((is_v ? a.c.vs : a.c.ks)[scale_at(a.c, page, h, tok) + 4 * j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 0);
        const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 1);
        const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 2);
        const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 3);
        const float x[8] = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[8 * i + e] = (T)x[e];
    }
#endif
}

// -- attention ------------------------------------------------------------------------

struct AttnArgs {
    const void* q;
    void* o;
    long long qt, qh, ot, oh;
    Cache c;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* cu;  // NULL: one query a request
    int W, T, B, Hq, max_q, causal;
    float scale;
};

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ int cu_at(const AttnArgs& a, int b) {
    return a.cu ? min(max(a.cu[b], 0), a.T) : b;
}
#endif

// One wave per query row and head: 64 keys at a time, a score per lane, then a
// pair of dims per lane (D = 64: one).
template <class T>
__global__ void __launch_bounds__(64) attn_rows_kernel(const AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float qs[128], ps[64];
    __shared__ long long code_s[64], scale_s[64];
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int D = a.c.D, hk = h / (a.Hq / a.c.Hkv);
    int b = -1, first = 0, n = 0;
    for (int i = 0; i < a.B; ++i) {
        const int lo = cu_at(a, i), hi = cu_at(a, i + 1);
        if (row >= lo && row < hi && b < 0) {
            b = i;
            first = lo;
            n = hi - lo;
        }
    }
    if (b < 0 || row - first >= a.max_q) return;
    const long long len = max(0, a.lens[b]);
    const long long seen = a.causal ? len - n + (row - first) + 1 : len;
    const T* q = (const T*)a.q + row * a.qt + h * a.qh;
    for (int d = lane; d < D; d += 64) qs[d] = (float)q[d];
    __syncthreads();
    float m = kNoMax, l = 0.f, o0 = 0.f, o1 = 0.f;
    const long long cols = min(seen, (long long)a.W * a.c.page);
    for (long long j0 = 0; j0 < cols; j0 += 64) {
        const long long j = j0 + lane;
        const int page = a.table[b * a.table_stride + j0 / a.c.page];
        if (page < 0 || page >= a.c.pages) continue;
        const int tok = (int)(j % a.c.page);
        const long long ca = code_at(a.c, page, hk, tok), sa = scale_at(a.c, page, hk, tok);
        float s = -INFINITY;
        if (j < seen) {
            s = 0.f;
            for (int i = 0; i < D / 8; ++i) {
                const unsigned w = *reinterpret_cast<const unsigned*>(a.c.kc + ca + 4 * i);
                const float e = e8m0(a.c.ks[sa + 4 * (i / 4)]);
                const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, e, 0);
                const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, e, 1);
                const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, e, 2);
                const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, e, 3);
                s += qs[8 * i] * p0[0] + qs[8 * i + 1] * p0[1] + qs[8 * i + 2] * p1[0] +
                     qs[8 * i + 3] * p1[1] + qs[8 * i + 4] * p2[0] + qs[8 * i + 5] * p2[1] +
                     qs[8 * i + 6] * p3[0] + qs[8 * i + 7] * p3[1];
            }
            s *= a.scale * kLog2e;
        }
        const float mn = fmaxf(m, wave_max(s)), w = exp2f(m - mn), p = exp2f(s - mn);
        l = l * w + wave_sum(p);
        o0 *= w;
        o1 *= w;
        m = mn;
        ps[lane] = p;
        code_s[lane] = ca;
        scale_s[lane] = sa;
        __syncthreads();
        if (2 * lane < D)
            for (int i = 0; i < 64 && j0 + i < seen; ++i) {
                const unsigned c = a.c.vc[code_s[i] + lane];
                const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(
                    c, e8m0(a.c.vs[scale_s[i] + 4 * (lane / 16)]), 0);
                o0 += ps[i] * x[0];
                o1 += ps[i] * x[1];
            }
        __syncthreads();
    }
    T* o = (T*)a.o + row * a.ot + h * a.oh;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    if (2 * lane < D) {
        o[2 * lane] = (T)(o0 * inv);
        o[2 * lane + 1] = (T)(o1 * inv);
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
    const int grid = (int)std::min<long long>(256, std::max<long long>(1, (work + 1023) / 1024));
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
    a.n = (long long)T * Hkv * (D / 32);
    const long long groups = (2 * a.n + 255) / 256;
    if (groups >= (1LL << 31)) return g_err.fail("kv4_store: too many rows");
    if (dtype == KV4_DTYPE_F16)
        hipLaunchKernelGGL(store_kernel<f16>, dim3((unsigned)groups), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(store_kernel<bf16>, dim3((unsigned)groups), dim3(256), 0, stream, a);
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
    a.n = (long long)T * Hkv * (D / 32);
    const long long groups = (2 * a.n + 255) / 256;
    if (groups >= (1LL << 31)) return g_err.fail("kv4_load: too many rows");
    if (dtype == KV4_DTYPE_F16)
        hipLaunchKernelGGL(load_kernel<f16>, dim3((unsigned)groups), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(load_kernel<bf16>, dim3((unsigned)groups), dim3(256), 0, stream, a);
    return g_err.launched("kv4_load", hipGetLastError());
}

extern "C" size_t kv4_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int D, int max_q,
                                           int max_len) {
    (void)T, (void)B, (void)Hq, (void)Hkv, (void)D, (void)max_q, (void)max_len;
    return 0;
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
    const long long oe[2] = {T, Hq};
    if (!rows_apart(o_strides, oe, 2, D)) return g_err.fail("kv4_attn: o's rows overlap");
    if (!(scale > -INFINITY && scale < INFINITY)) return g_err.fail("kv4_attn: scale must be finite");
    (void)workspace, (void)workspace_bytes;
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
    a.max_q = cu_q ? max_q : 1;
    a.causal = causal;
    a.scale = scale;
    if (dtype == KV4_DTYPE_F16)
        hipLaunchKernelGGL(attn_rows_kernel<f16>, dim3(T, Hq), dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL(attn_rows_kernel<bf16>, dim3(T, Hq), dim3(64), 0, stream, a);
    return g_err.launched("kv4_attn", hipGetLastError());
}
