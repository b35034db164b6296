// What the kernels of the 8-bit cache share: the cache, its codes in the element types,
// checks on the host. The format is described in gfx906_amd_attn.h. Internal.
#pragma once

#include "gfx906_amd_attn.h"
#include "longctx.h"

namespace gfx906_amd {
namespace kv8 {

using namespace longctx;

constexpr int kBlock = KV8_BLOCK;
constexpr int kMaxRequests = KV8_MAX_REQUESTS;

// The message of kv8_last_error(), of the calling thread.
LastError& last_error();

// The cache as kernels see it. A block of 64 tokens of a kv head is 64 D bytes of keys' and
// of values' codes; its number counts [page][head][block of the page]. 64-bit offsets.
struct Cache {
    const uint8_t* kc;
    const float* ks;
    const uint8_t* vc;
    const float* vs;
    int pages, page, Hkv, D;
};

inline int check_cache(int Hkv, int D, int pages, int page, const void* kc, const void* ks,
                       const void* vc, const void* vs, const char* who) {
    LastError& e = last_error();
    if (D != 64 && D != 128) return e.fail("%s: head dim must be 64 or 128", who);
    if (page != 64 && page != 128 && page != 256)
        return e.fail("%s: pages hold 64, 128 or 256 tokens", who);
    if (Hkv <= 0 || Hkv > 65535) return e.fail("%s: bad number of kv heads", who);
    if (pages < 0 || (long long)pages * page >= (1LL << 31))
        return e.fail("%s: the cache must hold fewer than 2^31 tokens", who);
    if (pages > 0 && (!kc || !ks || !vc || !vs)) return e.fail("%s: null cache", who);
    if (!aligned(kc, 16) || !aligned(vc, 16) || !aligned(ks, 4) || !aligned(vs, 4))
        return e.fail("%s: codes must be 16-byte and scales 4-byte aligned", who);
    return 0;
}

#if defined(__HIP_DEVICE_COMPILE__)
typedef const __attribute__((address_space(4))) float* ConstFloats;

__device__ __forceinline__ long long block_at(const Cache& c, long long page, int h, int part) {
    return (page * c.Hkv + h) * (c.page / kBlock) + part;
}
// Place of a block's token in a row of the values' codes.
__device__ __forceinline__ int place(int t) {
    return 16 * (t >> 2 & 3) + 8 * (t >> 5) + 4 * (t >> 4 & 1) + (t & 3);
}

// Two codes (the low or the high ones of w) times s in the element type: exact, for the scales
// that a cache has.
template <class T, bool HIGH>
__device__ __forceinline__ typename Elem<T>::x2 expand2(unsigned w, float s) {
    if constexpr (__is_same(T, f16))
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, HIGH);
    else
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HIGH);
}
template <class T>
__device__ __forceinline__ typename Elem<T>::x8 expand(unsigned lo, unsigned hi, float s) {
    auto u = [](typename Elem<T>::x2 x) { return __builtin_bit_cast(unsigned, x); };
    return __builtin_bit_cast(typename Elem<T>::x8,
                              u32x4{u(expand2<T, false>(lo, s)), u(expand2<T, true>(lo, s)),
                                    u(expand2<T, false>(hi, s)), u(expand2<T, true>(hi, s))});
}
// 0x80 in every byte of w that is a NaN code.
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
#endif

}  // namespace kv8
}  // namespace gfx906_amd
