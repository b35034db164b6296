// PyTorch binding of the 4-bit key/value cache (gfx906_amd_attn.h): kv4_plan_pages,
// kv4_store, kv4_load and kv4_attn. The Python layer (gfx906_amd.kv4) documents the
// arguments. Every op runs on the current HIP stream of its tensors' device without
// synchronising; what cannot be run raises RuntimeError.
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "bindings.h"
#include "gfx906_amd_attn.h"

namespace {

using torch::Tensor;

int dtype_of(at::ScalarType t, const char* who) {
    TORCH_CHECK(t == torch::kHalf || t == torch::kBFloat16, who, ": fp16 or bf16 needed");
    return t == torch::kBFloat16 ? KV4_DTYPE_BF16 : KV4_DTYPE_F16;
}

void check_ints(const Tensor& t, int64_t n, const c10::Device& dev, const char* who,
                const char* name) {
    TORCH_CHECK(t.device() == dev && t.dtype() == torch::kInt && t.dim() == 1 &&
                    (n < 0 || t.size(0) == n) && t.is_contiguous(),
                who, ": ", name, " must be a contiguous int32 vector of the right length on the "
                "other tensors' device");
}

// The four tensors of a cache, checked against each other.
struct Parts {
    int pages, Hkv, page, D;
    Parts(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs, const char* who) {
        TORCH_CHECK(k.is_cuda() && k.dim() == 4 && ks.dim() == 6, who,
                    ": the cache must be [pages, heads, page, D/2] codes and [pages, heads, "
                    "page/64, 16, D/32, 4] scales on a GPU");
        for (const Tensor* t : {&k, &ks, &v, &vs})
            TORCH_CHECK(t->device() == k.device() && t->dtype() == torch::kByte &&
                            t->is_contiguous(),
                        who, ": the cache must be contiguous uint8 tensors on one device");
        TORCH_CHECK(v.sizes() == k.sizes() && vs.sizes() == ks.sizes(), who,
                    ": key and value parts of the cache differ in shape");
        TORCH_CHECK(k.size(0) < (1LL << 31) && k.size(1) > 0 && k.size(1) < 65536 &&
                        k.size(2) > 0 && k.size(2) <= 256 && k.size(3) <= 256,
                    who, ": cache too large, or without heads or tokens");
        pages = (int)k.size(0);
        Hkv = (int)k.size(1);
        page = (int)k.size(2);
        D = (int)k.size(3) * 2;
        TORCH_CHECK(ks.size(0) == pages && ks.size(1) == Hkv && ks.size(2) * 64 == page &&
                        ks.size(3) == 16 && ks.size(4) * 32 == D && ks.size(5) == 4,
                    who, ": scales do not match the codes' shape");
    }
};

// [T, H, D] rows the kernels read in place: contiguous head dim, the other strides
// multiples of 8, 16-byte aligned. Anything else is copied.
Tensor rows_of(const Tensor& t) {
    const bool ok = (t.stride(2) == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(0) == 1 || (t.stride(0) >= 0 && t.stride(0) % 8 == 0)) &&
                    (t.size(1) == 1 || (t.stride(1) >= 0 && t.stride(1) % 8 == 0));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
std::array<long long, 2> strides2(const Tensor& t) {
    return {t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1)};
}

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
void check_rc(int rc) {
    TORCH_CHECK(rc == 0, "kernel: ", kv4_last_error() ? kv4_last_error() : "launch failed");
}

}  // namespace

std::vector<Tensor> kv4_plan_pages_op(Tensor lens, Tensor new_lens, Tensor table, Tensor free_pages,
                                      Tensor used, int64_t page, int64_t tokens) {
    const char* who = "plan_pages";
    TORCH_CHECK(lens.is_cuda(), who, ": lens must be on a GPU");
    const auto dev = lens.device();
    check_ints(lens, -1, dev, who, "lens");
    const int64_t B = lens.size(0);
    check_ints(new_lens, B, dev, who, "new_lens");
    check_ints(free_pages, -1, dev, who, "free_pages");
    check_ints(used, 1, dev, who, "used");
    TORCH_CHECK(table.device() == dev && table.dtype() == torch::kInt && table.dim() == 2 &&
                    table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1) &&
                    (B <= 1 || table.stride(0) >= table.size(1)),
                who, ": table must be int32 [B, W] with contiguous rows that do not overlap");
    TORCH_CHECK(B <= KV4_MAX_REQUESTS && tokens >= 0 && tokens < (1LL << 31) && page > 0 &&
                    page <= 256 && table.size(1) < (1LL << 31) && free_pages.size(0) < (1LL << 31),
                who, ": sizes out of range");
    for (const Tensor* t : {&lens, &new_lens, &free_pages, &used}) at::assert_no_overlap(table, *t);
    const c10::DeviceGuard guard(dev);
    // One buffer for every result: slots, cu_new, lens, used, missing.
    const Tensor buf = at::empty({tokens + 2 * B + 3}, lens.options());
    // (made by hand: five views through the dispatcher take 2 us of the call's 7)
    int64_t at = 0;
    auto next = [&](int64_t n) {
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()),
                                                            buf.key_set(), buf.dtype());
        t.unsafeGetTensorImpl()->set_storage_offset(at);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(n);
        at += n;
        return t;
    };
    const Tensor slots = next(tokens), cu = next(B + 1), out = next(B), u = next(1), miss = next(1);
    check_rc(kv4_plan_pages(lens.data_ptr<int>(), new_lens.data_ptr<int>(), table.data_ptr<int>(),
                            B <= 1 ? table.size(1) : table.stride(0), (int)table.size(1),
                            free_pages.data_ptr<int>(), (int)free_pages.size(0),
                            used.data_ptr<int>(), (int)B, (int)page, (int)tokens,
                            slots.data_ptr<int>(), cu.data_ptr<int>(), out.data_ptr<int>(),
                            u.data_ptr<int>(), miss.data_ptr<int>(), stream()));
    return {slots, cu, out, u, miss};
}

void kv4_store_op(Tensor k, Tensor v, Tensor slots, Tensor kc, Tensor ks, Tensor vc, Tensor vs) {
    const char* who = "store";
    const Parts c(kc, ks, vc, vs, who);
    TORCH_CHECK(k.dim() == 3 && k.size(1) == c.Hkv && k.size(2) == c.D && v.sizes() == k.sizes(),
                who, ": k and v must be [T, heads, D] of the cache's heads and head dim");
    TORCH_CHECK(k.device() == kc.device() && v.device() == kc.device() && v.dtype() == k.dtype(),
                who, ": k and v must have one dtype and the cache's device");
    TORCH_CHECK(k.size(0) < (1LL << 31), who, ": too many rows");
    const int dt = dtype_of(k.scalar_type(), who);
    check_ints(slots, k.size(0), kc.device(), who, "slots");
    const c10::DeviceGuard guard(kc.device());
    if (k.numel() == 0) return;
    const Tensor kr = rows_of(k), vr = rows_of(v);
    const auto sk = strides2(kr), sv = strides2(vr);
    check_rc(kv4_store(kr.data_ptr(), vr.data_ptr(), sk.data(), sv.data(), dt, (int)k.size(0),
                       c.Hkv, c.D, slots.data_ptr<int>(), kc.data_ptr(), ks.data_ptr(),
                       vc.data_ptr(), vs.data_ptr(), c.pages, c.page, stream()));
}

std::vector<Tensor> kv4_load_op(Tensor kc, Tensor ks, Tensor vc, Tensor vs, Tensor slots,
                                at::ScalarType dtype) {
    const char* who = "load";
    const Parts c(kc, ks, vc, vs, who);
    const int dt = dtype_of(dtype, who);
    check_ints(slots, -1, kc.device(), who, "slots");
    TORCH_CHECK(slots.size(0) < (1LL << 31), who, ": too many rows");
    const c10::DeviceGuard guard(kc.device());
    const int64_t T = slots.size(0);
    Tensor k = at::empty({T, c.Hkv, c.D}, kc.options().dtype(dtype)), v = at::empty_like(k);
    if (k.numel())
        check_rc(kv4_load(k.data_ptr(), v.data_ptr(), dt, (int)T, c.Hkv, c.D,
                          slots.data_ptr<int>(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
                          vs.data_ptr(), c.pages, c.page, stream()));
    return {k, v};
}

Tensor kv4_attn_op(Tensor q, Tensor kc, Tensor ks, Tensor vc, Tensor vs, Tensor table, Tensor lens,
                   double scale, c10::optional<Tensor> cu_q, int64_t max_q, bool causal,
                   c10::optional<Tensor> out) {
    const char* who = "attn";
    const Parts c(kc, ks, vc, vs, who);
    const auto dev = kc.device();
    TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.size(2) == c.D, who,
                ": q must be [T, heads, D] on the cache's device, with its head dim");
    const int dt = dtype_of(q.scalar_type(), who);
    check_ints(lens, -1, dev, who, "lens");
    const int64_t T = q.size(0), Hq = q.size(1), B = lens.size(0);
    TORCH_CHECK(T < (1LL << 31) && Hq < 65536 && B <= KV4_MAX_REQUESTS, who,
                ": sizes out of range");
    TORCH_CHECK(Hq > 0 && Hq % c.Hkv == 0, who, ": query heads must be a multiple of kv heads");
    if (cu_q.has_value())
        check_ints(*cu_q, B + 1, dev, who, "cu_q");
    else
        TORCH_CHECK(T == B, who, ": without cu_q, one query a request");
    TORCH_CHECK(table.device() == dev && table.dtype() == torch::kInt && table.dim() == 2 &&
                    table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1) &&
                    (B <= 1 || table.stride(0) >= 0) && table.size(1) * c.page < (1LL << 31),
                who, ": table must be int32 [B, W] with contiguous rows of fewer than 2^31 tokens");
    Tensor o;
    if (out.has_value()) {
        o = *out;
        TORCH_CHECK(o.device() == dev && o.dtype() == q.dtype() && o.sizes() == q.sizes(), who,
                    ": out must have q's shape, dtype and device");
        TORCH_CHECK(o.stride(2) == 1, who, ": out's head dim must be contiguous");
        at::assert_no_partial_overlap(o, q);
        for (const Tensor* t : {&kc, &ks, &vc, &vs, &table, &lens}) at::assert_no_overlap(o, *t);
        if (cu_q.has_value()) at::assert_no_overlap(o, *cu_q);
    } else {
        o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    }
    if (q.numel() == 0 || B == 0) return o;
    const c10::DeviceGuard guard(dev);
    if (max_q < 0 || max_q > T) max_q = T;
    if (!cu_q.has_value()) max_q = std::min<int64_t>(max_q, 1);  // (as the library plans it)
    // (rows may be done a second time, from q: it is copied where out is q)
    const bool in_place = o.data_ptr() == q.data_ptr();
    const Tensor qr = in_place ? q.clone(at::MemoryFormat::Contiguous) : rows_of(q);
    const auto sq = strides2(qr), so = strides2(o);
    const int W = (int)table.size(1);
    const size_t bytes = kv4_attn_workspace_bytes((int)T, (int)B, (int)Hq, c.Hkv, c.D, (int)max_q,
                                                  W * c.page);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, kc.options());
    check_rc(kv4_attn(qr.data_ptr(), o.data_ptr(), sq.data(), so.data(), dt, (int)T, (int)B,
                      (int)Hq, c.Hkv, c.D, kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
                      vs.data_ptr(), c.pages, c.page, table.data_ptr<int>(),
                      B <= 1 ? W : table.stride(0), W, lens.data_ptr<int>(),
                      cu_q.has_value() ? cu_q->data_ptr<int>() : nullptr, (int)max_q, (float)scale,
                      causal, bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return o;
}
