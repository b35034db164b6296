// Checks of tensors that the bindings of the caches and of the head norms share.
#pragma once

#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <array>

namespace gfx906_amd {

using torch::Tensor;

inline void check_ints(const Tensor& t, int64_t n, const c10::Device& dev, const char* who,
                const char* name) {
    TORCH_CHECK(t.device() == dev && t.dtype() == torch::kInt && t.dim() == 1 &&
                    (n < 0 || t.size(0) == n) && t.is_contiguous(),
                who, ": ", name, " must be a contiguous int32 vector of the right length on the "
                "other tensors' device");
}

// Table of pages, a row a request, and its row stride.
inline void check_table(const Tensor& table, int64_t B, int page, const c10::Device& dev,
                        const char* who) {
    TORCH_CHECK(table.device() == dev && table.dtype() == torch::kInt && table.dim() == 2 &&
                    table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1) &&
                    (B <= 1 || table.stride(0) >= 0) && table.size(1) * page < (1LL << 31),
                who, ": table must be int32 [B, W] with contiguous rows of fewer than 2^31 tokens");
}
inline int64_t table_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// [T, H, D] rows the kernels read in place: contiguous head dim, the other strides
// multiples of 8, 16-byte aligned. Anything else is copied.
inline Tensor rows_of(const Tensor& t) {
    const bool ok = (t.stride(2) == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(0) == 1 || (t.stride(0) >= 0 && t.stride(0) % 8 == 0)) &&
                    (t.size(1) == 1 || (t.stride(1) >= 0 && t.stride(1) % 8 == 0));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
inline std::array<long long, 2> strides2(const Tensor& t) {
    return {t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1)};
}

// {batch, token, head} of a [B, S, H, D] tensor.
inline std::array<long long, 3> strides3(const Tensor& t) {
    std::array<long long, 3> s;
    for (int d = 0; d < 3; ++d) s[d] = t.size(d) <= 1 ? 0 : t.stride(d);
    return s;
}

// Whether elements of a and b, both [B, S, H, D] of one type, may share memory: they do not where their
// ranges lie apart, nor where they do so modulo a period. Dims whose strides are multiples of the period
// do not count for that, the others span a range: q, k and v are different parts of every
// batch's, token's or head's elements of one buffer, in whatever order.
inline bool may_overlap(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    auto at = [](const Tensor& t) {
        return (long long)(reinterpret_cast<intptr_t>(t.data_ptr()) / t.element_size());
    };
    auto extent = [](const Tensor& t, long long period) {  // elements that t spans (0: of all dims)
        long long n = 1;
        for (int d = 0; d < 4; ++d)
            if (!period || t.stride(d) % period) n += (t.size(d) - 1) * t.stride(d);
        return n;
    };
    const long long p = at(a), q = at(b);
    if (p + extent(a, 0) <= q || q + extent(b, 0) <= p) return false;
    for (const Tensor* t : {&a, &b})
        for (int d = 0; d < 3; ++d) {
            const long long period = t->stride(d);
            if (period <= 0 || t->size(d) <= 1) continue;
            const long long from = ((q - p) % period + period) % period;
            if (from >= extent(a, period) && from + extent(b, period) <= period) return false;
        }
    return true;
}

// A contiguous part of a one-dimensional buffer, made by hand: a view through the dispatcher takes
// 0.7 us, as much as a tenth of a small call.
inline Tensor part(const Tensor& buf, int64_t offset, at::IntArrayRef sizes) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(),
                                                        buf.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

inline hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

}  // namespace gfx906_amd
