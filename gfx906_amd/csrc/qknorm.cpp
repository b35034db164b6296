// PyTorch binding of the norms of queries and keys with the position rotation
// (gfx906_amd_attn.h). The Python layer (gfx906_amd.qknorm) documents the arguments. Runs on
// the current HIP stream of the tensors' device without synchronising; what cannot be run raises
// RuntimeError.
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>

#include "bindings.h"
#include "gfx906_amd_attn.h"
#include "tensors.h"

namespace {

using namespace gfx906_amd;

const char* kWho = "norm_rotate";

bool rows_ok(const Tensor& t) {
    bool ok = (t.size(3) <= 1 || t.stride(3) == 1) &&
              reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (long long s : strides3(t)) ok = ok && s >= 0 && s % 8 == 0;
    return ok;
}

}  // namespace

std::vector<Tensor> norm_rotate_op(Tensor q, c10::optional<Tensor> k, c10::optional<Tensor> q_weight,
                                   c10::optional<Tensor> k_weight, c10::optional<Tensor> cos,
                                   c10::optional<Tensor> sin, c10::optional<Tensor> positions,
                                   double eps, bool neighbours, c10::optional<Tensor> q_out,
                                   c10::optional<Tensor> k_out) {
    const char* who = kWho;
    TORCH_CHECK(q.is_cuda() && (q.dim() == 3 || q.dim() == 4), who,
                ": q must be [T, heads, D] or [B, S, heads, D] on a GPU");
    const auto dev = q.device();
    const auto type = q.scalar_type();
    TORCH_CHECK(type == torch::kHalf || type == torch::kBFloat16, who, ": fp16 or bf16 needed");
    const bool flat = q.dim() == 3;
    const int64_t D = q.size(-1);
    // [x, result] of q and of k, 4-D
    Tensor x[2], y[2], given[2];
    const c10::optional<Tensor>* out[2] = {&q_out, &k_out};
    // Small contiguous results of both lie in one buffer (an allocation is a tenth of such a call).
    const bool both = k.has_value() && !q_out.has_value() && !k_out.has_value() &&
                      q.numel() + k->numel() <= (1 << 20) &&
                      (q.is_contiguous() || !q.is_non_overlapping_and_dense()) &&
                      (k->is_contiguous() || !k->is_non_overlapping_and_dense());
    Tensor buf;
    const int64_t nq = (q.numel() + 7) / 8 * 8;
    if (both) {
        const c10::DeviceGuard guard(dev);
        buf = at::empty({nq + k->numel()}, q.options());
    }
    for (int i = 0; i < 2; ++i) {
        if (i == 1 && !k.has_value()) {
            TORCH_CHECK(!k_out.has_value(), who, ": a result for k without k");
            break;
        }
        const Tensor& t = i ? *k : q;
        TORCH_CHECK(t.device() == dev && t.scalar_type() == type && t.dim() == q.dim() &&
                        t.size(0) == q.size(0) && (flat || t.size(1) == q.size(1)) &&
                        t.size(-1) == D,
                    who, ": q and k must agree in everything but their heads");
        if (out[i]->has_value()) {
            given[i] = **out[i];
            TORCH_CHECK(given[i].device() == dev && given[i].scalar_type() == type &&
                            given[i].sizes() == t.sizes(),
                        who, ": results must have the shape, type and device of their inputs");
        } else {
            given[i] = both ? part(buf, i ? nq : 0, t.sizes()) : at::empty_like(t);
            // (a dense input whose head dim is not the innermost one is copied; its order would not do)
            if (t.numel() && given[i].stride(-1) != 1) given[i] = at::empty(t.sizes(), t.options());
        }
        x[i] = flat ? t.unsqueeze(0) : t;
        y[i] = flat ? given[i].unsqueeze(0) : given[i];
        TORCH_CHECK(t.numel() == 0 || rows_ok(y[i]), who,
                    ": rows of the results must be contiguous, 16-byte aligned and lie a multiple "
                    "of 8 elements apart");
    }
    const bool has_k = k.has_value();
    for (int i = 0; i < (has_k ? 2 : 1); ++i) {
        if (!out[i]->has_value()) continue;
        const bool same = y[i].data_ptr() == x[i].data_ptr() && strides3(y[i]) == strides3(x[i]);
        TORCH_CHECK(same || !may_overlap(y[i], x[i]), who,
                    ": a result must be its input or must not overlap it");
        TORCH_CHECK(!has_k || (!may_overlap(y[i], x[1 - i]) && !may_overlap(y[i], y[1 - i])), who,
                    ": a result overlaps the other tensors");
    }
    const int64_t B = x[0].size(0), S = x[0].size(1);
    TORCH_CHECK(B < (1LL << 31) && S < (1LL << 31) && x[0].size(2) < 65536 &&
                    (!has_k || x[1].size(2) < 65536),
                who, ": sizes out of range");

    Tensor w[2];
    bool w32 = false;
    const c10::optional<Tensor>* ws[2] = {&q_weight, &k_weight};
    for (int i = 0; i < 2; ++i) {
        if (!ws[i]->has_value()) continue;
        TORCH_CHECK(i == 0 || has_k, who, ": a weight for k without k");
        const Tensor& t = **ws[i];
        TORCH_CHECK(t.device() == dev && t.dim() == 1 && t.size(0) == D &&
                        (t.scalar_type() == type || t.scalar_type() == torch::kFloat),
                    who, ": weights must be [D], of the rows' type or fp32, on their device");
        w[i] = t.contiguous();
        w32 = w32 || t.scalar_type() == torch::kFloat;
    }
    if (w32)  // (one of them alone in fp32: both are read so)
        for (Tensor& t : w)
            if (t.defined()) t = t.to(torch::kFloat);

    TORCH_CHECK(cos.has_value() == sin.has_value(), who, ": cos and sin go together");
    Tensor c, s, pos;
    int64_t R = 0, N = 0;
    std::array<long long, 2> ps{};
    if (cos.has_value()) {
        for (const Tensor* t : {&*cos, &*sin})
            TORCH_CHECK(t->device() == dev && t->dtype() == torch::kFloat && t->dim() == 2 &&
                            t->sizes() == cos->sizes(),
                        who, ": cos and sin must be fp32 [rows, pairs] on q's device");
        c = *cos;
        s = *sin;
        R = 2 * c.size(1);
        N = c.size(0);
        TORCH_CHECK(N < (1LL << 31) && R <= D, who, ": cos and sin too large");
        auto in_place = [&](const Tensor& t) {
            return (t.size(1) <= 1 || t.stride(1) == 1) && t.stride(0) >= 0 && t.stride(0) % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
        };
        if (!in_place(c) || !in_place(s) || c.stride(0) != s.stride(0)) {
            c = c.clone(at::MemoryFormat::Contiguous);
            s = s.clone(at::MemoryFormat::Contiguous);
        }
        if (positions.has_value()) {
            pos = flat ? positions->unsqueeze(0) : *positions;
            TORCH_CHECK(pos.device() == dev && pos.dtype() == torch::kInt && pos.dim() == 2 &&
                            pos.size(0) == B && pos.size(1) == S,
                        who, ": positions must be int32, one a token, on q's device");
            ps = strides2(pos);
        } else {
            TORCH_CHECK(N >= S, who, ": fewer rows of cos and sin than tokens");
        }
    } else {
        TORCH_CHECK(!positions.has_value(), who, ": positions without cos and sin");
    }
    for (int i = 0; i < (has_k ? 2 : 1); ++i)
        if (out[i]->has_value())
            for (const Tensor* t : {&w[0], &w[1], &c, &s, &pos})
                if (t->defined()) at::assert_no_overlap(given[i], *t);
    const c10::DeviceGuard guard(dev);
    std::vector<Tensor> result{given[0]};
    if (has_k) result.push_back(given[1]);
    std::array<long long, 3> xs[2]{}, ys[2]{};
    for (int i = 0; i < (has_k ? 2 : 1); ++i) {
        if (!rows_ok(x[i])) x[i] = x[i].clone(at::MemoryFormat::Contiguous);
        xs[i] = strides3(x[i]);
        ys[i] = strides3(y[i]);
    }
    auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const int Hq = (int)x[0].size(2), Hk = has_k ? (int)x[1].size(2) : 0;
    const int rc = qk_norm_rotate(
        ptr(x[0]), ptr(x[1]), ptr(y[0]), ptr(y[1]), xs[0].data(), xs[1].data(), ys[0].data(),
        ys[1].data(), type == torch::kBFloat16 ? KV8_DTYPE_BF16 : KV8_DTYPE_F16, (int)B, (int)S, Hq,
        Hk, (int)std::min<int64_t>(D, 1 << 30), ptr(w[0]), ptr(w[1]), w32, (float)eps,
        R ? c.data_ptr<float>() : nullptr, R ? s.data_ptr<float>() : nullptr,
        R && N > 1 ? c.stride(0) : 0, (int)N, (int)R, neighbours,
        pos.defined() ? pos.data_ptr<int>() : nullptr, ps.data(), stream());
    TORCH_CHECK(rc == 0, "kernel: ",
                qk_norm_rotate_last_error() ? qk_norm_rotate_last_error() : "launch failed");
    return result;
}
