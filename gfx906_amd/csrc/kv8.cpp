// PyTorch binding of the 8-bit key/value cache, its attention weights and eviction
// (gfx906_amd_attn.h). The Python layer (gfx906_amd.kv8) documents the arguments. Every op runs
// on the current HIP stream of its tensors' device without synchronising; what cannot be run raises
// RuntimeError.
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>

#include "bindings.h"
#include "gfx906_amd_attn.h"
#include "tensors.h"

namespace {

using namespace gfx906_amd;

int dtype_of(at::ScalarType t, const char* who) {
    TORCH_CHECK(t == torch::kHalf || t == torch::kBFloat16, who, ": fp16 or bf16 needed");
    return t == torch::kBFloat16 ? KV8_DTYPE_BF16 : KV8_DTYPE_F16;
}

// The four tensors of a cache, checked against each other.
struct Parts {
    int pages, Hkv, page, D;
    Parts(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs, const char* who) {
        TORCH_CHECK(k.is_cuda() && k.dim() == 4 && v.dim() == 5 && ks.dim() == 3, who,
                    ": the cache must be [pages, heads, page, D] and [pages, heads, page/64, D, 64] "
                    "codes and [pages, heads, page/64] scales on a GPU");
        for (const Tensor* t : {&k, &ks, &v, &vs})
            TORCH_CHECK(t->device() == k.device() && t->is_contiguous() &&
                            t->dtype() == (t == &k || t == &v ? torch::kByte : torch::kFloat),
                        who, ": codes must be uint8, scales fp32, contiguous and on one device");
        TORCH_CHECK(k.size(0) < (1LL << 31) && k.size(1) > 0 && k.size(1) < 65536 &&
                        k.size(2) > 0 && k.size(2) <= 256 && k.size(3) <= 256,
                    who, ": cache too large, or without heads or tokens");
        pages = (int)k.size(0);
        Hkv = (int)k.size(1);
        page = (int)k.size(2);
        D = (int)k.size(3);
        TORCH_CHECK(page % KV8_BLOCK == 0 &&
                        v.sizes() == at::IntArrayRef({pages, Hkv, page / KV8_BLOCK, D, KV8_BLOCK}) &&
                        ks.sizes() == at::IntArrayRef({pages, Hkv, page / KV8_BLOCK}) &&
                        vs.sizes() == ks.sizes(),
                    who, ": the parts of the cache do not match");
    }
};

void check_weights(const Tensor& w, const Parts& c, const c10::Device& dev, const char* who) {
    TORCH_CHECK(w.device() == dev && w.dtype() == torch::kFloat && w.is_contiguous() &&
                    w.sizes() == at::IntArrayRef({c.pages, c.Hkv, c.page / KV8_BLOCK}),
                who, ": weights must be contiguous fp32 [pages, heads, page/64] on the cache's device");
}

// Queries over a cache, as attn and weigh take them.
struct Queries {
    int dt;
    int64_t T, Hq, B;
    Queries(const Tensor& q, const Parts& c, const Tensor& table, const Tensor& lens,
            const c10::optional<Tensor>& cu_q, int64_t& max_q, const c10::Device& dev,
            const char* who) {
        TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.size(2) == c.D, who,
                    ": q must be [T, heads, D] on the cache's device, with its head dim");
        dt = dtype_of(q.scalar_type(), who);
        check_ints(lens, -1, dev, who, "lens");
        T = q.size(0);
        Hq = q.size(1);
        B = lens.size(0);
        TORCH_CHECK(T < (1LL << 31) && Hq < 65536 && B <= KV8_MAX_REQUESTS, who,
                    ": sizes out of range");
        TORCH_CHECK(Hq > 0 && Hq % c.Hkv == 0, who,
                    ": query heads must be a multiple of kv heads");
        if (cu_q.has_value())
            check_ints(*cu_q, B + 1, dev, who, "cu_q");
        else
            TORCH_CHECK(T == B, who, ": without cu_q, one query a request");
        check_table(table, B, c.page, dev, who);
        if (max_q < 0 || max_q > T) max_q = T;
        if (!cu_q.has_value()) max_q = std::min<int64_t>(max_q, 1);
    }
};

const int* ints(const c10::optional<Tensor>& t) {
    return t.has_value() ? t->data_ptr<int>() : nullptr;
}
void check_rc(int rc) {
    TORCH_CHECK(rc == 0, "kernel: ", kv8_last_error() ? kv8_last_error() : "launch failed");
}

}  // namespace

void kv8_store_op(Tensor k, Tensor v, Tensor kc, Tensor ks, Tensor vc, Tensor vs, Tensor table,
                  Tensor lens, c10::optional<Tensor> cu_new, c10::optional<Tensor> weights) {
    const char* who = "store";
    const Parts c(kc, ks, vc, vs, who);
    const auto dev = kc.device();
    TORCH_CHECK(k.dim() == 3 && k.size(1) == c.Hkv && k.size(2) == c.D && v.sizes() == k.sizes(),
                who, ": k and v must be [T, heads, D] of the cache's heads and head dim");
    TORCH_CHECK(k.device() == dev && v.device() == dev && v.dtype() == k.dtype(), who,
                ": k and v must have one dtype and the cache's device");
    TORCH_CHECK(k.size(0) < (1LL << 31), who, ": too many rows");
    const int dt = dtype_of(k.scalar_type(), who);
    check_ints(lens, -1, dev, who, "lens");
    const int64_t T = k.size(0), B = lens.size(0);
    TORCH_CHECK(B <= KV8_MAX_REQUESTS, who, ": too many requests");
    if (cu_new.has_value())
        check_ints(*cu_new, B + 1, dev, who, "cu_new");
    else
        TORCH_CHECK(T == B, who, ": without cu_new, one row a request");
    check_table(table, B, c.page, dev, who);
    if (weights.has_value()) check_weights(*weights, c, dev, who);
    const c10::DeviceGuard guard(dev);
    if (k.numel() == 0 || B == 0) return;
    const Tensor kr = rows_of(k), vr = rows_of(v);
    const auto sk = strides2(kr), sv = strides2(vr);
    check_rc(kv8_store(kr.data_ptr(), vr.data_ptr(), sk.data(), sv.data(), dt, (int)T, (int)B, c.Hkv,
                       c.D, kc.data_ptr(), ks.data_ptr<float>(), vc.data_ptr(),
                       vs.data_ptr<float>(), c.pages, c.page, table.data_ptr<int>(),
                       table_stride(table), (int)table.size(1), lens.data_ptr<int>(), ints(cu_new),
                       weights.has_value() ? weights->data_ptr<float>() : nullptr, stream()));
}

std::vector<Tensor> kv8_load_op(Tensor kc, Tensor ks, Tensor vc, Tensor vs, Tensor slots,
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
        check_rc(kv8_load(k.data_ptr(), v.data_ptr(), dt, (int)T, c.Hkv, c.D,
                          slots.data_ptr<int>(), kc.data_ptr(), ks.data_ptr<float>(), vc.data_ptr(),
                          vs.data_ptr<float>(), c.pages, c.page, stream()));
    return {k, v};
}

std::vector<Tensor> kv8_attn_op(Tensor q, Tensor kc, Tensor ks, Tensor vc, Tensor vs, Tensor table,
                                Tensor lens, double scale, c10::optional<Tensor> cu_q,
                                int64_t max_q, bool causal, c10::optional<Tensor> out, bool lse) {
    const char* who = "attn";
    const Parts c(kc, ks, vc, vs, who);
    const auto dev = kc.device();
    const Queries n(q, c, table, lens, cu_q, max_q, dev, who);
    Tensor o;
    bool in_place = false;
    if (out.has_value()) {
        o = *out;
        TORCH_CHECK(o.device() == dev && o.dtype() == q.dtype() && o.sizes() == q.sizes(), who,
                    ": out must have q's shape, dtype and device");
        TORCH_CHECK(o.stride(2) == 1, who, ": out's head dim must be contiguous");
        in_place = o.data_ptr() == q.data_ptr() && strides2(o) == strides2(q);
        TORCH_CHECK(in_place || !may_overlap(o.unsqueeze(0), q.unsqueeze(0)), who,
                    ": out overlaps a part of q");
        for (const Tensor* t : {&kc, &ks, &vc, &vs, &table, &lens}) at::assert_no_overlap(o, *t);
        if (cu_q.has_value()) at::assert_no_overlap(o, *cu_q);
    } else {
        o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    }
    std::vector<Tensor> result{o};
    if (lse) result.push_back(at::empty({n.T, n.Hq}, q.options().dtype(torch::kFloat)));
    if (q.numel() == 0 || n.B == 0) return result;
    const c10::DeviceGuard guard(dev);
    // (a workgroup may read rows of q after another has written theirs: q is copied where out is q)
    const Tensor qr = in_place ? q.clone(at::MemoryFormat::Contiguous) : rows_of(q);
    const auto sq = strides2(qr), so = strides2(o);
    const int W = (int)table.size(1);
    const size_t bytes = kv8_attn_workspace_bytes((int)n.T, (int)n.B, (int)n.Hq, c.Hkv, c.D,
                                                  (int)max_q, W * c.page);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, kc.options());
    check_rc(kv8_attn(qr.data_ptr(), o.data_ptr(), lse ? result[1].data_ptr<float>() : nullptr,
                      sq.data(), so.data(), n.dt, (int)n.T, (int)n.B, (int)n.Hq, c.Hkv, c.D,
                      kc.data_ptr(), ks.data_ptr<float>(), vc.data_ptr(), vs.data_ptr<float>(),
                      c.pages, c.page, table.data_ptr<int>(), table_stride(table), W,
                      lens.data_ptr<int>(), ints(cu_q), (int)max_q, (float)scale, causal,
                      bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return result;
}

void kv8_weigh_op(Tensor weights, Tensor q, Tensor lse, Tensor kc, Tensor ks, Tensor vc, Tensor vs,
                  Tensor table, Tensor lens, double scale, c10::optional<Tensor> cu_q,
                  int64_t max_q, bool causal) {
    const char* who = "weigh";
    const Parts c(kc, ks, vc, vs, who);
    const auto dev = kc.device();
    const Queries n(q, c, table, lens, cu_q, max_q, dev, who);
    check_weights(weights, c, dev, who);
    TORCH_CHECK(lse.device() == dev && lse.dtype() == torch::kFloat && lse.is_contiguous() &&
                    lse.dim() == 2 && lse.size(0) == n.T && lse.size(1) == n.Hq,
                who, ": lse must be contiguous fp32 [T, heads] on the cache's device");
    at::assert_no_overlap(weights, lse);
    const c10::DeviceGuard guard(dev);
    if (q.numel() == 0 || n.B == 0) return;
    const Tensor qr = rows_of(q);
    const auto sq = strides2(qr);
    const size_t bytes = kv8_weigh_workspace_bytes((int)n.T, (int)n.B, (int)n.Hq, c.Hkv, (int)max_q,
                                                   (int)table.size(1), c.page);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, kc.options());
    check_rc(kv8_weigh(weights.data_ptr<float>(), qr.data_ptr(), sq.data(), n.dt,
                       lse.data_ptr<float>(), (int)n.T, (int)n.B, (int)n.Hq, c.Hkv, c.D,
                       kc.data_ptr(), ks.data_ptr<float>(), c.pages, c.page, table.data_ptr<int>(),
                       table_stride(table), (int)table.size(1), lens.data_ptr<int>(), ints(cu_q),
                       (int)max_q, (float)scale, causal, bytes ? ws.data_ptr() : nullptr, bytes,
                       stream()));
}

std::vector<Tensor> kv8_evict_op(Tensor weights, Tensor table, Tensor lens, Tensor keep,
                                 Tensor free_pages, Tensor used, int64_t first, int64_t recent) {
    const char* who = "evict";
    TORCH_CHECK(weights.is_cuda() && weights.dim() == 3 && weights.dtype() == torch::kFloat &&
                    weights.is_contiguous() && weights.size(0) < (1LL << 31) &&
                    weights.size(1) > 0 && weights.size(1) < 65536 && weights.size(2) > 0 &&
                    weights.size(2) <= 4,
                who, ": weights must be contiguous fp32 [pages, heads, page/64] on a GPU");
    const auto dev = weights.device();
    const int page = (int)weights.size(2) * KV8_BLOCK;
    check_ints(lens, -1, dev, who, "lens");
    const int64_t B = lens.size(0);
    TORCH_CHECK(B <= KV8_MAX_REQUESTS, who, ": too many requests");
    check_ints(keep, B, dev, who, "keep");
    check_ints(free_pages, -1, dev, who, "free_pages");
    check_ints(used, 1, dev, who, "used");
    TORCH_CHECK(free_pages.size(0) < (1LL << 31), who, ": free_pages too long");
    check_table(table, B, page, dev, who);
    TORCH_CHECK(first >= 0 && recent >= 1, who, ": first must be at least 0 and recent at least 1");
    for (const Tensor* t : {&lens, &keep, &free_pages, &used, &weights})
        at::assert_no_overlap(table, *t);
    for (const Tensor* t : {&lens, &keep, &used, &weights}) at::assert_no_overlap(free_pages, *t);
    const c10::DeviceGuard guard(dev);
    const int W = (int)table.size(1);
    const Tensor buf = at::empty({B + 2}, lens.options());
    const Tensor out = part(buf, 0, {B}), u = part(buf, B, {1}), lost = part(buf, B + 1, {1});
    const size_t bytes = kv8_evict_workspace_bytes((int)B, W);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, lens.options().dtype(torch::kByte));
    check_rc(kv8_evict(weights.data_ptr<float>(), (int)weights.size(0), (int)weights.size(1), page,
                       table.data_ptr<int>(), table_stride(table), W, lens.data_ptr<int>(),
                       keep.data_ptr<int>(), (int)B, (int)std::min<int64_t>(first, 0x7fffffff),
                       (int)std::min<int64_t>(recent, 0x7fffffff), free_pages.data_ptr<int>(),
                       (int)free_pages.size(0), used.data_ptr<int>(), out.data_ptr<int>(),
                       u.data_ptr<int>(), lost.data_ptr<int>(), bytes ? ws.data_ptr() : nullptr,
                       bytes, stream()));
    return {out, u, lost};
}
