// PyTorch binding of sparse attention (gfx906_amd_attn.h): sparse_block_means,
// sparse_select, sparse_choose and sparse_attn. The Python layer (gfx906_amd.sparse) documents the
// arguments. Every op runs on the current HIP stream of its tensors' device without
// synchronising; what cannot be run raises RuntimeError.
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "bindings.h"
#include "gfx906_amd_attn.h"

namespace {

using torch::Tensor;

int dtype_of(const Tensor& t, const char* who) {
    TORCH_CHECK(t.is_cuda() && (t.dtype() == torch::kHalf || t.dtype() == torch::kBFloat16), who,
                ": CUDA fp16 or bf16 tensors needed");
    TORCH_CHECK(t.dim() == 4, who, ": tensors must be 4-D [B, H, S, D]");
    for (int d = 0; d < 4; ++d)
        TORCH_CHECK(t.size(d) < (1LL << 30), who, ": tensor too large");
    return t.dtype() == torch::kBFloat16 ? SPARSE_DTYPE_BF16 : SPARSE_DTYPE_F16;
}

std::array<long long, 3> strides3(const Tensor& t) {
    std::array<long long, 3> s;
    for (int d = 0; d < 3; ++d) s[d] = t.size(d) == 1 ? 0 : t.stride(d);
    return s;
}

// Read in place where the head dim is contiguous, the other strides are multiples of
// 8, rows lie apart and the data is 16-byte aligned; copied otherwise.
Tensor rows_of(const Tensor& t) {
    bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    const auto s = strides3(t);
    for (int d = 0; d < 3; ++d) ok = ok && s[d] >= 0 && s[d] % 8 == 0;
    ok = ok && s[2] <= (1 << 22) && (t.size(2) == 1 || s[2] >= t.size(3));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
void check_rc(int rc) {
    TORCH_CHECK(rc == 0, "kernel: ", sparse_last_error() ? sparse_last_error() : "launch failed");
}

int64_t blocks(int64_t s, int64_t block) { return (s + block - 1) / block; }

void check_block(int64_t block, const char* who) {
    TORCH_CHECK(block == 64 || block == 128, who, ": blocks have 64 or 128 rows");
}

void check_count(int64_t count, const char* who) {
    TORCH_CHECK(count >= 1 && count <= SPARSE_MAX_COUNT, who, ": count must be 1 .. ",
                SPARSE_MAX_COUNT);
}

}  // namespace

Tensor sparse_block_means_op(Tensor x, int64_t block) {
    const char* who = "block_means";
    const int dt = dtype_of(x, who);
    check_block(block, who);
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), H = x.size(1), S = x.size(2), D = x.size(3);
    Tensor m = at::empty({B, H, blocks(S, block), D}, x.options().dtype(torch::kFloat));
    if (m.numel() == 0) return m;
    const Tensor r = rows_of(x);
    const auto st = strides3(r);
    check_rc(sparse_block_means(r.data_ptr(), st.data(), dt, (int)B, (int)H, (int)S, (int)D,
                                (int)block, m.data_ptr<float>(), stream()));
    return m;
}

Tensor sparse_select_op(Tensor qm, Tensor km, int64_t count, int64_t q_len, int64_t k_len,
                        int64_t block, bool causal) {
    const char* who = "select";
    check_block(block, who);
    check_count(count, who);
    TORCH_CHECK(q_len >= 0 && k_len >= 0 && q_len < (1 << 30) && k_len < (1 << 30), who,
                ": bad lengths");
    for (const Tensor* t : {&qm, &km})
        TORCH_CHECK(t->is_cuda() && t->dtype() == torch::kFloat && t->dim() == 4 &&
                        t->device() == qm.device(),
                    who, ": means must be 4-D fp32 CUDA tensors on one device");
    TORCH_CHECK(qm.size(0) == km.size(0) && qm.size(3) == km.size(3) &&
                    qm.size(2) == blocks(q_len, SPARSE_Q_BLOCK) &&
                    km.size(2) == blocks(k_len, block),
                who, ": means do not match each other or the lengths");
    for (int d = 0; d < 4; ++d)
        TORCH_CHECK(qm.size(d) < (1LL << 30) && km.size(d) < (1LL << 30), who, ": tensor too large");
    const c10::DeviceGuard guard(qm.device());
    const int B = (int)qm.size(0), Hq = (int)qm.size(1), Hkv = (int)km.size(1),
              D = (int)qm.size(3);
    Tensor index = at::empty({B, Hq, qm.size(2), count}, qm.options().dtype(torch::kInt));
    if (index.numel() == 0) return index;
    const Tensor qc = qm.contiguous(), kc = km.contiguous();
    const size_t bytes =
        sparse_select_workspace_bytes(B, Hq, (int)q_len, (int)k_len, (int)block);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, qm.options().dtype(torch::kByte));
    check_rc(sparse_select(qc.data_ptr<float>(), kc.data_ptr<float>(), B, Hq, Hkv, (int)q_len,
                           (int)k_len, D, (int)block, (int)count, causal, index.data_ptr<int>(),
                           bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return index;
}

Tensor sparse_choose_op(Tensor q, Tensor km, int64_t count, int64_t k_len, int64_t block,
                        bool causal) {
    const char* who = "choose";
    const int dt = dtype_of(q, who);
    check_block(block, who);
    check_count(count, who);
    TORCH_CHECK(km.device() == q.device() && km.dtype() == torch::kFloat && km.dim() == 4 &&
                    k_len >= 0 && k_len < (1 << 30) && km.size(0) == q.size(0) &&
                    km.size(3) == q.size(3) && km.size(2) == blocks(k_len, block) &&
                    km.size(1) < (1LL << 30),
                who, ": means must be fp32 [B, heads, ceil(k_len/block), D] on q's device");
    const c10::DeviceGuard guard(q.device());
    const int B = (int)q.size(0), Hq = (int)q.size(1), Sq = (int)q.size(2), D = (int)q.size(3);
    Tensor index =
        at::empty({B, Hq, blocks(Sq, SPARSE_Q_BLOCK), count}, q.options().dtype(torch::kInt));
    if (index.numel() == 0) return index;
    const Tensor qr = rows_of(q), kc = km.contiguous();
    const auto st = strides3(qr);
    const size_t bytes =
        sparse_choose_workspace_bytes(B, Hq, Sq, (int)k_len, D, (int)block);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(torch::kByte));
    check_rc(sparse_choose(qr.data_ptr(), st.data(), dt, kc.data_ptr<float>(), B, Hq,
                           (int)km.size(1), Sq, (int)k_len, D, (int)block, (int)count, causal,
                           index.data_ptr<int>(), bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return index;
}

Tensor sparse_attn_op(Tensor q, Tensor k, Tensor v, double scale, Tensor index, int64_t block,
                      bool causal, c10::optional<Tensor> out) {
    const char* who = "attn_blocks";
    const int dt = dtype_of(q, who);
    check_block(block, who);
    dtype_of(k, who);
    dtype_of(v, who);
    TORCH_CHECK(k.device() == q.device() && v.device() == q.device() && k.dtype() == q.dtype() &&
                    v.dtype() == q.dtype(),
                who, ": q, k and v must have one dtype and device");
    const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3), Hkv = k.size(1),
                  Skv = k.size(2);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D && Hkv > 0 &&
                    Hq % Hkv == 0,
                who, ": q/k/v shape mismatch");
    TORCH_CHECK(index.device() == q.device() && index.dtype() == torch::kInt && index.dim() == 4 &&
                    index.size(0) == B && index.size(1) == Hq &&
                    index.size(2) == blocks(Sq, SPARSE_Q_BLOCK),
                who, ": index must be int32 [B, heads, ceil(Sq/128), count] on q's device");
    check_count(index.size(3), who);
    Tensor o;
    if (out.has_value()) {
        o = *out;
        TORCH_CHECK(o.device() == q.device() && o.dtype() == q.dtype() && o.sizes() == q.sizes(),
                    who, ": out must have q's shape, dtype and device");
        TORCH_CHECK(o.stride(3) == 1, who, ": out's head dim must be contiguous");
        at::assert_no_partial_overlap(o, q);
        at::assert_no_overlap(o, k);
        at::assert_no_overlap(o, v);
        at::assert_no_overlap(o, index);
    } else {
        o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    }
    if (q.numel() == 0) return o;
    const c10::DeviceGuard guard(q.device());
    const Tensor qr = rows_of(q), kr = rows_of(k), vr = rows_of(v), ix = index.contiguous();
    const auto sq = strides3(qr), sk = strides3(kr), sv = strides3(vr), so = strides3(o);
    const int count = (int)index.size(3);
    const size_t bytes = sparse_attn_workspace_bytes((int)B, (int)Hq, (int)Sq, (int)Skv, (int)D,
                                                     (int)block, count);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(torch::kByte));
    check_rc(sparse_attn(qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), o.data_ptr(), sq.data(),
                         sk.data(), sv.data(), so.data(), dt, (int)B, (int)Hq, (int)Hkv, (int)Sq,
                         (int)Skv, (int)D, (float)scale, ix.data_ptr<int>(), (int)block, count,
                         causal, bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return o;
}
