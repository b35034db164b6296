// The torch extension module: attn (attention forward) and conv3d (implicit-GEMM
// conv3d), the ops of the reference's two extensions (attn.cpp:21 and
// hip_conv/conv3d.cpp:53) in one module, and the ops behind gfx906_amd.kv4, kv8, qknorm and
// sparse, which have no counterpart there.
#include "bindings.h"

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("attn", &attn, "fp16/bf16 attention forward on gfx950 (q, k, v, scale, out=None)",
          pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("scale"),
          pybind11::arg("out") = pybind11::none());
    m.def("conv3d", &conv3d,
          "fp16 NDHWC implicit-GEMM conv3d on gfx950 "
          "(x, w, bias, res, out, dims, xs, os, rs)");
    m.def("kv4_plan_pages", &kv4_plan_pages_op, "pages and slots of a paged cache");
    m.def("kv4_store", &kv4_store_op, "rows of k and v into the 4-bit cache");
    m.def("kv4_load", &kv4_load_op, "rows of the 4-bit cache");
    m.def("kv4_attn", &kv4_attn_op, "attention over the 4-bit cache");
    m.def("sparse_block_means", &sparse_block_means_op, "means of row blocks");
    m.def("sparse_select", &sparse_select_op, "key blocks of every query block");
    m.def("sparse_choose", &sparse_choose_op, "key blocks of every query block, from its rows");
    m.def("sparse_attn", &sparse_attn_op, "attention over selected key blocks");
    m.def("norm_rotate", &norm_rotate_op, "norms of queries and keys with the position rotation");
    m.def("kv8_store", &kv8_store_op, "rows of k and v into the 8-bit cache");
    m.def("kv8_load", &kv8_load_op, "rows of the 8-bit cache");
    m.def("kv8_attn", &kv8_attn_op, "attention over the 8-bit cache");
    m.def("kv8_weigh", &kv8_weigh_op, "attention weights of the 8-bit cache's blocks");
    m.def("kv8_evict", &kv8_evict_op, "eviction of pages by their attention weights");
}
