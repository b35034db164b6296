// Functions of the torch extension module (registered in module.cpp).
#pragma once

#include <torch/extension.h>

#include <vector>

torch::Tensor attn(torch::Tensor q, torch::Tensor k, torch::Tensor v, double scale,
                   c10::optional<torch::Tensor> out);

void conv3d(torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> bias,
            c10::optional<torch::Tensor> res, torch::Tensor out, std::vector<int64_t> dims,
            std::vector<int64_t> xs, std::vector<int64_t> os, std::vector<int64_t> rs);

std::vector<torch::Tensor> kv4_plan_pages_op(torch::Tensor lens, torch::Tensor new_lens,
                                             torch::Tensor table, torch::Tensor free_pages,
                                             torch::Tensor used, int64_t page, int64_t tokens);
void kv4_store_op(torch::Tensor k, torch::Tensor v, torch::Tensor slots, torch::Tensor kc,
                  torch::Tensor ks, torch::Tensor vc, torch::Tensor vs);
std::vector<torch::Tensor> kv4_load_op(torch::Tensor kc, torch::Tensor ks, torch::Tensor vc,
                                       torch::Tensor vs, torch::Tensor slots,
                                       at::ScalarType dtype);
torch::Tensor kv4_attn_op(torch::Tensor q, torch::Tensor kc, torch::Tensor ks, torch::Tensor vc,
                          torch::Tensor vs, torch::Tensor table, torch::Tensor lens, double scale,
                          c10::optional<torch::Tensor> cu_q, int64_t max_q, bool causal,
                          c10::optional<torch::Tensor> out);

torch::Tensor sparse_block_means_op(torch::Tensor x, int64_t block);
torch::Tensor sparse_select_op(torch::Tensor qm, torch::Tensor km, int64_t count, int64_t q_len,
                               int64_t k_len, int64_t block, bool causal);
torch::Tensor sparse_choose_op(torch::Tensor q, torch::Tensor km, int64_t count, int64_t k_len,
                               int64_t block, bool causal);
torch::Tensor sparse_attn_op(torch::Tensor q, torch::Tensor k, torch::Tensor v, double scale,
                             torch::Tensor index, int64_t block, bool causal,
                             c10::optional<torch::Tensor> out);
