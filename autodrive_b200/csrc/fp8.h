// The 8-bit quantisers and product as C++ functions (fp8_quant.cu,
// fp8_gemm.cu), for the linear layer that joins them (fp8_linear.cpp). Operands are checked by
// their callers' entry points.
#pragma once

#include <torch/extension.h>

#include <utility>
#include <vector>

namespace fp8 {

// A matrix [rows, K] with contiguous columns -> {q, scale}.
std::pair<torch::Tensor, torch::Tensor> quantize_rows(const torch::Tensor& x);
// A matrix with contiguous columns -> {q, scale}, or with `transposed` {q, scale, q^T, scale^T}.
std::vector<torch::Tensor> quantize_blocks(const torch::Tensor& w, bool transposed);
// Sums of a matrix's columns, in fp32, as `out_type`.
torch::Tensor column_sums(const torch::Tensor& x, torch::ScalarType out_type);
// a b^T (+ bias, fp32 or undefined) of operands whose rows start 16 bytes apart.
torch::Tensor matmul(const torch::Tensor& a, const torch::Tensor& a_scale, const torch::Tensor& b,
                     const torch::Tensor& b_scale, const torch::Tensor& bias, torch::ScalarType out_dtype,
                     const torch::Tensor& status, int64_t wait_ns);
// a^T b of matrices [K, M] and [K, N], both bf16 or both fp16, with 16-byte aligned rows, fp32 sums.
torch::Tensor weight_gradient(const torch::Tensor& a, const torch::Tensor& b, torch::ScalarType out_type,
                              const torch::Tensor& status);
// `t` as a matrix with contiguous columns: a view where its layout allows one.
torch::Tensor as_matrix(const torch::Tensor& t);
// 1: fp32, bf16 or fp16.
bool known_type(torch::ScalarType t);

constexpr int64_t kWaitNs = 2000000000ll;

}  // namespace fp8
