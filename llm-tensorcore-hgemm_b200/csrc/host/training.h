// Torch-facing host layer of the training operators (llm_hgemm.training): the
// argument checks, autograd functions and launches through the C ABI in
// hgemm_sm100_train.h. No reference counterpart (the reference is
// inference-only).
#pragma once

#include <cstdint>
#include <string>

#include <torch/extension.h>

// y = (silu(x gate^T) * (x up^T)) down^T over the last dimension of x;
// differentiable in all four tensors.
torch::Tensor gated_ffn(const torch::Tensor& x, const torch::Tensor& gate, const torch::Tensor& up,
                        const torch::Tensor& down);

// Cross entropy of the logits x weight^T, FP32; differentiable in x and weight.
torch::Tensor linear_cross_entropy(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& target,
                                   const std::string& reduction, int64_t ignore_index);

// The last two dimensions of g orthogonalised by Newton-Schulz steps.
torch::Tensor orthogonalize(const torch::Tensor& g, int64_t steps, double a, double b, double c, double eps);

// Status of the kernels launched by the functions above so far, as far as they
// have run (0, or HGEMM_SM100_ERR_PIPELINE_TIMEOUT); with `clear` it is reset.
// Does not wait for the device. The next of those calls raises it too.
int32_t training_status(bool clear);
// Address of that word, writable by the host and all devices.
int64_t training_status_address();
