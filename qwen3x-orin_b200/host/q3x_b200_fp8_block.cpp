// Thin forwards from the C++ front end of the FP8 operators with a scale per block of 128 to the C ABI.
#include "q3x_b200_fp8_block.hpp"

#include "q3x_b200.h"

namespace q3x::quantization {

static_assert(kFp8BlockWidth == Q3X_B200_FP8_BLOCK);

std::size_t fp8_block_activation_scale_count(std::size_t rows, std::size_t cols) noexcept {
  return (cols / kFp8BlockWidth + (cols % kFp8BlockWidth != 0U ? 1U : 0U)) * rows;
}

int launch_fp8_block_quantize_activations_cuda(const std::uint16_t* input, std::size_t rows, std::size_t cols,
                                               Fp8BlockActivation activation, void* cuda_stream) noexcept {
  return q3x_b200_fp8_block_quantize(input, rows, cols, activation.codes, activation.scales, cuda_stream);
}

int launch_residual_add_centered_rms_norm_fp8_block_cuda(const std::uint16_t* left, const std::uint16_t* right,
                                                         const std::uint16_t* weight, std::size_t token_count,
                                                         std::size_t hidden_size, float epsilon,
                                                         std::uint16_t* residual_output, std::uint16_t* normalized_output,
                                                         Fp8BlockActivation activation, void* cuda_stream) noexcept {
  return q3x_b200_residual_add_rms_norm_fp8_block(left, right, weight, token_count, hidden_size, epsilon, residual_output,
                                                  normalized_output, activation.codes, activation.scales, cuda_stream);
}

int launch_silu_mul_fp8_block_cuda(const std::uint16_t* gate, const std::uint16_t* up, std::size_t row_stride,
                                   std::size_t token_count, std::size_t intermediate_size, Fp8BlockActivation activation,
                                   void* cuda_stream) noexcept {
  return q3x_b200_silu_mul_fp8_block(gate, up, row_stride, token_count, intermediate_size, activation.codes,
                                     activation.scales, cuda_stream);
}

int launch_fp8_block_projection_to_bf16_cuda(const Fp8BlockProjectionWeight& weight, Fp8BlockActivation activation,
                                             std::size_t token_count, std::uint16_t* output, void* cuda_stream) noexcept {
  return q3x_b200_fp8_block_gemm_bf16(weight.codes, weight.scales, activation.codes, activation.scales, token_count,
                                      weight.out_features, weight.in_features, output, cuda_stream);
}

int fp8_block_projection_error() noexcept { return q3x_b200_fp8_block_gemm_error(); }

}  // namespace q3x::quantization
