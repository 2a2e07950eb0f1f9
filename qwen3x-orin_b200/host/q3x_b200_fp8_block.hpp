// C++17 front end of the FP8 operators with a scale per block of 128 of libq3x_b200.so.
//
// The reference project has no operand of this kind (its FP8 weights carry one scale per tensor and multiply bf16
// activations), so these functions have no declaration to mirror; they follow the conventions of the reference's launchers
// all the same (decode_ops.h:172-176): `int` is a cudaError_t, pointers are device pointers, the caller owns every buffer,
// nothing is allocated, copied or synchronised, `cuda_stream` is a cudaStream_t.
#pragma once

#include <cstddef>
#include <cstdint>

namespace q3x::quantization {

inline constexpr std::size_t kFp8BlockWidth = 128U;  // columns (activations), rows x columns (weights) of one FP32 scale

// An activation [rows, cols]: E4M3 codes, row-major, and block-major scales [ceil(cols / 128), rows].
struct Fp8BlockActivation {
  std::uint8_t* codes = nullptr;  // rows * cols bytes
  float* scales = nullptr;        // fp8_block_activation_scale_count(rows, cols) floats
};
[[nodiscard]] std::size_t fp8_block_activation_scale_count(std::size_t rows, std::size_t cols) noexcept;

// A weight [out_features, in_features]: E4M3 codes, row-major, and scales [ceil(out_features / 128), ceil(in_features / 128)].
struct Fp8BlockProjectionWeight {
  const std::uint8_t* codes = nullptr;
  const float* scales = nullptr;
  std::size_t out_features = 0U;
  std::size_t in_features = 0U;
};

// Any bf16 tensor.
[[nodiscard]] int launch_fp8_block_quantize_activations_cuda(const std::uint16_t* input, std::size_t rows, std::size_t cols,
                                                             Fp8BlockActivation activation,
                                                             void* cuda_stream = nullptr) noexcept;

// launch_residual_add_centered_rms_norm_*_5120_cuda (decode_ops.h:238-272) with the FP8 operand of the next projection;
// normalized_output may be null.
[[nodiscard]] int launch_residual_add_centered_rms_norm_fp8_block_cuda(
    const std::uint16_t* left, const std::uint16_t* right, const std::uint16_t* weight, std::size_t token_count,
    std::size_t hidden_size, float epsilon, std::uint16_t* residual_output, std::uint16_t* normalized_output,
    Fp8BlockActivation activation, void* cuda_stream = nullptr) noexcept;

// launch_silu_mul_reference_cuda (decode_ops.h:290-293) with the FP8 operand of the down projection as its only output; rows
// of gate and up are row_stride elements apart.
[[nodiscard]] int launch_silu_mul_fp8_block_cuda(const std::uint16_t* gate, const std::uint16_t* up, std::size_t row_stride,
                                                 std::size_t token_count, std::size_t intermediate_size,
                                                 Fp8BlockActivation activation, void* cuda_stream = nullptr) noexcept;

// out [token_count, out_features] bf16 = activation x weight^T, from one token on: where the reference's
// launch_projection_to_bf16_cuda (model_weights.h:794-841) multiplies bf16 activations.
[[nodiscard]] int launch_fp8_block_projection_to_bf16_cuda(const Fp8BlockProjectionWeight& weight,
                                                           Fp8BlockActivation activation, std::size_t token_count,
                                                           std::uint16_t* output, void* cuda_stream = nullptr) noexcept;

// The current device's sticky word, read after waiting for all its streams: 0 = every wait of every product on the tensor
// cores ended in time.
[[nodiscard]] int fp8_block_projection_error() noexcept;

}  // namespace q3x::quantization
