// The C++ front end of the FP8 operators with a scale per block of 128.  Without an argument: refusals, which the argument
// checks answer before any device work (no GPU needed).  With "gpu": an MLP block's four calls through the front end and
// through the C ABI, byte for byte.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include <cuda_runtime_api.h>

#include "q3x_b200.h"
#include "q3x_b200_fp8_block.hpp"

namespace qz = q3x::quantization;

static int failures = 0;
#define EXPECT(cond)                                                  \
  do {                                                                \
    if (!(cond)) {                                                    \
      ++failures;                                                     \
      std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);     \
    }                                                                 \
  } while (0)

static void test_refusals() {
  constexpr int kInvalid = 1, kUnsupported = 801;
  auto* p = reinterpret_cast<std::uint16_t*>(0x10000000);  // never dereferenced on these paths
  auto* q = reinterpret_cast<std::uint16_t*>(0x20000000);
  auto* w = reinterpret_cast<std::uint16_t*>(0x30000000);
  auto* r = reinterpret_cast<std::uint16_t*>(0x40000000);
  auto* codes = reinterpret_cast<std::uint8_t*>(0x50000000);
  auto* scales = reinterpret_cast<float*>(0x60000000);
  const qz::Fp8BlockActivation a{codes, scales};
  EXPECT(qz::fp8_block_activation_scale_count(7, 5120) == 280 && qz::fp8_block_activation_scale_count(7, 144) == 14 &&
         qz::fp8_block_activation_scale_count(0, 144) == 0 && qz::fp8_block_activation_scale_count(7, 0) == 0);
  EXPECT(qz::launch_fp8_block_quantize_activations_cuda(p, 4, 24, a) == kInvalid);
  EXPECT(qz::launch_fp8_block_quantize_activations_cuda(p, 4, 256, {}) == kInvalid);
  EXPECT(qz::launch_fp8_block_quantize_activations_cuda(p + 1, 4, 256, a) == kUnsupported);
  EXPECT(qz::launch_fp8_block_quantize_activations_cuda(nullptr, 0, 256, {}) == 0);
  EXPECT(qz::launch_residual_add_centered_rms_norm_fp8_block_cuda(p, q, w, 4, 24, 1e-6F, r, nullptr, a) == kInvalid);
  EXPECT(qz::launch_residual_add_centered_rms_norm_fp8_block_cuda(p, q, w, 4, 256, -1.0F, r, nullptr, a) == kInvalid);
  EXPECT(qz::launch_residual_add_centered_rms_norm_fp8_block_cuda(p, q, w, 4, 32784, 1e-6F, r, nullptr, a) == kUnsupported);
  EXPECT(qz::launch_silu_mul_fp8_block_cuda(p, q, 128, 4, 256, a) == kInvalid);      // rows closer than their width
  EXPECT(qz::launch_silu_mul_fp8_block_cuda(p, q, 260, 4, 256, a) == kUnsupported);  // rows off the vectors
  EXPECT(qz::launch_silu_mul_fp8_block_cuda(nullptr, nullptr, 256, 0, 256, {}) == 0);
  const auto* wc = reinterpret_cast<const std::uint8_t*>(0x70000000);
  const auto* ws = reinterpret_cast<const float*>(0x78000000);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({wc, ws, 12, 256}, a, 4, r) == kInvalid);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({wc, ws, 16, 40}, a, 4, r) == kInvalid);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({nullptr, ws, 16, 256}, a, 4, r) == kInvalid);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({wc + 8, ws, 16, 256}, a, 4, r) == kUnsupported);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({wc, ws, 16, 256}, {}, 0, nullptr) == 0);
}

template <typename T>
struct Buffer {
  T* p = nullptr;
  std::size_t count;
  explicit Buffer(std::size_t n) : count(n) {
    EXPECT(cudaMalloc(reinterpret_cast<void**>(&p), n * sizeof(T)) == cudaSuccess);
    EXPECT(cudaMemset(p, 0, n * sizeof(T)) == cudaSuccess);
  }
  ~Buffer() { (void)cudaFree(p); }
  void fill(const std::vector<T>& v) { EXPECT(cudaMemcpy(p, v.data(), count * sizeof(T), cudaMemcpyHostToDevice) == cudaSuccess); }
  std::vector<T> get() const {
    std::vector<T> v(count);
    EXPECT(cudaMemcpy(v.data(), p, count * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess);
    return v;
  }
};

static std::uint32_t state = 12345U;
static std::uint32_t next_bits() { return state = state * 1664525U + 1013904223U; }
static std::vector<std::uint16_t> random_bf16(std::size_t n) {  // +-[0.5, 2)
  std::vector<std::uint16_t> v(n);
  for (auto& x : v) x = static_cast<std::uint16_t>(0x3f00U | (next_bits() >> 24) | ((next_bits() >> 16) & 0x8000U));
  return v;
}
static std::vector<std::uint8_t> random_codes(std::size_t n) {
  std::vector<std::uint8_t> v(n);
  for (auto& x : v) x = static_cast<std::uint8_t>((next_bits() >> 25) % 0x78U | ((next_bits() >> 24) & 0x80U));
  return v;
}
static std::vector<float> random_scales(std::size_t n) {
  std::vector<float> v(n);
  for (auto& x : v) x = 0.0001F + static_cast<float>(next_bits() >> 8) * 1e-11F;
  return v;
}

static void test_mlp_block_on_gpu() {
  constexpr std::size_t T = 37, H = 272, I = 400, HB = 3, IB = 4, MB = 7;  // blocks of H, I and 2 I
  Buffer<std::uint16_t> left(T * H), right(T * H), norm(H), residual(T * H), normalized(T * H), merged(T * 2 * I), down(T * H);
  Buffer<std::uint8_t> x(T * H), h(T * I), w1(2 * I * H), w2(H * I), y(T * H);
  Buffer<float> xs(T * HB), hs(T * IB), s1(MB * HB), s2(HB * IB), ys(T * HB);
  left.fill(random_bf16(T * H));
  right.fill(random_bf16(T * H));
  norm.fill(random_bf16(H));
  w1.fill(random_codes(2 * I * H));
  w2.fill(random_codes(H * I));
  s1.fill(random_scales(MB * HB));
  s2.fill(random_scales(HB * IB));
  EXPECT(qz::launch_residual_add_centered_rms_norm_fp8_block_cuda(left.p, right.p, norm.p, T, H, 1e-6F, residual.p, normalized.p,
                                                                  {x.p, xs.p}) == 0);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({w1.p, s1.p, 2 * I, H}, {x.p, xs.p}, T, merged.p) == 0);
  EXPECT(qz::launch_silu_mul_fp8_block_cuda(merged.p, merged.p + I, 2 * I, T, I, {h.p, hs.p}) == 0);
  EXPECT(qz::launch_fp8_block_projection_to_bf16_cuda({w2.p, s2.p, H, I}, {h.p, hs.p}, T, down.p) == 0);
  EXPECT(qz::launch_fp8_block_quantize_activations_cuda(down.p, T, H, {y.p, ys.p}) == 0);
  EXPECT(qz::fp8_block_projection_error() == 0);

  Buffer<std::uint16_t> residual2(T * H), normalized2(T * H), merged2(T * 2 * I), down2(T * H);
  Buffer<std::uint8_t> x2(T * H), h2(T * I), y2(T * H);
  Buffer<float> xs2(T * HB), hs2(T * IB), ys2(T * HB);
  EXPECT(q3x_b200_residual_add_rms_norm_fp8_block(left.p, right.p, norm.p, T, H, 1e-6F, residual2.p, normalized2.p, x2.p, xs2.p,
                                                  nullptr) == 0);
  EXPECT(q3x_b200_fp8_block_gemm_bf16(w1.p, s1.p, x2.p, xs2.p, T, 2 * I, H, merged2.p, nullptr) == 0);
  EXPECT(q3x_b200_silu_mul_fp8_block(merged2.p, merged2.p + I, 2 * I, T, I, h2.p, hs2.p, nullptr) == 0);
  EXPECT(q3x_b200_fp8_block_gemm_bf16(w2.p, s2.p, h2.p, hs2.p, T, H, I, down2.p, nullptr) == 0);
  EXPECT(q3x_b200_fp8_block_quantize(down2.p, T, H, y2.p, ys2.p, nullptr) == 0);
  EXPECT(cudaDeviceSynchronize() == cudaSuccess);
  EXPECT(residual.get() == residual2.get() && normalized.get() == normalized2.get() && x.get() == x2.get());
  EXPECT(merged.get() == merged2.get() && h.get() == h2.get() && down.get() == down2.get() && y.get() == y2.get());
  EXPECT(std::memcmp(xs.get().data(), xs2.get().data(), T * HB * 4) == 0 &&
         std::memcmp(hs.get().data(), hs2.get().data(), T * IB * 4) == 0 &&
         std::memcmp(ys.get().data(), ys2.get().data(), T * HB * 4) == 0);
  std::size_t nonzero = 0;
  for (const std::uint16_t v : down.get()) nonzero += (v & 0x7fffU) != 0 ? 1 : 0;
  EXPECT(nonzero > T * H / 2);
}

int main(int argc, char** argv) {
  if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) test_mlp_block_on_gpu();
  else test_refusals();
  if (failures == 0) std::printf("fp8 block front end tests passed\n");
  return failures == 0 ? 0 : 1;
}
