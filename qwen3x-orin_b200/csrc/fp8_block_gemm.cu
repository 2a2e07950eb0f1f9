// The projection of E4M3 activations with E4M3 weights, both with one FP32 scale per block of 128:
//   out[t, n] = bf16( sum over blocks b of sa[b, t] * sw[n / 128, b] * (sum over k in b of a[t, k] * w[n, k]) )
// sa [ceil(K / 128), T] as the quantisers of fp8_block.cu write it, sw [ceil(N / 128), ceil(K / 128)].  A block's products
// are summed in FP32, multiplied by the two scales and added to the running FP32 sum; the one rounding is to bf16.
#include "device_utils.cuh"
#include "host_checks.hpp"
#include "q3x_b200.h"

namespace q3x {
namespace {

constexpr int kBlockK = Q3X_B200_FP8_BLOCK;  // 128
constexpr int kTile = 64, kStep = 32, kThreads = 256;

__device__ __forceinline__ float2 decode2(uint32_t pair) {  // two E4M3 codes -> two floats, exactly
  uint32_t half2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(half2) : "h"(static_cast<uint16_t>(pair)));
  float2 f;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.f32.f16 %0, lo;\ncvt.f32.f16 %1, hi;\n}" : "=f"(f.x), "=f"(f.y) : "r"(half2));
  return f;
}

// 64 tokens x 64 outputs per CTA, 4 x 4 per thread, codes widened to FP32 in shared memory 32 columns at a time.
__global__ void __launch_bounds__(kThreads) block_gemm_kernel(const uint8_t* __restrict__ w, const float* __restrict__ sw,
                                                              const uint8_t* __restrict__ a, const float* __restrict__ sa,
                                                              size_t tokens, size_t n, size_t k, uint16_t* __restrict__ out) {
  __shared__ float as[kStep][kTile + 4], ws[kStep][kTile + 4];
  const size_t t0 = static_cast<size_t>(blockIdx.y) * kTile, n0 = static_cast<size_t>(blockIdx.x) * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const size_t blocks = (k + kBlockK - 1) / kBlockK;
  float total[4][4] = {};
  for (size_t b = 0; b < blocks; ++b) {
    float part[4][4] = {};
    for (int step = 0; step < kBlockK; step += kStep) {
      const int r = threadIdx.x / 4, c = (threadIdx.x % 4) * 8;
      const size_t col = b * kBlockK + step + c;
      const uint2 av = t0 + r < tokens && col < k ? *reinterpret_cast<const uint2*>(a + (t0 + r) * k + col) : make_uint2(0, 0);
      const uint2 wv = n0 + r < n && col < k ? *reinterpret_cast<const uint2*>(w + (n0 + r) * k + col) : make_uint2(0, 0);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 fa = decode2((i < 2 ? av.x : av.y) >> (16 * (i & 1)) & 0xffffu);
        const float2 fw = decode2((i < 2 ? wv.x : wv.y) >> (16 * (i & 1)) & 0xffffu);
        as[c + 2 * i][r] = fa.x;
        as[c + 2 * i + 1][r] = fa.y;
        ws[c + 2 * i][r] = fw.x;
        ws[c + 2 * i + 1][r] = fw.y;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kStep; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[kk][ty * 4 + i], ws[kk][tx * 4 + j], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t t = t0 + ty * 4 + i;
      const float s = t < tokens ? sa[b * tokens + t] : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const size_t o = n0 + tx * 4 + j;
        if (o < n) total[i][j] = fmaf(__fmul_rn(s, sw[o / kBlockK * blocks + b]), part[i][j], total[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const size_t t = t0 + ty * 4 + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const size_t o = n0 + tx * 4 + j;
      if (t < tokens && o < n) out[t * n + o] = float_to_bf16(total[i][j]);
    }
  }
}

}  // namespace
}  // namespace q3x

using namespace q3x;
using namespace q3x::host;

extern "C" int q3x_b200_fp8_block_gemm_bf16(const uint8_t* weights, const float* weight_scales, const uint8_t* activations,
                                            const float* activation_scales, size_t tokens, size_t out_features,
                                            size_t in_features, uint16_t* out, void* stream) {
  if (tokens == 0 || out_features == 0) return kOk;
  if (in_features == 0 || in_features % 16 != 0 || out_features % 8 != 0) return kInvalid;
  if (tokens > 0x7fffffffu || out_features > 0x7fffffffu || in_features > 0x7fffffffu) return kInvalid;
  if (weights == nullptr || weight_scales == nullptr || activations == nullptr || activation_scales == nullptr || out == nullptr)
    return kInvalid;
  const size_t blocks = (in_features + kBlockK - 1) / kBlockK;
  const Span so = span(out, tokens * out_features * 2);
  const Span inputs[] = {span(weights, out_features * in_features), span(activations, tokens * in_features),
                         span(weight_scales, (out_features + kBlockK - 1) / kBlockK * blocks * sizeof(float)),
                         span(activation_scales, blocks * tokens * sizeof(float))};
  if (wraps(so)) return kInvalid;
  for (const Span& i : inputs)
    if (wraps(i) || overlap(so, i)) return kInvalid;
  if (!aligned16(weights) || !aligned16(activations) || !aligned16(out) ||
      (reinterpret_cast<uintptr_t>(weight_scales) & 3u) != 0 || (reinterpret_cast<uintptr_t>(activation_scales) & 3u) != 0)
    return kNotSupported;
  const size_t token_tiles = (tokens + kTile - 1) / kTile, out_tiles = (out_features + kTile - 1) / kTile;
  if (token_tiles > 65535u) return kNotSupported;
  clear_stale_error();
  block_gemm_kernel<<<dim3(static_cast<unsigned>(out_tiles), static_cast<unsigned>(token_tiles)), kThreads, 0,
                      as_stream(stream)>>>(weights, weight_scales, activations, activation_scales, tokens, out_features,
                                           in_features, out);
  return launch_status();
}
