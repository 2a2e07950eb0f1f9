// Activations in E4M3 with one FP32 scale per row and block of 128 columns, the operand of q3x_b200_fp8_block_gemm_bf16:
// the block quantiser of a bf16 tensor, and the residual add + centred RMSNorm and the SwiGLU that quantise their result
// in the same pass.  No counterpart in the reference (its FP8 weights carry one scale per tensor and multiply bf16
// activations, src/kernels/reference/gemv_reference.cpp:113-140).
//
//   amax  = largest finite |y| of the block        scale = amax == 0 ? 1 : max(amax / 448, 2^-126)
//   code  = E4M3(y * (1 / scale)), round to nearest even, saturating at 448; a NaN stays a NaN, an infinity saturates
//
// 448 is the largest E4M3 value; the floor keeps 1 / scale finite.  y is the operator's FP32 result: it is rounded once,
// to E4M3, and not to bf16 on the way (two roundings in a row move values next to a midpoint to the wrong side).  Scales
// lie block-major, [ceil(columns / 128), rows]: the product reads one block's scales of neighbouring rows together.
//
// Every kernel is a stream that reads its operands once.  A lane owns eight neighbouring columns (one 128-bit load per
// operand, one 64-bit store of codes), sixteen lanes own a block, so a block's amax takes four shuffles and nothing leaves
// registers between the arithmetic and the codes.  Many rows are bound by HBM and, in long runs, by the power that the
// instructions take beside it (SwiGLU of 8192 x 17408: 120 us at first, 140 after two seconds, at 1.65 GHz).
#include <type_traits>

#include "device_utils.cuh"
#include "host_checks.hpp"
#include "internal.hpp"
#include "norm_math.cuh"
#include "pointwise_ops.cuh"
#include "q3x_b200.h"

namespace q3x {
namespace {

constexpr int kBlockCols = Q3X_B200_FP8_BLOCK;    // 128
constexpr int kBlockLanes = kBlockCols / 8;       // 16 lanes of eight columns
constexpr float kTopE4m3 = 448.0f;
constexpr float kSmallestScale = 1.1754943508222875e-38f;  // 2^-126

// Largest finite magnitude of eight values, 0 if there is none: fmaxf drops a NaN next to a number (hence the last
// fmaxf with 0, for eight of them), and only a vector that holds an infinity is looked at again.
__device__ __forceinline__ float finite_amax8(const float (&y)[8]) {
  float t = fmaxf(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))),
                  fmaxf(fmaxf(fabsf(y[4]), fabsf(y[5])), fmaxf(fabsf(y[6]), fabsf(y[7]))));
  if (t == INFINITY) {
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaxf(t, fabsf(y[i]) == INFINITY ? 0.0f : fabsf(y[i]));
  }
  return fmaxf(t, 0.0f);
}
__device__ __forceinline__ float block_amax(float t) {
#pragma unroll
  for (int o = kBlockLanes / 2; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(kFullMask, t, o));
  return t;
}
// amax / 448 correctly rounded, from the rounded reciprocal, the remainder (exact: q * 448 has 27 bits) and one correction
// (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990).  The quotient is A 2^s / 7
// steps for an integer A, so at least 1/14 step away from every midpoint, and the corrected value is 2^-25 step off: it
// rounds the same way.  (Below 2^-126 the floor decides, and nothing there comes out above it.)  Every lane does this, and
// the streams are held back by the power that their instructions take: 8192 x 6144 28.7 -> 27.6 us against a division.
__device__ __forceinline__ float scale_of_amax(float amax) {
  constexpr float kReciprocal = 1.0f / kTopE4m3;
  const float q = __fmul_rn(amax, kReciprocal), rest = __fmaf_rn(-q, kTopE4m3, amax);
  return amax == 0.0f ? 1.0f : fmaxf(__fmaf_rn(rest, kReciprocal, q), kSmallestScale);
}
// Eight codes, column i in byte i.
__device__ __forceinline__ uint2 encode8(const float (&y)[8], float inverse) {
  uint16_t pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // two products per instruction, each rounded like __fmul_rn
    const float2 q = mul2(make_float2(y[2 * i], y[2 * i + 1]), make_float2(inverse, inverse));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair[i]) : "f"(q.y), "f"(q.x));
  }
  return make_uint2(pair[0] | (static_cast<uint32_t>(pair[1]) << 16), pair[2] | (static_cast<uint32_t>(pair[3]) << 16));
}

// ---- pointwise sources: FP32 result of eight columns -----------------------------------------------------------
struct FromTensor {
  static constexpr bool kTwoInputs = false;
  static __device__ __forceinline__ void apply(const uint4& a, const uint4&, float (&y)[8]) { unpack8(a, y); }
};
struct FromSiluMul {  // first operand = gate, second = up
  static constexpr bool kTwoInputs = true;
  static __device__ __forceinline__ void apply(const uint4& a, const uint4& b, float (&y)[8]) {
    float g[8], u[8];
    unpack8(a, g);
    unpack8(b, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = SiluMul::apply(g[i], u[i]);
  }
};

constexpr int kThreads = 256;

// kPerRow threads of a CTA share a row (a power of two, so that narrow rows do not leave a CTA idle: 8192 x 256 took 9 us
// with a CTA per row), each with kDepth vectors of every operand in flight; the grid's second dimension splits wide rows
// when there are few of them.
template <class Source, int kPerRow, int kDepth>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b,
                                                                 size_t row_stride, size_t rows, int row_vectors,
                                                                 uint8_t* __restrict__ codes, float* __restrict__ scales) {
  release_next_kernel();
  wait_for_prior_kernels();
  const size_t row = static_cast<size_t>(blockIdx.x) * (kThreads / kPerRow) + threadIdx.x / kPerRow;
  const int lane = threadIdx.x % kPerRow, step = gridDim.y * kPerRow;
  const bool live = row < rows;
  const uint16_t* a_row = a + row * row_stride;
  const uint16_t* b_row = Source::kTwoInputs ? b + row * row_stride : nullptr;
  uint8_t* code_row = codes + row * static_cast<size_t>(row_vectors) * 8;
  // (a whole warp makes the same turns, whatever its lanes' last vector: all of them take part in the shuffles)
  for (int first = blockIdx.y * kPerRow; first < row_vectors; first += kDepth * step) {
    uint4 x[kDepth], z[kDepth];
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const int v = first + k * step + lane;
      x[k] = z[k] = make_uint4(0, 0, 0, 0);
      if (live && v < row_vectors) {
        x[k] = ld_stream(a_row + static_cast<size_t>(v) * 8);
        if (Source::kTwoInputs) z[k] = ld_stream(b_row + static_cast<size_t>(v) * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const int v = first + k * step + lane;
      if (first + k * step >= row_vectors) break;
      float y[8];
      Source::apply(x[k], z[k], y);
      const float scale = scale_of_amax(block_amax(finite_amax8(y)));
      if (live && v < row_vectors) {
        *reinterpret_cast<uint2*>(code_row + static_cast<size_t>(v) * 8) = encode8(y, __frcp_rn(scale));
        if ((lane & (kBlockLanes - 1)) == 0) scales[static_cast<size_t>(v / kBlockLanes) * rows + row] = scale;
      }
    }
  }
}

// One CTA per row, kDepth vectors per thread; the row stays in registers between the sum of squares and the codes, and the
// weights are requested with it.
constexpr int kMostThreads = 512;
template <int kDepth>
__global__ void __launch_bounds__(kDepth == 1 ? 1024 : kMostThreads)
    residual_norm_fp8_kernel(const uint16_t* left, const uint16_t* right, const uint16_t* __restrict__ weight, size_t rows,
                             int row_vectors, float inv_width, float eps, uint16_t* residual_out, uint16_t* normalized_out,
                             bool coherent, uint8_t* __restrict__ codes, float* __restrict__ scales) {
  __shared__ float scratch[32];
  release_next_kernel();
  wait_for_prior_kernels();
  const size_t row = blockIdx.x;
  const size_t base = row * static_cast<size_t>(row_vectors) * 8;
  uint4 x[kDepth], r[kDepth], w[kDepth];
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    const int v = threadIdx.x + k * blockDim.x;
    x[k] = r[k] = w[k] = make_uint4(0, 0, 0, 0);
    if (v < row_vectors) {
      x[k] = ld_stream(left + base + v * 8);
      r[k] = coherent ? ld_vec(right + base + v * 8) : ld_stream(right + base + v * 8);
      w[k] = ld_weight(weight + v * 8);
    }
  }
  float partial = 0.0f;
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    const int v = threadIdx.x + k * blockDim.x;
    float l[8], rr[8];
    unpack8(x[k], l);
    unpack8(r[k], rr);
    add8(l, rr);
    x[k] = pack8(l);
    if (v < row_vectors) st_vec(residual_out + base + v * 8, x[k]);
    partial += sum_squares8(x[k]);
  }
  // the sum over the CTA's warps, in the same order in every thread
  partial = group_sum<32>(partial);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = partial;
  __syncthreads();
  float total = 0.0f;
  for (int i = 0; i < blockDim.x / 32; ++i) total += scratch[i];
  const float inv = inverse_rms(total, inv_width, eps);
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    const int v = threadIdx.x + k * blockDim.x;
    float y[8], wf[8];
    unpack8(x[k], y);
    unpack8(w[k], wf);
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 gamma = add2(make_float2(wf[i], wf[i + 1]), make_float2(1.0f, 1.0f));
      const float2 n = mul2(mul2(make_float2(y[i], y[i + 1]), inv2), gamma);
      y[i] = n.x;
      y[i + 1] = n.y;
    }
    // (a lane past the row's end holds 0 * inv: not NaN unless the row's own sum is, and then fmaxf drops it)
    const float scale = scale_of_amax(block_amax(finite_amax8(y)));
    if (v < row_vectors) {
      if (normalized_out != nullptr) st_vec(normalized_out + base + v * 8, pack8(y));
      *reinterpret_cast<uint2*>(codes + base + v * 8) = encode8(y, __frcp_rn(scale));
      if ((threadIdx.x & (kBlockLanes - 1)) == 0) scales[static_cast<size_t>(v / kBlockLanes) * rows + row] = scale;
    }
  }
}

size_t block_count(size_t cols) { return (cols + kBlockCols - 1) / kBlockCols; }

// Checks of the codes and scales of a [rows, cols] result against each other; the shape is known not to overflow.
int check_codes(const uint8_t* codes, const float* scales, size_t rows, size_t cols, host::Span* sc, host::Span* ss) {
  using namespace host;
  if (codes == nullptr || scales == nullptr) return kInvalid;
  *sc = span(codes, rows * cols);
  *ss = span(scales, rows * block_count(cols) * sizeof(float));
  if (wraps(*sc) || wraps(*ss) || overlap(*sc, *ss)) return kInvalid;
  return kOk;
}
bool codes_aligned(const uint8_t* codes, const float* scales) {
  return host::aligned16(codes) && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0;
}

template <class Source, int kPerRow, int kDepth>
void launch_quantize_deep(const uint16_t* a, const uint16_t* b, size_t row_stride, size_t rows, int row_vectors, uint8_t* codes,
                             float* scales, cudaStream_t s) {
  constexpr auto kernel = quantize_rows_kernel<Source, kPerRow, kDepth>;
  const size_t ctas = (rows + kThreads / kPerRow - 1) / (kThreads / kPerRow), chunks = (row_vectors + kPerRow - 1) / kPerRow;
  const size_t resident = host::resident_grid(kernel, kThreads);
  size_t splits = ctas >= resident ? 1 : (resident + ctas - 1) / ctas;
  if (splits > chunks) splits = chunks;
  // (overlapping with the kernel before takes half a microsecond off at every size: 333 x 6144 2.75 -> 2.2 us)
  host::launch_kernel(kernel, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(splits)), dim3(kThreads), 0, s, true, a, b,
                      row_stride, rows, row_vectors, codes, scales);
}

// Three vectors in flight per thread once the rows alone fill the GPU (8192 x 6144: 25.5 us, 0.91 of a copy's rate; with scales
// by division three took 26.9, one 30.3, two 29.0, four 29.1; SwiGLU of 8192 x 17408: 118.6 us, 0.92; 122.5, 125.9, 128.9,
// 134.4), one while they do not (333 x 6144: 2.2 us; SwiGLU of 1 x 17408 1.4 us against 1.5).
template <class Source, int kPerRow>
void launch_quantize_per_row(const uint16_t* a, const uint16_t* b, size_t row_stride, size_t rows, int row_vectors, uint8_t* codes,
                             float* scales, cudaStream_t s) {
  if (rows / (kThreads / kPerRow) >= host::resident_grid(quantize_rows_kernel<Source, kPerRow, 3>, kThreads))
    launch_quantize_deep<Source, kPerRow, 3>(a, b, row_stride, rows, row_vectors, codes, scales, s);
  else
    launch_quantize_deep<Source, kPerRow, 1>(a, b, row_stride, rows, row_vectors, codes, scales, s);
}

template <class Source>
int launch_quantize_rows(const uint16_t* a, const uint16_t* b, size_t row_stride, size_t rows, size_t cols, uint8_t* codes,
                         float* scales, void* stream) {
  using namespace host;
  const int vectors = static_cast<int>(cols / 8);
  cudaStream_t s = as_stream(stream);
  clear_stale_error();
  if (vectors <= 16) launch_quantize_per_row<Source, 16>(a, b, row_stride, rows, vectors, codes, scales, s);
  else if (vectors <= 64) launch_quantize_per_row<Source, 64>(a, b, row_stride, rows, vectors, codes, scales, s);
  else if (vectors <= 128) launch_quantize_per_row<Source, 128>(a, b, row_stride, rows, vectors, codes, scales, s);
  else launch_quantize_per_row<Source, 256>(a, b, row_stride, rows, vectors, codes, scales, s);
  return launch_status();
}

template <int kDepth>
void launch_residual_norm(size_t rows, cudaStream_t s, const uint16_t* left, const uint16_t* right, const uint16_t* weight,
                          int row_vectors, float inv_width, float eps, uint16_t* residual_out, uint16_t* normalized_out,
                          bool coherent, uint8_t* codes, float* scales) {
  const int threads = ((row_vectors + kDepth - 1) / kDepth + 31) / 32 * 32;
  // Overlapping with the kernel before takes half a microsecond off (777 x 5120: 7.7 -> 7.2 us), but not where all rows are
  // resident with room to spare: they come to lie unevenly, where the kernel before left room (333 x 5120: 4.5 -> 5.0 us).
  // Half of an SM's 2048 threads separates the two.
  const bool overlap =
      host::latency_bound_launch(rows) || rows * threads >= static_cast<size_t>(host::current_device_sm_count()) * 1024;
  host::launch_kernel(residual_norm_fp8_kernel<kDepth>, dim3(static_cast<unsigned>(rows)), dim3(threads), 0, s, overlap,
                      left, right, weight, rows, row_vectors, inv_width, eps, residual_out, normalized_out, coherent, codes,
                      scales);
}

constexpr size_t kWidestRow = kMostThreads * 8 * 8;  // eight vectors of eight columns per thread

}  // namespace
}  // namespace q3x

using namespace q3x;
using namespace q3x::host;

extern "C" int q3x_b200_fp8_block_quantize(const uint16_t* in, size_t rows, size_t cols, uint8_t* codes, float* scales,
                                           void* stream) {
  if (cols % 16 != 0 || mul3_overflows(rows, cols, sizeof(uint16_t))) return kInvalid;
  if (rows == 0 || cols == 0) return kOk;
  if (in == nullptr) return kInvalid;
  Span sc, ss;
  if (check_codes(codes, scales, rows, cols, &sc, &ss) != kOk) return kInvalid;
  const Span si = span(in, rows * cols * 2);
  if (wraps(si) || overlap(si, sc) || overlap(si, ss)) return kInvalid;
  if (!aligned16(in) || !codes_aligned(codes, scales) || rows > 0x7fffffffu || cols > 0x7fffffffu) return kNotSupported;
  return launch_quantize_rows<FromTensor>(in, nullptr, cols, rows, cols, codes, scales, stream);
}

extern "C" int q3x_b200_silu_mul_fp8_block(const uint16_t* gate, const uint16_t* up, size_t row_stride, size_t tokens,
                                           size_t intermediate, uint8_t* codes, float* scales, void* stream) {
  if (intermediate % 16 != 0 || row_stride < intermediate || mul3_overflows(tokens, row_stride, sizeof(uint16_t))) return kInvalid;
  if (tokens == 0 || intermediate == 0) return kOk;
  if (gate == nullptr || up == nullptr) return kInvalid;
  Span sc, ss;
  if (check_codes(codes, scales, tokens, intermediate, &sc, &ss) != kOk) return kInvalid;
  const size_t bytes = ((tokens - 1) * row_stride + intermediate) * 2;  // first to last element of either operand
  const Span sg = span(gate, bytes), su = span(up, bytes);
  if (wraps(sg) || wraps(su)) return kInvalid;
  if (overlap(sg, sc) || overlap(sg, ss) || overlap(su, sc) || overlap(su, ss)) return kInvalid;
  if (!aligned16(gate) || !aligned16(up) || row_stride % 8 != 0 || !codes_aligned(codes, scales) || tokens > 0x7fffffffu ||
      intermediate > 0x7fffffffu)
    return kNotSupported;
  return launch_quantize_rows<FromSiluMul>(gate, up, row_stride, tokens, intermediate, codes, scales, stream);
}

extern "C" int q3x_b200_residual_add_rms_norm_fp8_block(const uint16_t* left, const uint16_t* right, const uint16_t* weight,
                                                        size_t tokens, size_t hidden, float eps, uint16_t* residual_out,
                                                        uint16_t* normalized_out, uint8_t* codes, float* scales,
                                                        void* stream) {
  bool done;
  const int st = check_residual_norm(left, right, weight, tokens, hidden, eps, residual_out, normalized_out, &done);
  if (st != kOk) return st;
  if (hidden % 16 != 0) return kInvalid;
  if (done) return kOk;
  Span sc, ss;
  if (check_codes(codes, scales, tokens, hidden, &sc, &ss) != kOk) return kInvalid;
  const size_t bytes = tokens * hidden * 2;
  const Span others[] = {span(left, bytes), span(right, bytes), span(weight, hidden * 2), span(residual_out, bytes),
                         span(normalized_out, normalized_out ? bytes : 0)};
  for (const Span& o : others)
    if (overlap(o, sc) || overlap(o, ss)) return kInvalid;
  if (!aligned16(left) || !aligned16(right) || !aligned16(weight) || !aligned16(residual_out) ||
      (normalized_out != nullptr && !aligned16(normalized_out)) || !codes_aligned(codes, scales) || hidden > kWidestRow ||
      tokens > 0x7fffffffu)
    return kNotSupported;
  clear_stale_error();
  const int row_vectors = static_cast<int>(hidden / 8);
  const float inv_width = 1.0f / static_cast<float>(hidden);
  cudaStream_t s = as_stream(stream);
  const bool coherent = normalized_out == right;
  auto launch = [&](auto depth) {
    launch_residual_norm<decltype(depth)::value>(tokens, s, left, right, weight, row_vectors, inv_width, eps, residual_out,
                                                 normalized_out, coherent, codes, scales);
  };
  // One vector per thread while the call is bound by latency (1 x 5120: 1.8 us, with three 2.4), three when it streams (8192 x
  // 5120: 47.8 us, 0.94 of a copy's rate; with scales by division three took 49.0, one 57.6, two 50.3, four 51.3), eight for
  // rows beyond that.
  if (row_vectors <= 64 || (row_vectors <= 1024 && latency_bound_launch(tokens))) launch(std::integral_constant<int, 1>{});
  else if (row_vectors <= 3 * kMostThreads) launch(std::integral_constant<int, 3>{});
  else launch(std::integral_constant<int, 8>{});
  return launch_status();
}
