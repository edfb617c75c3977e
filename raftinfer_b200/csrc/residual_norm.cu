// Residual addition, RMS norm and 8-bit output of hidden rows.
//
//   h = x + r,   y = h / sqrt(mean(h^2) + eps) * w,   codes = round(y / s),  s = 2^e of the group's largest |y|
//
// One CTA a row; the row stays in registers between the sum of squares and the output, eight columns a thread at a time, all
// in FP32.  One rounding per output.  Bytes: x, r read, h and the output written, once each; bound by memory.

#include "kv_cache.hpp"
#include "residual_norm.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rib200 {
namespace {

template <class T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <class T> struct alignas(16) Eight { T at[8]; };

constexpr int kThreads = 256;
constexpr int kMaxPieces = kResidualNormMaxColumns / (8 * kThreads);

template <class T, class W> __global__ void __launch_bounds__(kThreads) residual_norm_kernel(const ResidualNormArgs p) {
  __shared__ float partial[kThreads / 32];
  __shared__ float row_amax[kThreads / 32];
  grid_dependency_wait();
  grid_dependents_may_launch();
  const std::size_t row = blockIdx.x;
  const std::uint32_t pieces = p.columns / 8;
  float h[kMaxPieces][8];
  float sum = 0.0F;
#pragma unroll
  for (int i = 0; i < kMaxPieces; ++i) {
    const std::uint32_t piece = threadIdx.x + i * kThreads;
    if (piece < pieces) {
      const std::size_t at = row * pieces + piece;
      const Eight<T> x = static_cast<const Eight<T> *>(p.input)[at];
      Eight<T> r{};
      if (p.residual != nullptr) {
        r = static_cast<const Eight<T> *>(p.residual)[at];
      }
      Eight<T> back;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = to_float(x.at[e]) + (p.residual != nullptr ? to_float(r.at[e]) : 0.0F);
        sum = fmaf(h[i][e], h[i][e], sum);
        back.at[e] = from_float<T>(h[i][e]);
      }
      if (p.residual_out != nullptr) {
        static_cast<Eight<T> *>(p.residual_out)[at] = back;
      }
    }
  }
  for (int step = 16; step > 0; step /= 2) {
    sum += __shfl_xor_sync(0xFFFFFFFFU, sum, step);
  }
  if (threadIdx.x % 32 == 0) {
    partial[threadIdx.x / 32] = sum;
  }
  __syncthreads();
  sum = 0.0F;
  for (int w = 0; w < kThreads / 32; ++w) {
    sum += partial[w];
  }
  const float factor = 1.0F / sqrtf(sum / static_cast<float>(p.columns) + p.epsilon);
  float amax = 0.0F;
#pragma unroll
  for (int i = 0; i < kMaxPieces; ++i) {
    const std::uint32_t piece = threadIdx.x + i * kThreads;
    if (piece < pieces) {
      const Eight<W> w = static_cast<const Eight<W> *>(p.weight)[piece];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = h[i][e] * factor * to_float(w.at[e]);
        amax = fmaxf(amax, kv8_finite_magnitude(h[i][e]));
      }
    }
  }
  if (!p.eight_bit) {
#pragma unroll
    for (int i = 0; i < kMaxPieces; ++i) {
      const std::uint32_t piece = threadIdx.x + i * kThreads;
      if (piece < pieces) {
        Eight<T> out;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          out.at[e] = from_float<T>(h[i][e]);
        }
        static_cast<Eight<T> *>(p.output)[row * pieces + piece] = out;
      }
    }
    return;
  }
  if (p.group_columns == 0) {
    for (int step = 16; step > 0; step /= 2) {
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFU, amax, step));
    }
    if (threadIdx.x % 32 == 0) {
      row_amax[threadIdx.x / 32] = amax;
    }
    __syncthreads();
    amax = 0.0F;
    for (int w = 0; w < kThreads / 32; ++w) {
      amax = fmaxf(amax, row_amax[w]);
    }
    if (threadIdx.x == 0) {
      p.scales[row] = kv8_scale(amax);
    }
  }
  const std::uint32_t group_pieces = p.group_columns / 8; // 4 or 16 neighbouring lanes
#pragma unroll
  for (int i = 0; i < kMaxPieces; ++i) {
    const std::uint32_t piece = threadIdx.x + i * kThreads;
    const bool live = piece < pieces;
    float group_amax = amax;
    if (p.group_columns != 0) {
      group_amax = 0.0F;
      if (live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          group_amax = fmaxf(group_amax, kv8_finite_magnitude(h[i][e]));
        }
      }
      for (std::uint32_t step = group_pieces / 2; step > 0; step /= 2) {
        group_amax = fmaxf(group_amax, __shfl_xor_sync(0xFFFFFFFFU, group_amax, step));
      }
    }
    if (live) {
      const float scale = kv8_scale(group_amax);
      const float inverse = kv8_inverse(scale);
      if (p.group_columns != 0 && piece % group_pieces == 0) {
        p.scales[row * (p.columns / p.group_columns) + piece / group_pieces] = scale;
      }
      std::uint32_t w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        w[k] = kv8_codes2(h[i][4 * k] * inverse, h[i][4 * k + 1] * inverse) |
               (kv8_codes2(h[i][4 * k + 2] * inverse, h[i][4 * k + 3] * inverse) << 16);
      }
      static_cast<uint2 *>(p.output)[row * pieces + piece] = make_uint2(w[0], w[1]);
    }
  }
}

template <class T> void launch_for(const ResidualNormArgs &a, cudaStream_t stream) {
  auto run = [&](auto kernel) {
    launch_programmatic(kernel, dim3(a.rows), dim3(kThreads), 0, stream, "RMS norm launch", a);
  };
  a.weight_dtype == RIB200_DTYPE_F32 ? run(residual_norm_kernel<T, float>) : run(residual_norm_kernel<T, __nv_bfloat16>);
}

} // namespace

void launch_residual_norm(const ResidualNormArgs &a, cudaStream_t stream) {
  if (a.dtype == RIB200_DTYPE_F32) {
    launch_for<float>(a, stream);
  } else if (a.dtype == RIB200_DTYPE_F16) {
    launch_for<__half>(a, stream);
  } else {
    launch_for<__nv_bfloat16>(a, stream);
  }
}

} // namespace rib200
