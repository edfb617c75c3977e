// Residual addition, RMS norm and 8-bit output of hidden rows.
//
//   h = x + r,   y = h / sqrt(mean(h^2) + eps) * w,   codes = round(y / s),  s = 2^e of the group's largest |y|
//
// A CTA takes a row at a time, eight columns to a thread in each of one, two or four pieces; the row stays in registers
// between the sum of squares and the output.  h is FP32; codes are the value rounded once (see below), other outputs FP32
// arithmetic rounded once, for rows of any magnitude.  Bytes: x, r read, h and the output written, once each; bound by memory.
// Many rows: all CTAs are resident, keep their columns' weights and fetch their next row while the current one is reduced.
// 4096 rows of 4096 columns: BF16 to BF16 23.3 us (5.8 TB/s), BF16 to 8 bits 27 (4.4 TB/s, two thirds of the copy rate: issue
// slots, and warps that wait for the row's barrier and the group's shuffles; 21.9 with codes that one value in a million misses);
// 2709 FP32 rows to FP32 30.5 (5.8 TB/s).  A CTA for each row took 71.6 (8 bits) and 40.1 (FP32).

#include "kv_cache.hpp"
#include "residual_norm.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

namespace rib200 {
namespace {

constexpr float kLargest = 3.4028234663852886e38F;
constexpr std::uint32_t kNear = 4; // units of the last place

// Eight neighbouring columns as they lie in memory, and as FP32.
template <class T> struct alignas(16) Eight { std::uint32_t word[sizeof(T) * 2]; };

template <class T> __device__ __forceinline__ void unpack(const Eight<T> &v, float (&out)[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) * 2); ++i) {
    if constexpr (sizeof(T) == 4) {
      out[i] = __uint_as_float(v.word[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      out[2 * i] = __uint_as_float(v.word[i] << 16);
      out[2 * i + 1] = __uint_as_float(v.word[i] & 0xFFFF0000U);
    } else {
      const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&v.word[i]));
      out[2 * i] = two.x;
      out[2 * i + 1] = two.y;
    }
  }
}
template <class T> __device__ __forceinline__ Eight<T> pack(const float (&v)[8]) {
  Eight<T> out;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) * 2); ++i) {
    if constexpr (sizeof(T) == 4) {
      out.word[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      out.word[i] = *reinterpret_cast<const std::uint32_t *>(&two);
    } else {
      const __half2 two = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      out.word[i] = *reinterpret_cast<const std::uint32_t *>(&two);
    }
  }
  return out;
}

// Each warp's sum or maximum into `slots`, which holds a value for each of 16 warps (zeros for those that the CTA does not
// have) and which no one may still read.
template <class V, class Op> __device__ __forceinline__ void over_warps(V v, V *slots, Op op) {
#pragma unroll
  for (int step = 16; step > 0; step /= 2) {
    v = op(v, __shfl_xor_sync(0xFFFFFFFFU, v, step));
  }
  if (threadIdx.x % 32 == 0) {
    slots[threadIdx.x / 32] = v;
  }
  __syncthreads();
}

// Mean of a row's squares, from the warps' sums, plus epsilon.
template <int Warps>
__device__ __forceinline__ double mean_of(const double *slots, double one_column, double epsilon) {
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < Warps; i += 2) {
    const double2 two = reinterpret_cast<const double2 *>(slots)[i / 2];
    total += two.x + two.y;
  }
  return fma(total, one_column, epsilon);
}
// m^(-1/2), good to the last place but one: m = r 4^k with r in [1/2, 2), an approximation, and Newton's step twice.
__device__ __forceinline__ double wide_factor(double m) {
  if (!(m > 0.0) || m > 1.0e300) { // zeros, infinities, not-a-numbers; the squares of FP32 numbers are in between
    return static_cast<double>(rsqrtf(static_cast<float>(m)));
  }
  const int k = (__double2hiint(m) >> 21) - 511;
  const double r = __hiloint2double(__double2hiint(m) - (k << 21), __double2loint(m));
  double f = static_cast<double>(rsqrtf(static_cast<float>(r)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f = fma(0.5 * f, fma(-r * f, f, 1.0), f);
  }
  return __hiloint2double(__double2hiint(f) - (k << 20), __double2loint(f));
}

// Group: columns that share a scale (32 or 128; 0 a whole row), -1 an output in T.
template <class T, class W, int Pieces, int Group>
__global__ void __launch_bounds__(sizeof(T) == 2 && Pieces <= 2 ? 256 : 512, sizeof(T) == 2 && Pieces <= 2 ? 4 : 1)
    residual_norm_kernel(const ResidualNormArgs p) {
  constexpr int kWarps = Pieces <= 2 ? 8 : 16;
  __shared__ alignas(16) double sum_slots[2][16]; // [row parity][warp]
  __shared__ alignas(16) float max_slots[2][16];
  if (threadIdx.x < 32) {
    sum_slots[threadIdx.x / 16][threadIdx.x % 16] = 0.0;
    max_slots[threadIdx.x / 16][threadIdx.x % 16] = 0.0F;
  }
  __syncthreads();
  grid_dependency_wait();
  grid_dependents_may_launch();
  const std::uint32_t pieces = p.columns / 8;
  const bool has_residual = p.residual != nullptr;
  const Eight<T> *input = static_cast<const Eight<T> *>(p.input);
  const Eight<T> *residual = static_cast<const Eight<T> *>(p.residual);
  Eight<W> weight[Pieces]{};
  Eight<T> next_x[Pieces];
  Eight<T> next_r[Pieces];
  auto fetch = [&](std::size_t row) {
#pragma unroll
    for (int i = 0; i < Pieces; ++i) {
      const std::uint32_t piece = threadIdx.x + i * blockDim.x;
      if (piece < pieces) {
        next_x[i] = input[row * pieces + piece];
        if (has_residual) {
          next_r[i] = residual[row * pieces + piece];
        }
      }
    }
  };
  fetch(blockIdx.x);
#pragma unroll
  for (int i = 0; i < Pieces; ++i) {
    const std::uint32_t piece = threadIdx.x + i * blockDim.x;
    if (piece < pieces) {
      weight[i] = static_cast<const Eight<W> *>(p.weight)[piece];
    }
  }
  const double one_column = 1.0 / static_cast<double>(p.columns);
  const double epsilon = static_cast<double>(p.epsilon);
  // |w| <= 2^16 keeps h * factor * w apart from what underflows: where h * factor (|h| factor <= 2^7) is under the smallest normal
  // number, y is under 2^-110 and its code 0 at the smallest scale.
  bool large_weights = false;
#pragma unroll
  for (int i = 0; i < (Group >= 0 ? Pieces : 0); ++i) {
    float w[8];
    unpack<W>(weight[i], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      large_weights = large_weights || !(fabsf(w[e]) <= 65536.0F);
    }
  }
  std::uint32_t parity = 0;
  for (std::size_t row = blockIdx.x; row < p.rows; row += gridDim.x, parity ^= 1U) {
    float h[Pieces][8];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < Pieces; ++i) {
      const std::uint32_t piece = threadIdx.x + i * blockDim.x;
      if (piece < pieces) {
        unpack<T>(next_x[i], h[i]);
        if (has_residual) {
          float r[8];
          unpack<T>(next_r[i], r);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            h[i][e] += r[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum = fma(static_cast<double>(h[i][e]), static_cast<double>(h[i][e]), sum);
        }
        if (p.residual_out != nullptr) {
          static_cast<Eight<T> *>(p.residual_out)[row * pieces + piece] = pack<T>(h[i]);
        }
      }
    }
    if (row + gridDim.x < p.rows) {
      fetch(row + gridDim.x);
    }
    // The squares are summed in 64 bits: large rows do not overflow, and the factor, whose error would move all of a row's
    // values towards a code's border together, is good to the last place.  (A few columns may hold most of the sum, so that 32-bit
    // errors do not average out.)  It is an approximation f of m^(-1/2) and what Newton's step adds to it, f (1 - m f^2) / 2.
    over_warps(sum, sum_slots[parity], [](double a, double b) { return a + b; });
    const double mean = mean_of<kWarps>(sum_slots[parity], one_column, epsilon);
    // y = h scale w factor.  8 bit: scale is 1, and factor is a not-a-number where these products may leave FP32's range.  Else
    // scale is a power of two that brings the row to about one (2^126 and 2^-126 at most), so that they do not.
    float scale = 1.0F;
    float factor = __uint_as_float(0x7FFFFFFFU);
    double scaled = mean;
    if (Group < 0 && mean > 0.0 && mean < 1.0e300) {
      const int k = min(max((__double2hiint(mean) >> 21) - 511, -126), 126);
      scale = __uint_as_float(static_cast<std::uint32_t>(127 - k) << 23);
      scaled = __hiloint2double(__double2hiint(mean) - (k << 21), __double2loint(mean));
    }
    if (Group < 0 || (!large_weights && mean > 1.0e-30 && mean < 1.0e30)) {
      const float m = static_cast<float>(scaled), m_rest = static_cast<float>(scaled - static_cast<double>(m));
      factor = rsqrtf(m);
      if (Group >= 0 || (m > 0.0F && m < kLargest)) {
        const float square = factor * factor, square_rest = fmaf(factor, factor, -square);
        factor = fmaf(0.5F * factor, fmaf(-m, square_rest, fmaf(-m_rest, square, fmaf(-m, square, 1.0F))), factor);
      }
    }
#pragma unroll
    for (int i = 0; i < Pieces; ++i) {
      float w[8];
      unpack<W>(weight[i], w);
      float y[8];
      std::uint32_t near = 0xFFFFFFFFU;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = Group < 0 ? h[i][e] * scale * w[e] * factor : h[i][e] * factor * w[e];
        near = min(near, (__float_as_uint(y[e]) + kNear) & 0x7FFFFU);
      }
      if constexpr (Group >= 0) {
        // The middle between two codes, and the largest value of a scale, have nineteen zeros at the end, and y (three
        // roundings) is within three units of its last place.  Where it comes near such a number (one value in 58000; zeros are
        // what they are) its piece is worked out again in 64 bits, and the last bit says on which side of it the value lies: a
        // code is the value rounded once.  So is every value of a row whose factor, or of a thread whose weights, may take the
        // products out of FP32's range: factor and y are then the not-a-number whose bits but the sign are ones, which looks the
        // same.
        bool again = false;
        if (near <= 2 * kNear) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            again = again || (y[e] != 0.0F && ((__float_as_uint(y[e]) + kNear) & 0x7FFFFU) <= 2 * kNear);
          }
        }
        if (again) {
          const double wide = wide_factor(mean_of<kWarps>(sum_slots[parity], one_column, epsilon));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double exact = static_cast<double>(h[i][e]) * static_cast<double>(w[e]) * wide;
            y[e] = static_cast<float>(exact);
            // within 2^-50 of such a number, about what the sum of squares leaves uncertain, a value counts as the number
            const double left = exact - static_cast<double>(y[e]);
            const std::uint32_t bits = __float_as_uint(y[e]);
            const bool middle = (bits & 0x7FFFFU) == 0 && fabsf(y[e]) <= kLargest && fabs(left) > 0x1p-50 * fabs(exact);
            y[e] = middle ? __uint_as_float((left > 0.0) == (exact > 0.0) ? bits + 1 : bits - 1) : y[e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = y[e];
      }
    }
    if constexpr (Group < 0) {
#pragma unroll
      for (int i = 0; i < Pieces; ++i) {
        const std::uint32_t piece = threadIdx.x + i * blockDim.x;
        if (piece < pieces) {
          static_cast<Eight<T> *>(p.output)[row * pieces + piece] = pack<T>(h[i]);
        }
      }
    } else {
      // Largest magnitudes.  A maximum passes over a not-a-number but not over an infinity, so a group with one is gone
      // through again, finite values alone.
      auto largest = [&](int i) {
        float amax = fabsf(h[i][0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) {
          amax = fmaxf(amax, fabsf(h[i][e]));
        }
        if (!(amax <= kLargest)) {
          amax = 0.0F;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            amax = fmaxf(amax, kv8_finite_magnitude(h[i][e]));
          }
        }
        return threadIdx.x + i * blockDim.x < pieces ? amax : 0.0F;
      };
      float amax[Pieces];
#pragma unroll
      for (int i = 0; i < Pieces; ++i) {
        amax[i] = largest(i);
      }
      if constexpr (Group == 0) {
        float row_amax = amax[0];
#pragma unroll
        for (int i = 1; i < Pieces; ++i) {
          row_amax = fmaxf(row_amax, amax[i]);
        }
        over_warps(row_amax, max_slots[parity], [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
        for (int i = 0; i < kWarps; i += 4) {
          const float4 four = reinterpret_cast<const float4 *>(max_slots[parity])[i / 4];
          row_amax = fmaxf(row_amax, fmaxf(fmaxf(four.x, four.y), fmaxf(four.z, four.w)));
        }
#pragma unroll
        for (int i = 0; i < Pieces; ++i) {
          amax[i] = row_amax;
        }
      } else {
#pragma unroll
        for (int step = Group / 16; step > 0; step /= 2) {
#pragma unroll
          for (int i = 0; i < Pieces; ++i) {
            amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xFFFFFFFFU, amax[i], step));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < Pieces; ++i) {
        const std::uint32_t piece = threadIdx.x + i * blockDim.x;
        if (piece < pieces) {
          const float scale = kv8_scale(amax[i]);
          const float inverse = kv8_inverse(scale);
          if constexpr (Group == 0) {
            if (piece == 0) {
              p.scales[row] = scale;
            }
          } else if (piece % (Group / 8) == 0) {
            p.scales[row * (pieces / (Group / 8)) + piece / (Group / 8)] = scale;
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
  }
}

template <class T, class W, int Pieces> void launch_pieces(const ResidualNormArgs &a, cudaStream_t stream) {
  const std::uint32_t threads = (a.columns / 8 + 32 * Pieces - 1) / (32 * Pieces) * 32;
  auto run = [&](auto kernel) {
    int device = 0, sms = 0, resident = 0;
    cuda_ok(cudaGetDevice(&device), "cudaGetDevice");
    cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "SM count query");
    std::uint32_t ctas = a.rows;
    if (a.rows > static_cast<std::uint32_t>(sms)) { // every CTA resident, rows dealt in turn
      cuda_ok(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, static_cast<int>(threads), 0),
              "RMS norm occupancy");
      ctas = std::min(a.rows, static_cast<std::uint32_t>(sms * std::max(resident, 1)));
    }
    launch_programmatic(kernel, dim3(ctas), dim3(threads), 0, stream, "RMS norm launch", a);
  };
  if (!a.eight_bit) {
    run(residual_norm_kernel<T, W, Pieces, -1>);
  } else if (a.group_columns == 0) {
    run(residual_norm_kernel<T, W, Pieces, 0>);
  } else if (a.group_columns == 32) {
    run(residual_norm_kernel<T, W, Pieces, 32>);
  } else {
    run(residual_norm_kernel<T, W, Pieces, 128>);
  }
}

template <class T, class W> void launch_weight(const ResidualNormArgs &a, cudaStream_t stream) {
  if (a.columns <= 8 * 256) {
    launch_pieces<T, W, 1>(a, stream);
  } else if (a.columns <= 8 * 512) {
    launch_pieces<T, W, 2>(a, stream);
  } else {
    launch_pieces<T, W, 4>(a, stream);
  }
}

template <class T> void launch_for(const ResidualNormArgs &a, cudaStream_t stream) {
  a.weight_dtype == RIB200_DTYPE_F32 ? launch_weight<T, float>(a, stream) : launch_weight<T, __nv_bfloat16>(a, stream);
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
