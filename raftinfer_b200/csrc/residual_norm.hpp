// Arguments of the residual RMS norm kernel.
#pragma once

#include "common.hpp"

#include <cstdint>

namespace rib200 {

constexpr std::uint32_t kResidualNormMaxColumns = 16384;

struct ResidualNormArgs {
  const void *input, *residual, *weight;
  void *output;
  float *scales;
  void *residual_out;
  std::uint32_t rows, columns, group_columns;
  float epsilon;
  int32_t dtype, weight_dtype;
  bool eight_bit;
};
void launch_residual_norm(const ResidualNormArgs &args, cudaStream_t stream);

} // namespace rib200
