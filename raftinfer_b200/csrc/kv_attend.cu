// Attention of single rows over a KV cache, the simple form: a CTA for one query row and head, a warp for every fourth
// visible token, a lane for eight dims; one pass with a running maximum and sum, FP32 throughout.  Single tokens are stored by
// a kernel in front.

#include "kv_store.hpp"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rib200 {
namespace {

constexpr float kLog2e = 1.4426950408889634F;

template <bool F32> __device__ __forceinline__ void load8(const void *base, std::size_t index, float (&v)[8]) {
  for (int e = 0; e < 8; ++e) {
    v[e] = F32 ? static_cast<const float *>(base)[index + e]
               : __bfloat162float(static_cast<const __nv_bfloat16 *>(base)[index + e]);
  }
}

struct AttendArgs {
  const void *query, *gate;
  void *output;
  KvCaches caches;
  const std::uint32_t *positions; // or null: row i is at past + i of one sequence
  std::uint32_t past, query_heads, window, sinks;
  unsigned int *status;
};

template <bool F32> __global__ void __launch_bounds__(128) kv_attend_kernel(const AttendArgs p) {
  __shared__ float warp_max[4], warp_sum[4], warp_acc[4][256];
  grid_dependency_wait();
  grid_dependents_may_launch();
  const std::uint32_t row = blockIdx.x;
  const std::uint32_t head = blockIdx.y;
  const std::uint32_t sequence = p.positions != nullptr ? row : 0;
  const std::uint32_t pos = p.positions != nullptr ? p.positions[row] : p.past + row;
  std::uint32_t why;
  if (!kv_servable(p.caches, sequence, pos, why)) {
    return;
  }
  const KvView view = kv_view(p.caches, sequence);
  const std::uint32_t kv_head = head / (p.query_heads / p.caches.kv_heads);
  const std::uint32_t low = pos + 1 > p.window ? pos + 1 - p.window : 0U;
  const std::uint32_t first = min(p.sinks, low);
  const std::uint32_t seen = first + (pos + 1 - low);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const std::size_t index = (static_cast<std::size_t>(row) * p.query_heads + head) * kKvHeadDim + lane * 8;
  float q[8], acc[8] = {};
  load8<F32>(p.query, index, q);
  float m = -3.0e38F, l = 0.0F;
  for (std::uint32_t i = warp; i < seen; i += 4) {
    const std::uint32_t token = i < first ? i : low + (i - first);
    const unsigned char *k_plane = view.plane(0, kv_head, token);
    const unsigned char *v_plane = view.plane(1, kv_head, token);
    if (k_plane == nullptr) {
      if (lane == 0) {
        atomicOr(p.status, static_cast<unsigned int>(RIB200_DEVICE_PAGE_OUT_OF_RANGE));
      }
      continue;
    }
    const std::uint32_t r = view.row_in_plane(token);
    float k[8], v[8];
    if (view.eight_bit) {
      const std::size_t record = static_cast<std::size_t>(r / kKv8BlockTokens) * kKv8BlockBytes;
      const float ks = *reinterpret_cast<const float *>(k_plane + record + kKv8CodeBytes);
      const float vs = *reinterpret_cast<const float *>(v_plane + record + kKv8CodeBytes);
      const unsigned char *kc = k_plane + record + (r % kKv8BlockTokens) * kKvHeadDim + lane * 8;
      const unsigned char *vc = v_plane + record + (r % kKv8BlockTokens) * kKvHeadDim + lane * 8;
      for (int e = 0; e < 8; ++e) {
        k[e] = kv8_values2(kc[e]).x * ks;
        v[e] = kv8_values2(vc[e]).x * vs;
      }
    } else {
      load8<false>(k_plane, static_cast<std::size_t>(r) * kKvHeadDim + lane * 8, k);
      load8<false>(v_plane, static_cast<std::size_t>(r) * kKvHeadDim + lane * 8, v);
    }
    float s = 0.0F;
    for (int e = 0; e < 8; ++e) {
      s += q[e] * k[e];
    }
    for (int step = 16; step > 0; step /= 2) {
      s += __shfl_xor_sync(0xFFFFFFFFU, s, step);
    }
    s *= 0.0625F;
    const float next = fmaxf(m, s);
    const float keep = exp2f((m - next) * kLog2e), take = exp2f((s - next) * kLog2e);
    l = l * keep + take;
    for (int e = 0; e < 8; ++e) {
      acc[e] = acc[e] * keep + v[e] * take;
    }
    m = next;
  }
  if (lane == 0) {
    warp_max[warp] = m;
    warp_sum[warp] = l;
  }
  for (int e = 0; e < 8; ++e) {
    warp_acc[warp][lane * 8 + e] = acc[e];
  }
  __syncthreads();
  if (warp == 0) {
    float total_max = m, total = 0.0F, out[8] = {};
    for (int w = 1; w < 4; ++w) {
      total_max = fmaxf(total_max, warp_max[w]);
    }
    for (int w = 0; w < 4; ++w) {
      const float weight = exp2f((warp_max[w] - total_max) * kLog2e);
      total += warp_sum[w] * weight;
      for (int e = 0; e < 8; ++e) {
        out[e] += warp_acc[w][lane * 8 + e] * weight;
      }
    }
    float gate[8];
    load8<F32>(p.gate, index, gate);
    for (int e = 0; e < 8; ++e) {
      const float y = out[e] / total / (1.0F + expf(-gate[e]));
      if constexpr (F32) {
        static_cast<float *>(p.output)[index + e] = y;
      } else {
        static_cast<__nv_bfloat16 *>(p.output)[index + e] = __float2bfloat16_rn(y);
      }
    }
  }
}

} // namespace

void launch_kv_prefill(const KvPrefillArgs &a, cudaStream_t stream) {
  launch_kv_store(a, stream);
  AttendArgs p{a.query, a.gate, a.output, a.caches, nullptr, a.past, a.query_heads, a.window, a.sinks, device_status_word()};
  auto run = [&](auto attend) {
    launch_programmatic(attend, dim3(a.tokens, a.query_heads), dim3(128), 0, stream, "KV attention launch", p);
  };
  a.activations_f32 ? run(kv_attend_kernel<true>) : run(kv_attend_kernel<false>);
}

} // namespace rib200
