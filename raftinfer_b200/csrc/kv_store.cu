// Prompt rows into a KV cache, and the rows that the prompt's attention reads into BF16.
//
// A CTA takes one block of 16 tokens of one head's K or V.  Rows of the chunk come from the inputs (FP32 or BF16), rows in
// front of it from the cache.  For an 8-bit cache the CTA finds the largest finite magnitude of the new rows, takes the block's
// scale 2^e from it (not below the one that rows in front already have), rounds value / 2^e to e4m3 and writes codes and
// scale.  Whatever the chunk's queries see is also written to the workspace as BF16, which is exact: a code has four
// significant bits and the scale is a power of two.  The attention kernel then reads nothing but BF16 tiles, so each element
// is converted once here and not once for every query tile and head there.
// Bytes: inputs and cache rows once, workspace rows once; bound by memory, or by launch latency for short chunks: 2709 tokens
// add 3.5 us to attention's 57, 512 behind 16384 7 to 102.

#include "kv_cache.hpp"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rib200 {
namespace {

struct KvStoreArgs {
  const void *key, *value;
  KvCaches caches;
  std::uint32_t tokens, past;
  std::uint32_t sink_blocks;  // blocks of 16 tokens [0, sink_blocks), then [window_block, ...)
  std::uint32_t window_block;
  std::uint32_t seen_low;
  void *staged; // BF16 [K, V][kv head][staged_rows][256]: tokens [0, seen_sinks), from row staged_low on those from seen_low on
  std::uint32_t staged_rows;
  std::uint32_t staged_low;
  unsigned int *status;
};

constexpr int kThreads = 128; // eight threads a row, which take 8 of every 64 dims
constexpr int kPieces = 4;

__device__ __forceinline__ std::uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const std::uint32_t *>(&v);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8]) {
  const std::uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000U);
  }
}
template <bool F32> __device__ __forceinline__ void load8(const void *base, std::size_t index, float (&v)[8]) {
  if constexpr (F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + index);
    const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + index + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(base) + index), v);
  }
}

// grid = (blocks of 16 tokens, KV heads, 2)
template <bool F32, bool EightBit> __global__ void __launch_bounds__(kThreads) kv_store_kernel(const KvStoreArgs p) {
  __shared__ float warp_amax[kThreads / 32];
  grid_dependency_wait();
  grid_dependents_may_launch();
  const std::uint32_t block = blockIdx.x < p.sink_blocks ? blockIdx.x : blockIdx.x - p.sink_blocks + p.window_block;
  const std::uint32_t head = blockIdx.y;
  const std::uint32_t is_value = blockIdx.z;
  const std::uint32_t context = p.past + p.tokens;
  const std::uint32_t token = block * kKv8BlockTokens + threadIdx.x / 8;
  const bool is_new = token >= p.past && token < context;
  const bool in_front = token < p.past;
  const std::uint32_t dim0 = (threadIdx.x & 7) * 8;

  const KvView view = kv_view(p.caches, 0);
  unsigned char *plane = view.plane(is_value, head, block * kKv8BlockTokens);
  if (plane == nullptr) {
    if (threadIdx.x == 0) {
      atomicOr(p.status, static_cast<unsigned int>(RIB200_DEVICE_PAGE_OUT_OF_RANGE));
    }
    return;
  }
  const std::uint32_t row = view.row_in_plane(token);
  unsigned char *record = EightBit ? plane + static_cast<std::size_t>(row / kKv8BlockTokens) * kKv8BlockBytes : plane;
  unsigned char *cells = EightBit ? record + (row % kKv8BlockTokens) * kKvHeadDim : plane + static_cast<std::size_t>(row) * kKvHeadDim * 2;

  float x[kPieces][8];
  if (is_new) {
    const std::size_t index = ((static_cast<std::size_t>(token - p.past)) * p.caches.kv_heads + head) * kKvHeadDim + dim0;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      load8<F32>(is_value != 0 ? p.value : p.key, index + 64 * j, x[j]);
    }
  }
  if constexpr (EightBit) {
    float amax = 0.0F;
    if (is_new) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          amax = fmaxf(amax, kv8_finite_magnitude(x[j][e]));
        }
      }
    }
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFU, amax, step));
    }
    if ((threadIdx.x & 31) == 0) {
      warp_amax[threadIdx.x / 32] = amax;
    }
    float *stored_scale = reinterpret_cast<float *>(record + kKv8CodeBytes);
    const bool has_front = block * kKv8BlockTokens < p.past;
    const float before = has_front ? *stored_scale : 0.0F;
    __syncthreads(); // also: everyone has read the stored scale
    amax = fmaxf(fmaxf(warp_amax[0], warp_amax[1]), fmaxf(warp_amax[2], warp_amax[3]));
    const bool has_new = (block + 1) * kKv8BlockTokens > p.past;
    float scale = before;
    if (has_new) {
      scale = fmaxf(kv8_scale(amax), before);
      if (threadIdx.x == 0) {
        *stored_scale = scale;
      }
    }
    const float inverse = kv8_inverse(scale);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      uint2 *at = reinterpret_cast<uint2 *>(cells + dim0 + 64 * j);
      uint2 codes = make_uint2(0U, 0U);
      if (in_front) {
        codes = *at;
      }
      if (in_front && scale != before) {
        const float ratio = before * inverse; // a power of two
        std::uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 a = kv8_values2(w[i] & 0xFFFFU);
          const float2 b = kv8_values2(w[i] >> 16);
          w[i] = kv8_codes2(a.x * ratio, a.y * ratio) | (kv8_codes2(b.x * ratio, b.y * ratio) << 16);
        }
        codes = make_uint2(w[0], w[1]);
        *at = codes;
      }
      if (is_new) {
        std::uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = kv8_codes2(x[j][4 * i] * inverse, x[j][4 * i + 1] * inverse) |
                 (kv8_codes2(x[j][4 * i + 2] * inverse, x[j][4 * i + 3] * inverse) << 16);
        }
        codes = make_uint2(w[0], w[1]);
        *at = codes;
      }
      const std::uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 a = kv8_values2(w[i] & 0xFFFFU);
        const float2 b = kv8_values2(w[i] >> 16);
        x[j][4 * i] = a.x * scale;
        x[j][4 * i + 1] = a.y * scale;
        x[j][4 * i + 2] = b.x * scale;
        x[j][4 * i + 3] = b.y * scale;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      uint4 *at = reinterpret_cast<uint4 *>(cells) + (dim0 + 64 * j) / 8;
      if (is_new) {
        *at = pack8(x[j]);
      } else if (in_front) {
        unpack8(*at, x[j]);
      }
    }
  }
  if (p.staged == nullptr || !(is_new || in_front)) {
    return;
  }
  __nv_bfloat16 *stage = static_cast<__nv_bfloat16 *>(p.staged) +
                         (static_cast<std::size_t>(is_value) * p.caches.kv_heads + head) * p.staged_rows * kKvHeadDim;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint4 raw = pack8(x[j]);
    if (token < p.staged_low) { // (sinks behind it lie in the window: the rows below)
      *reinterpret_cast<uint4 *>(stage + static_cast<std::size_t>(token) * kKvHeadDim + dim0 + 64 * j) = raw;
    }
    if (token >= p.seen_low) {
      *reinterpret_cast<uint4 *>(stage + static_cast<std::size_t>(token - p.seen_low + p.staged_low) * kKvHeadDim + dim0 +
                                 64 * j) = raw;
    }
  }
}

void launch_kv_store(const KvPrefillArgs &a, cudaStream_t stream) {
  KvStoreArgs p{};
  p.key = a.key;
  p.value = a.value;
  p.caches = a.caches;
  p.tokens = a.tokens;
  p.past = a.past;
  const KvVisible seen = kv_visible(a.tokens, a.past, a.window, a.sinks);
  p.seen_low = seen.low;
  p.staged = a.workspace;
  p.staged_rows = static_cast<std::uint32_t>(kv_staged_rows(seen, a.past + a.tokens));
  p.staged_low = kv_staged_low(seen);
  // every block with a visible row once: those of the sinks, then those from the first window on
  p.sink_blocks = (seen.sinks + kKv8BlockTokens - 1) / kKv8BlockTokens;
  p.window_block = seen.low / kKv8BlockTokens > p.sink_blocks ? seen.low / kKv8BlockTokens : p.sink_blocks;
  p.status = device_status_word();
  const std::uint32_t end = (a.past + a.tokens - 1) / kKv8BlockTokens + 1;
  const dim3 grid(p.sink_blocks + (end - p.window_block), a.caches.kv_heads, 2);
  auto launch = [&](auto kernel) { launch_programmatic(kernel, grid, dim3(kThreads), 0, stream, "KV store launch", p); };
  if (a.caches.eight_bit) {
    a.activations_f32 ? launch(kv_store_kernel<true, true>) : launch(kv_store_kernel<false, true>);
  } else {
    a.activations_f32 ? launch(kv_store_kernel<true, false>) : launch(kv_store_kernel<false, false>);
  }
}

} // namespace

// The rows into the cache (and into the workspace, for what attention does not read as it lies there), then attention.
void launch_kv_prefill(const KvPrefillArgs &a, cudaStream_t stream) {
  const KvVisible seen = kv_visible(a.tokens, a.past, a.window, a.sinks);
  PrefillArgs args{};
  args.query = a.query;
  args.key = a.key;
  args.value = a.value;
  args.gate = a.gate;
  args.output = a.output;
  args.kv_cache = a.caches.single;
  args.tokens = a.tokens;
  args.past_tokens = a.past;
  args.max_context_tokens = a.caches.single_rows;
  args.query_heads = a.query_heads;
  args.kv_heads = a.caches.kv_heads;
  args.activations_f32 = a.activations_f32;
  args.window = PrefillWindow{a.window, a.sinks, seen.low, seen.sinks, a.workspace,
                              static_cast<std::uint32_t>(kv_staged_rows(seen, a.past + a.tokens))};
  if (a.workspace != nullptr) {
    launch_kv_store(a, stream);
  }
  launch_prefill_attention(args, stream);
}

} // namespace rib200
