// KV caches of the rib200_kv_* calls: where rows lie, the scale rule of the 8-bit kind, and the launchers' arguments.
#pragma once

#include "common.hpp"

#include <cuda_fp8.h>

#include <cstdint>

namespace rib200 {

constexpr std::uint32_t kKvHeadDim = 256;
constexpr std::uint32_t kKv8BlockTokens = RIB200_KV8_BLOCK_TOKENS;
constexpr std::uint32_t kKv8BlockBytes = RIB200_KV8_BLOCK_BYTES;
constexpr std::uint32_t kKv8CodeBytes = kKv8BlockTokens * kKvHeadDim; // the scale follows
constexpr std::uint32_t kKvPageTokens = 256;

// Bytes of one K or V plane of a head in a cache of `rows` tokens.
__host__ __device__ inline std::size_t kv_plane_bytes(bool eight_bit, std::size_t rows) {
  return eight_bit ? (rows + kKv8BlockTokens - 1) / kKv8BlockTokens * kKv8BlockBytes : rows * kKvHeadDim * 2;
}

// The caches of a call: one contiguous cache, an array of them, or pages named by tables.
struct KvCaches {
  bool eight_bit;
  std::uint32_t kv_heads;
  void *single; // or the page pool
  std::uint32_t single_rows;
  void *const *caches; // device array
  const std::uint32_t *capacities;
  const std::uint32_t *tables; // [sequence][max_blocks]
  std::uint32_t max_blocks;
  std::uint32_t pool_pages;
};

// One token of each sequence of a batch.
struct KvDecodeArgs {
  const void *query, *key, *value, *gate;
  void *output;
  KvCaches caches;
  const std::uint32_t *positions;
  std::uint32_t batch;
  std::uint32_t query_heads;
  std::uint32_t window; // 0xFFFFFFFF: the whole context
  std::uint32_t sinks;
  bool activations_f32;
  void *workspace;
};
std::size_t kv_decode_workspace_bytes();
void launch_kv_decode(const KvDecodeArgs &args, cudaStream_t stream);

// A chunk of one sequence.
struct KvPrefillArgs {
  const void *query, *key, *value, *gate;
  void *output;
  KvCaches caches; // `single`, or the pool with one table
  std::uint32_t tokens;
  std::uint32_t past;
  std::uint32_t query_heads;
  std::uint32_t window;
  std::uint32_t sinks;
  bool activations_f32;
  void *workspace; // staged rows, see kv_staged_rows
};
void launch_kv_prefill(const KvPrefillArgs &args, cudaStream_t stream);

// What a chunk's queries see of the context: tokens [0, sinks) and [low, past + tokens).
struct KvVisible {
  std::uint32_t sinks; // of the sinks, those in front of the last query's window
  std::uint32_t low;   // first token of the first query's window
};
inline KvVisible kv_visible(std::uint32_t tokens, std::uint32_t past, std::uint32_t window, std::uint32_t sinks) {
  const std::uint32_t context = past + tokens;
  const std::uint32_t low_last = context > window ? context - window : 0U;
  return KvVisible{sinks < low_last ? sinks : low_last, past + 1 > window ? past + 1 - window : 0U};
}
// Staged BF16 rows of a chunk, [K, V][kv head][row]: its sinks, then tokens [low, past + tokens).  Sinks that reach into the first
// query's window are there once: what is visible is then one run of tokens, and token t is row t.
inline std::uint32_t kv_staged_low(const KvVisible &seen) { return seen.sinks < seen.low ? seen.sinks : seen.low; } // row of `low`
inline std::size_t kv_staged_rows(const KvVisible &seen, std::size_t context) {
  return kv_staged_low(seen) + (context - seen.low);
}

#ifdef __CUDACC__
// The block scale for a largest finite magnitude of `amax`: 2^e with e in [-100, 119] least such that amax <= 448 * 2^e;
// 448 = 1.75 * 2^8 is the largest code.
__device__ __forceinline__ float kv8_scale(float amax) {
  const std::uint32_t bits = __float_as_uint(amax);
  int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFU) > 0x600000U ? 1 : 0);
  e = max(-100, min(119, e));
  return __uint_as_float(static_cast<std::uint32_t>(e + 127) << 23);
}
// 1 / scale, exact; both are normal numbers
__device__ __forceinline__ float kv8_inverse(float scale) {
  return __uint_as_float((254U << 23) - __float_as_uint(scale));
}
// a, b as two codes, rounded once to nearest even; beyond +-448 (infinities) they saturate, a not-a-number stays one
__device__ __forceinline__ std::uint32_t kv8_codes2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 kv8_values2(std::uint32_t codes) {
  const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
  return __half22float2(__half2(raw));
}
// |x| for the scale: infinities and not-a-numbers do not count
__device__ __forceinline__ float kv8_finite_magnitude(float x) {
  const float m = fabsf(x);
  return m <= 3.4028234663852886e38F ? m : 0.0F;
}

// Where a sequence's rows lie, resolved on the device.
struct KvView {
  unsigned char *base;         // its cache, or the pool
  const std::uint32_t *table;  // null: contiguous
  std::uint32_t rows;          // capacity of the cache, or of a page
  std::uint32_t pool_pages;
  std::uint32_t kv_heads;
  bool eight_bit;

  __device__ __forceinline__ std::size_t plane_bytes() const { return kv_plane_bytes(eight_bit, rows); }
  // Start of the plane of (K or V, head) that holds `token`, or null where the table names a page that is not there.
  __device__ __forceinline__ unsigned char *plane(std::uint32_t is_value, std::uint32_t head, std::uint32_t token) const {
    unsigned char *cache = base;
    if (table != nullptr) {
      const std::uint32_t page = table[token / kKvPageTokens];
      if (page >= pool_pages) {
        return nullptr;
      }
      cache += static_cast<std::size_t>(page) * (2 * kv_heads * plane_bytes());
    }
    return cache + (static_cast<std::size_t>(is_value) * kv_heads + head) * plane_bytes();
  }
  __device__ __forceinline__ std::uint32_t row_in_plane(std::uint32_t token) const {
    return table != nullptr ? token % kKvPageTokens : token;
  }
};
__device__ __forceinline__ KvView kv_view(const KvCaches &c, std::uint32_t sequence) {
  KvView v;
  v.base = static_cast<unsigned char *>(c.caches != nullptr ? c.caches[sequence] : c.single);
  v.table = c.tables != nullptr ? c.tables + static_cast<std::size_t>(sequence) * c.max_blocks : nullptr;
  v.rows = c.tables != nullptr ? kKvPageTokens : c.caches != nullptr ? c.capacities[sequence] : c.single_rows;
  v.pool_pages = c.pool_pages;
  v.kv_heads = c.kv_heads;
  v.eight_bit = c.eight_bit;
  return v;
}
// Why a sequence's token at `pos` cannot be served: status bits, kKvPadding for an entry that is to be skipped, or 0.
constexpr std::uint32_t kKvPadding = 1U << 31;
__device__ __forceinline__ std::uint32_t kv_refusal(const KvCaches &c, const KvView &view, std::uint32_t pos) {
  const std::uint32_t capacity = c.tables != nullptr ? c.max_blocks * kKvPageTokens : view.rows;
  std::uint32_t why = 0;
  // the pointers lie in device memory: the host cannot see them
  why = view.base == nullptr || reinterpret_cast<std::uintptr_t>(view.base) % 16 != 0 ? RIB200_DEVICE_POINTER_MISALIGNED : why;
  why = pos >= capacity ? RIB200_DEVICE_POSITION_OUT_OF_RANGE : why;
  return pos == RIB200_NO_POSITION ? kKvPadding : why;
}
#endif

} // namespace rib200
