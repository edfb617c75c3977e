// Host side of the rib200_kv_* calls and of rib200_residual_rms_norm: sizes, argument checks and dispatch.
// What they narrow: head_dim 256; a prompt's context up to 2^23 tokens, a chunk of it up to 65535 * 128, 256 KV heads and 1024
// query heads; up to four query heads for a KV head in single-token calls; tensor pointers 16-byte aligned.

#include "kv_cache.hpp"
#include "residual_norm.hpp"

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace rib200 {
namespace {

constexpr std::size_t kUnbounded = 0x7FFFFFFFU;
constexpr std::uint32_t kWholeContext = 0xFFFFFFFFU;

bool eight_bit_of(std::uint8_t cache_dtype, const char *unknown) {
  require(cache_dtype <= RIB200_KV_CACHE_E4M3, unknown);
  unsupported(cache_dtype != RIB200_KV_CACHE_F32, "KV attention: caches are BF16 or E4M3");
  return cache_dtype == RIB200_KV_CACHE_E4M3;
}

std::size_t one_cache_bytes(std::size_t kv_heads, std::size_t rows, bool eight_bit) {
  const char *what = "KV cache size overflows";
  const std::size_t plane = eight_bit ? mul(ceil_div(rows, kKv8BlockTokens, what), kKv8BlockBytes, what)
                                      : mul(rows, kKvHeadDim * 2, what);
  return mul(mul(2, kv_heads, what), plane, what);
}

std::uint32_t clamp_tokens(std::size_t tokens) { return static_cast<std::uint32_t>(std::min(tokens, kUnbounded)); }
std::uint32_t window_of(std::size_t window_tokens) { return window_tokens == 0 ? kWholeContext : clamp_tokens(window_tokens); }

void aligned(const void *pointer, const char *message) {
  require(reinterpret_cast<std::uintptr_t>(pointer) % 16 == 0, message);
}

void check_activations(const void *query, const void *key, const void *value, const void *gate, const void *output,
                       int32_t activation_dtype, const void *stream) {
  require(query != nullptr && key != nullptr && value != nullptr && gate != nullptr && output != nullptr,
          "KV attention: an activation pointer is null");
  require(stream != nullptr, "KV attention: CUDA stream is null");
  require(activation_dtype >= RIB200_DTYPE_F32 && activation_dtype <= RIB200_DTYPE_BF16,
          "KV attention: unknown activation dtype");
  unsupported(activation_dtype != RIB200_DTYPE_F16, "KV attention: activations are FP32 or BF16");
  aligned(query, "KV attention: query is not 16-byte aligned");
  aligned(key, "KV attention: key is not 16-byte aligned");
  aligned(value, "KV attention: value is not 16-byte aligned");
  aligned(gate, "KV attention: gate is not 16-byte aligned");
  aligned(output, "KV attention: output is not 16-byte aligned");
}

void check_prefill_shape(const Rib200AttentionShape *shape) {
  require(shape != nullptr, "attention shape pointer is null");
  const Rib200AttentionShape &s = *shape;
  require(s.tokens > 0, "KV attention: tokens must be positive");
  require(s.query_heads > 0 && s.kv_heads > 0, "KV attention: head counts must be positive");
  require(s.query_heads % s.kv_heads == 0, "KV attention: query_heads must be a multiple of kv_heads");
  require(s.max_context_tokens > 0, "KV attention: max_context_tokens must be positive");
  require(s.past_tokens <= s.max_context_tokens && s.tokens <= s.max_context_tokens - s.past_tokens,
          "KV attention: context exceeds the cache capacity");
  unsupported(s.head_dim == kKvHeadDim, "KV attention: built for head_dim 256");
  unsupported(s.query_heads <= 1024 && s.kv_heads <= 256, "KV attention: more than 1024 query heads or 256 KV heads");
  unsupported(s.past_tokens + s.tokens <= (1U << 23), "KV attention: a prompt's context is at most 2^23 tokens");
  unsupported(s.tokens <= kPrefillMaxTokens, "KV attention: a chunk is at most 65535 * 128 tokens");
  require(s.max_context_tokens <= kUnbounded, "KV attention: max_context_tokens exceeds 2^31");
}

std::size_t prefill_workspace(const Rib200AttentionShape &s, std::size_t window_tokens, std::size_t sink_tokens,
                              bool eight_bit, bool paged) {
  if (!eight_bit && !paged) {
    return 0;
  }
  const KvVisible seen = kv_visible(static_cast<std::uint32_t>(s.tokens), static_cast<std::uint32_t>(s.past_tokens),
                                    window_of(window_tokens), clamp_tokens(sink_tokens));
  const char *what = "KV attention: workspace size overflows";
  return mul(mul(2 * s.kv_heads, kv_staged_rows(seen, s.past_tokens + s.tokens), what), kKvHeadDim * 2, what);
}

void prefill(const void *query, const void *key, const void *value, const void *gate, void *output,
             const KvCaches &caches, void *workspace, std::size_t workspace_bytes, const Rib200AttentionShape &s,
             std::size_t window_tokens, std::size_t sink_tokens, int32_t activation_dtype, void *stream) {
  const std::size_t need =
      prefill_workspace(s, window_tokens, sink_tokens, caches.eight_bit, caches.tables != nullptr);
  if (need != 0) {
    require(workspace != nullptr, "KV attention: workspace is null");
    require(workspace_bytes >= need, "KV attention: workspace is too small");
    aligned(workspace, "KV attention: workspace is not 16-byte aligned");
  }
  KvPrefillArgs args{};
  args.query = query;
  args.key = key;
  args.value = value;
  args.gate = gate;
  args.output = output;
  args.caches = caches;
  args.tokens = static_cast<std::uint32_t>(s.tokens);
  args.past = static_cast<std::uint32_t>(s.past_tokens);
  args.query_heads = static_cast<std::uint32_t>(s.query_heads);
  args.window = window_of(window_tokens);
  args.sinks = clamp_tokens(sink_tokens);
  args.activations_f32 = activation_dtype == RIB200_DTYPE_F32;
  args.workspace = need != 0 ? workspace : nullptr; // a caller may hand one over where none is used
  launch_kv_prefill(args, static_cast<cudaStream_t>(stream));
}

void decode(const void *query, const void *key, const void *value, const void *gate, void *output, const KvCaches &caches,
            const std::uint32_t *positions, std::size_t batch, std::size_t query_heads, std::size_t window_tokens,
            std::size_t sink_tokens, int32_t activation_dtype, void *workspace, std::size_t workspace_bytes,
            void *stream) {
  require(positions != nullptr, "KV decode: positions pointer is null");
  require(batch > 0 && batch <= 65535, "KV decode: batch must be in 1..65535");
  require(query_heads > 0 && caches.kv_heads > 0, "KV decode: head counts must be positive");
  require(query_heads % caches.kv_heads == 0, "KV decode: query_heads must be a multiple of kv_heads");
  unsupported(query_heads / caches.kv_heads <= 4 && caches.kv_heads <= 256,
              "KV decode: built for 1 to 4 query heads for a KV head, 256 KV heads at most");
  require(workspace != nullptr, "KV decode: workspace is null");
  require(workspace_bytes >= kv_decode_workspace_bytes(), "KV decode: workspace is too small");
  aligned(workspace, "KV decode: workspace is not 16-byte aligned");
  KvDecodeArgs args{};
  args.query = query;
  args.key = key;
  args.value = value;
  args.gate = gate;
  args.output = output;
  args.caches = caches;
  args.positions = positions;
  args.batch = static_cast<std::uint32_t>(batch);
  args.query_heads = static_cast<std::uint32_t>(query_heads);
  args.window = window_of(window_tokens);
  args.sinks = clamp_tokens(sink_tokens);
  args.activations_f32 = activation_dtype == RIB200_DTYPE_F32;
  args.workspace = workspace;
  launch_kv_decode(args, static_cast<cudaStream_t>(stream));
}

KvCaches pool(void *page_pool, std::size_t pool_pages, const std::uint32_t *tables, std::size_t max_blocks,
              std::size_t kv_heads, bool eight_bit) {
  require(page_pool != nullptr && tables != nullptr, "KV attention: the page pool or the block table pointer is null");
  require(pool_pages > 0 && pool_pages <= kUnbounded, "KV attention: pool_pages out of range");
  require(max_blocks > 0 && max_blocks <= kUnbounded / kKvPageTokens, "KV attention: blocks per sequence out of range");
  aligned(page_pool, "KV attention: page pool is not 16-byte aligned");
  KvCaches c{};
  c.eight_bit = eight_bit;
  c.kv_heads = static_cast<std::uint32_t>(std::min<std::size_t>(kv_heads, kUnbounded));
  c.single = page_pool;
  c.tables = tables;
  c.max_blocks = static_cast<std::uint32_t>(max_blocks);
  c.pool_pages = static_cast<std::uint32_t>(pool_pages);
  return c;
}

} // namespace
} // namespace rib200

using namespace rib200;

extern "C" {

Rib200Status rib200_kv_cache_bytes(size_t kv_heads, size_t max_context_tokens, uint8_t cache_dtype, size_t *bytes) {
  return guarded([&] {
    require(bytes != nullptr, "size output pointer is null");
    require(kv_heads > 0 && max_context_tokens > 0, "KV cache: heads and tokens must be positive");
    *bytes = one_cache_bytes(kv_heads, max_context_tokens, eight_bit_of(cache_dtype, "unknown KV cache dtype"));
  });
}

Rib200Status rib200_kv_prefill_workspace_bytes(const Rib200AttentionShape *shape, size_t window_tokens,
                                               size_t sink_tokens, uint8_t cache_dtype, int32_t paged, size_t *bytes) {
  return guarded([&] {
    require(bytes != nullptr, "size output pointer is null");
    check_prefill_shape(shape);
    *bytes = prefill_workspace(*shape, window_tokens, sink_tokens, eight_bit_of(cache_dtype, "unknown KV cache dtype"),
                               paged != 0);
  });
}

Rib200Status rib200_kv_decode_workspace_bytes(size_t *bytes) {
  return guarded([&] {
    require(bytes != nullptr, "size output pointer is null");
    *bytes = kv_decode_workspace_bytes();
  });
}

Rib200Status rib200_kv_attention_prefill(const void *query, const void *key, const void *value, const void *gate,
                                         void *output, void *kv_cache, size_t kv_cache_bytes, void *workspace,
                                         size_t workspace_bytes, const Rib200AttentionShape *shape,
                                         size_t window_tokens, size_t sink_tokens, int32_t activation_dtype,
                                         uint8_t cache_dtype, void *stream) {
  return guarded([&] {
    check_activations(query, key, value, gate, output, activation_dtype, stream);
    check_prefill_shape(shape);
    const bool eight_bit = eight_bit_of(cache_dtype, "unknown KV cache dtype");
    require(kv_cache != nullptr, "KV attention: KV cache pointer is null");
    aligned(kv_cache, "KV attention: KV cache is not 16-byte aligned");
    require(kv_cache_bytes >= one_cache_bytes(shape->kv_heads, shape->max_context_tokens, eight_bit),
            "KV attention: KV cache is too small");
    KvCaches c{};
    c.eight_bit = eight_bit;
    c.kv_heads = static_cast<std::uint32_t>(shape->kv_heads);
    c.single = kv_cache;
    c.single_rows = static_cast<std::uint32_t>(shape->max_context_tokens);
    prefill(query, key, value, gate, output, c, workspace, workspace_bytes, *shape, window_tokens, sink_tokens,
            activation_dtype, stream);
  });
}

Rib200Status rib200_kv_paged_prefill(const void *query, const void *key, const void *value, const void *gate, void *output,
                                     void *page_pool, size_t pool_pages, const uint32_t *block_table, size_t max_blocks,
                                     void *workspace, size_t workspace_bytes, const Rib200AttentionShape *shape,
                                     size_t window_tokens, size_t sink_tokens, int32_t activation_dtype,
                                     uint8_t cache_dtype, void *stream) {
  return guarded([&] {
    check_activations(query, key, value, gate, output, activation_dtype, stream);
    check_prefill_shape(shape);
    const bool eight_bit = eight_bit_of(cache_dtype, "unknown KV cache dtype");
    const KvCaches c = pool(page_pool, pool_pages, block_table, max_blocks, shape->kv_heads, eight_bit);
    require(shape->max_context_tokens == max_blocks * kKvPageTokens,
            "KV attention: max_context_tokens must be 256 * max_blocks");
    prefill(query, key, value, gate, output, c, workspace, workspace_bytes, *shape, window_tokens, sink_tokens,
            activation_dtype, stream);
  });
}

Rib200Status rib200_kv_batched_decode(const void *query, const void *key, const void *value, const void *gate,
                                      void *output, void *const *kv_caches, const uint32_t *max_context_tokens,
                                      const uint32_t *positions, size_t batch, size_t query_heads, size_t kv_heads,
                                      size_t window_tokens, size_t sink_tokens, int32_t activation_dtype,
                                      uint8_t cache_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  return guarded([&] {
    check_activations(query, key, value, gate, output, activation_dtype, stream);
    require(kv_caches != nullptr && max_context_tokens != nullptr, "KV decode: the cache or capacity array is null");
    KvCaches c{};
    c.eight_bit = eight_bit_of(cache_dtype, "unknown KV cache dtype");
    c.kv_heads = static_cast<std::uint32_t>(std::min<std::size_t>(kv_heads, kUnbounded));
    c.caches = kv_caches;
    c.capacities = max_context_tokens;
    decode(query, key, value, gate, output, c, positions, batch, query_heads, window_tokens, sink_tokens,
           activation_dtype, workspace, workspace_bytes, stream);
  });
}

Rib200Status rib200_kv_paged_decode(const void *query, const void *key, const void *value, const void *gate, void *output,
                                    void *page_pool, size_t pool_pages, const uint32_t *block_tables,
                                    size_t max_blocks_per_sequence, const uint32_t *positions, size_t batch,
                                    size_t query_heads, size_t kv_heads, size_t window_tokens, size_t sink_tokens,
                                    int32_t activation_dtype, uint8_t cache_dtype, void *workspace,
                                    size_t workspace_bytes, void *stream) {
  return guarded([&] {
    check_activations(query, key, value, gate, output, activation_dtype, stream);
    const KvCaches c = pool(page_pool, pool_pages, block_tables, max_blocks_per_sequence, kv_heads,
                            eight_bit_of(cache_dtype, "unknown KV cache dtype"));
    decode(query, key, value, gate, output, c, positions, batch, query_heads, window_tokens, sink_tokens,
           activation_dtype, workspace, workspace_bytes, stream);
  });
}

Rib200Status rib200_residual_rms_norm(const void *input, const void *residual, const void *weight, void *output,
                                      float *scales, void *residual_out, size_t rows, size_t columns,
                                      size_t group_columns, float epsilon, int32_t dtype, int32_t weight_dtype,
                                      int32_t output_dtype, void *stream) {
  return guarded([&] {
    require(input != nullptr && weight != nullptr && output != nullptr, "RMS norm: a tensor pointer is null");
    require(stream != nullptr, "RMS norm: CUDA stream is null");
    require(rows > 0 && columns > 0, "RMS norm: rows and columns must be positive");
    require(std::isfinite(epsilon) && epsilon >= 0.0F, "RMS norm: epsilon must be finite and non-negative");
    require(dtype >= RIB200_DTYPE_F32 && dtype <= RIB200_DTYPE_BF16, "RMS norm: unknown dtype");
    require(weight_dtype >= RIB200_DTYPE_F32 && weight_dtype <= RIB200_DTYPE_BF16, "RMS norm: unknown weight dtype");
    unsupported(weight_dtype != RIB200_DTYPE_F16, "RMS norm: weights are FP32 or BF16");
    require(output_dtype >= RIB200_DTYPE_F32 && output_dtype <= RIB200_DTYPE_E4M3, "RMS norm: unknown output dtype");
    const bool eight_bit = output_dtype == RIB200_DTYPE_E4M3;
    unsupported(eight_bit || output_dtype == dtype, "RMS norm: output is of the input's dtype or E4M3");
    unsupported(columns % 8 == 0 && columns <= kResidualNormMaxColumns,
                "RMS norm: columns must be a multiple of 8 up to 16384");
    require(rows <= kUnbounded, "RMS norm: too many rows");
    if (eight_bit) {
      require(scales != nullptr, "RMS norm: scales pointer is null");
      unsupported(group_columns == 0 || group_columns == 32 || group_columns == 128,
                  "RMS norm: scales are for a row or for groups of 32 or 128 columns");
      require(group_columns == 0 || columns % group_columns == 0, "RMS norm: columns must be a multiple of group_columns");
      require(reinterpret_cast<std::uintptr_t>(scales) % 4 == 0, "RMS norm: scales are not 4-byte aligned");
    } else {
      require(scales == nullptr && group_columns == 0, "RMS norm: scales belong to an 8-bit output");
    }
    aligned(input, "RMS norm: input is not 16-byte aligned");
    aligned(residual, "RMS norm: residual is not 16-byte aligned");
    aligned(weight, "RMS norm: weight is not 16-byte aligned");
    aligned(output, "RMS norm: output is not 16-byte aligned");
    aligned(residual_out, "RMS norm: residual_out is not 16-byte aligned");
    ResidualNormArgs args{};
    args.input = input;
    args.residual = residual;
    args.weight = weight;
    args.output = output;
    args.scales = scales;
    args.residual_out = residual_out;
    args.rows = static_cast<std::uint32_t>(rows);
    args.columns = static_cast<std::uint32_t>(columns);
    args.group_columns = static_cast<std::uint32_t>(group_columns);
    args.epsilon = epsilon;
    args.dtype = dtype;
    args.weight_dtype = weight_dtype;
    args.eight_bit = eight_bit;
    launch_residual_norm(args, static_cast<cudaStream_t>(stream));
  });
}

} // extern "C"
