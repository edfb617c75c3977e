// The kernel that writes a chunk's rows into a cache and the rows it sees into the workspace.
#pragma once

#include "kv_cache.hpp"

namespace rib200 {

struct KvStoreArgs {
  const void *key, *value;
  KvCaches caches;
  std::uint32_t tokens, past;
  std::uint32_t sink_blocks;  // blocks of 16 tokens [0, sink_blocks), then [window_block, ...)
  std::uint32_t window_block;
  std::uint32_t seen_sinks, seen_low;
  void *staged; // BF16 [K, V][kv head][staged_rows][256]: tokens [0, seen_sinks), then from seen_low on
  std::uint32_t staged_rows;
  unsigned int *status;
};
void launch_kv_store(const KvPrefillArgs &args, cudaStream_t stream);

} // namespace rib200
