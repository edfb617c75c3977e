// Stand-ins for the rib200_kv_* launchers and rib200_residual_rms_norm that record their arguments, shapes field by field.
// Built by tests/test_kv_host.py, which compares what arrives from the native functions with what ctypes passes.
#include "../../include/rib200.h"

#include <cstddef>
#include <cstring>
#include <vector>

namespace {
std::vector<unsigned char> g_record;

template <class T> void put(T value) {
  const auto *bytes = reinterpret_cast<const unsigned char *>(&value);
  g_record.insert(g_record.end(), bytes, bytes + sizeof(T));
}
void put(const Rib200AttentionShape *s) {
  const size_t fields[6] = {s->tokens, s->query_heads, s->kv_heads, s->head_dim, s->max_context_tokens, s->past_tokens};
  for (const size_t field : fields) {
    put(field);
  }
}
template <auto> struct Stub;
template <class... A, Rib200Status (*Declared)(A...)> struct Stub<Declared> {
  static Rib200Status call(A... arguments) {
    g_record.clear();
    (put(arguments), ...);
    return Rib200Status{RIB200_STATUS_OK, nullptr};
  }
};
} // namespace

extern "C" void *stub_address(const char *name) {
#define RIB200_STUB(entry)                                \
  if (std::strcmp(name, #entry) == 0) {                   \
    return reinterpret_cast<void *>(&Stub<&entry>::call); \
  }
  RIB200_STUB(rib200_kv_attention_prefill)
  RIB200_STUB(rib200_kv_paged_prefill)
  RIB200_STUB(rib200_kv_batched_decode)
  RIB200_STUB(rib200_kv_paged_decode)
  RIB200_STUB(rib200_residual_rms_norm)
#undef RIB200_STUB
  return nullptr;
}

extern "C" std::size_t stub_record(unsigned char *out, std::size_t capacity) { // and forgets it
  const std::size_t bytes = g_record.size() < capacity ? g_record.size() : capacity;
  std::memcpy(out, g_record.data(), bytes);
  g_record.clear();
  return bytes;
}
