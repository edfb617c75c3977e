// Single-token attention over BF16 and 8-bit KV caches, whole or windowed, contiguous or paged.
//
//   out_h = sum_j w_j v_j / sum_j w_j * sigmoid(gate_h),  w_j = exp(q_h . k_j / 16 - max),  over the visible tokens j
//
// What bounds it: the visible rows are read once (8 bit: 257 bytes a row of K or V and head, BF16: 512) and every byte meets four
// flops, so it is a stream from HBM.  All query heads of a KV head are served by the CTA that reads its rows.
//
// Split.  The unit of work is a step, 16 tokens of one KV head.  The rows (sequence, KV head) of a batch are ragged and their
// lengths are known on the device alone, so every CTA finds its share from the positions: with many rows the steps of all
// rows, laid end to end, are cut into one equal piece per resident CTA, which may begin and end inside a row; with few rows
// (at most an eighth of the CTAs) each row is cut into pieces of its own, so that no CTA has two.  (8-bit sequences of 2 K to
// 8 K tokens, four rows each, us by rows and end to end: 2 sequences 13.8 and 20.6, 9 26.0 and 28.0, 12 34.4 and 32.6, 24 66.6
// and 48.8, 36 117 and 66.4; the rule's 36 rows of 296 CTAs lie between 9 and 12.)  What a CTA
// knows of a row that others share goes to the workspace as (maximum, sum, normalised values); a second kernel puts the
// parts of a row together.  A row that one CTA has to itself is written directly.
//
// Inside a CTA the warps take the steps of its piece in turn, each with a private ring of shared-memory slots filled by bulk
// copies two or three slots ahead; they meet once at the end of a row.
//
// Measured in replayed graphs: 8 bit, 131000 tokens 50.6 us (5.3 TB/s), 64 sequences of 1 K to 32 K 343 us (6.5 TB/s, the copy
// rate; 380 over two seconds, when the power cap has brought the SM clock to 1.68 GHz, where BF16 rows take 685),
// BF16 behind a window of 4096 168 us (6.2 TB/s), 777 tokens 8.4 us.
//
// Arithmetic: mma.sync m16n8k16, tokens (for values: dims) as the 16 rows, and as the 8 columns four query heads in two parts
// each, the value rounded to 16 bits and what is left of it, so that queries and weights count with 2^-16 of a value or
// better (FP32 activations: 2^-22 and better).  (A matrix instruction with 64 rows and more would be filled by four heads
// to a sixteenth.)  BF16 rows go into it as they are.  8-bit codes become FP16 in registers, which is exact; queries are
// scaled by a power of two to FP16's range, the block's K scale multiplies the logits, and its V scale the weights.  What is
// held of a weight is relative to the largest product of a weight and its block's V scale so far: two parts have 22 bits down
// to 2^-18 of that, and what is 2^-40 of it vanishes, however the blocks' scales compare.  Maxima are rounded up to
// integers and scales are powers of two, so nothing is rounded by moving from one to the other.  Logits, maxima, sums and
// outputs are FP32.
//
// The new token's row belongs to the last step of its row: the warp that has that step rounds the row, writes it to the cache
// and into its slot, and rounds the block's older rows again if the block's scale grew.

#include "kv_cache.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

namespace rib200 {
namespace {

constexpr std::uint32_t kGroup = 4;      // query heads of a KV head, at most
constexpr std::uint32_t kStep = 16;      // tokens
constexpr std::uint32_t kMaxCtas = 296;  // of the first kernel, which sizes the workspace
constexpr std::uint32_t kPartFloats = kGroup * (kKvHeadDim + 2); // values, then maxima, then sums
constexpr long long kWaitLimitCycles = 1LL << 28;
constexpr float kLog2e = 1.4426950408889634F;
constexpr float kLowest = -3.0e38F;
constexpr float kWeightUnit = 32768.0F;
constexpr std::uint32_t kNoSlot = 0xFFFFFFFFU;

// Slots.  BF16: row pairs (1 KiB, one copy) at a pitch of 1040 bytes; the row index m of the matrix instruction stands for
// token 2 (m % 8) + m / 8, so that the eight rows of an ldmatrix lie in eight different bank groups.  8 bit: groups of four
// rows (1 KiB, one copy; the block's scale comes with the last) at a pitch of 1056 bytes, read with 16-byte loads in which
// eight lanes meet eight different bank groups, see below; K and V of a step share a slot, which halves what a step spends on
// addresses, waits and fences.  (BF16 rows of one and a half steps are as much as fits.)
template <bool EightBit> struct Slot {
  static constexpr std::uint32_t kPitch = EightBit ? 1056 : 1040;
  static constexpr std::uint32_t kValues = EightBit ? 4224 : 0; // where the V rows begin
  static constexpr std::uint32_t kBytes = EightBit ? 2 * 4224 : 8 * 1040;
  static __device__ __forceinline__ std::uint32_t row(std::uint32_t token) {
    return EightBit ? (token >> 2) * kPitch + (token & 3U) * 256U : (token >> 1) * kPitch + (token & 1U) * 512U;
  }
};
constexpr std::uint32_t kSlotScale = 3 * 1056 + 1024; // of an 8-bit slot
constexpr std::uint32_t kMergePitch = kKvHeadDim + 8;

template <bool EightBit> struct Shape {
  static constexpr int kWarps = 4;
  static constexpr int kSlots = 3;
  static constexpr int kHalves = EightBit ? 1 : 2; // slots of a step
  static constexpr int kCtasPerSm = 2;
  static constexpr std::uint32_t kRingBytes = kWarps * kSlots * Slot<EightBit>::kBytes;
  static constexpr std::uint32_t kSmemBytes = kRingBytes + kWarps * kSlots * 8;
  static_assert(kWarps * kGroup * (kMergePitch + 2) * 4 <= kRingBytes, "the merge area lies in the ring");
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory");
};

struct DecodeParams {
  KvDecodeArgs a;
  float *parts; // [2 * kMaxCtas][kPartFloats]
  unsigned int *status;
  std::uint32_t group;
  std::uint32_t ctas;      // of the first kernel
  std::uint32_t min_steps; // of a piece
  std::uint32_t by_rows;   // rows are cut by themselves
};

// ---- schedule: the same arithmetic in both kernels, by every warp for itself (no barrier, no shared memory) ----
struct Row { // what one sequence's query sees
  std::uint32_t pos, low, sinks; // tokens [0, sinks) and [low, pos]
  std::uint32_t sink_steps, window_step; // steps [0, sink_steps), then from window_step on
  std::uint32_t steps;
  KvView view;
};

__device__ __forceinline__ Row row_of(const KvDecodeArgs &a, std::uint32_t sequence, std::uint32_t &why) {
  Row r;
  r.pos = a.positions[sequence];
  r.view = kv_view(a.caches, sequence);
  why = kv_refusal(a.caches, r.view, r.pos);
  r.low = r.pos + 1 > a.window ? r.pos + 1 - a.window : 0U;
  r.sinks = min(a.sinks, r.low);
  r.window_step = r.low / kStep;
  r.sink_steps = min((r.sinks + kStep - 1) / kStep, r.window_step);
  r.steps = why == 0 ? r.sink_steps + (r.pos / kStep - r.window_step + 1) : 0U;
  return r;
}

using Count = unsigned long long;

// exclusive prefix over the lanes, and the total
__device__ __forceinline__ Count scan(Count v, Count &total) {
  Count inclusive = v;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const Count below = __shfl_up_sync(0xFFFFFFFFU, inclusive, step);
    inclusive += threadIdx.x % 32 >= static_cast<std::uint32_t>(step) ? below : 0;
  }
  total = __shfl_sync(0xFFFFFFFFU, inclusive, 31);
  return inclusive - v;
}

struct Schedule {
  std::uint32_t target; // steps of a piece where rows are cut by themselves, else 0
  Count units;          // pieces or, laid end to end, steps
  std::uint32_t pieces; // CTAs with work
  Count each;           // units / pieces, and the remainder
  std::uint32_t more;
  // the lane's run of neighbouring sequences, the units in front of it, and the steps of its sequence if it has only one
  std::uint32_t first, last, share, only;
  Count before;

  // first unit of piece i
  __device__ __forceinline__ Count bound(std::uint32_t i) const { return each * i + min(i, more); }
  // units of one of the lane's sequences, for each head
  __device__ __forceinline__ std::uint32_t units_of(const DecodeParams &p, std::uint32_t sequence) const {
    std::uint32_t steps = only;
    if (share > 1) {
      std::uint32_t why;
      steps = row_of(p.a, sequence, why).steps;
    }
    return target != 0 ? (steps + target - 1) / target : steps;
  }
};

__device__ __forceinline__ Schedule make_schedule(const DecodeParams &p, bool report) {
  const std::uint32_t lane = threadIdx.x % 32;
  const std::uint32_t heads = p.a.caches.kv_heads;
  Schedule s;
  s.share = (p.a.batch + 31) / 32;
  s.first = min(p.a.batch, lane * s.share);
  s.last = min(p.a.batch, s.first + s.share);
  s.target = 0;
  s.only = 0;
  Count mine = 0;
  std::uint32_t why_all = 0;
#pragma unroll 4
  for (std::uint32_t i = s.first; i < s.last; ++i) {
    std::uint32_t why;
    s.only = row_of(p.a, i, why).steps;
    mine += s.only;
    why_all |= why;
  }
  why_all &= ~kKvPadding;
  if (report && why_all != 0) {
    atomicOr(p.status, why_all);
  }
  Count total;
  s.before = scan(mine, total) * heads;
  s.units = total * heads;
  if (p.by_rows != 0) {
    const std::uint32_t room = p.ctas - p.a.batch * heads;
    s.target = static_cast<std::uint32_t>(max(static_cast<Count>(p.min_steps), (s.units + room - 1) / room));
    mine = 0;
    for (std::uint32_t i = s.first; i < s.last; ++i) {
      mine += s.units_of(p, i);
    }
    s.before = scan(mine, total) * heads;
    s.units = total * heads;
    s.pieces = static_cast<std::uint32_t>(s.units);
  } else {
    s.pieces = static_cast<std::uint32_t>(min(static_cast<Count>(p.ctas), (s.units + p.min_steps - 1) / p.min_steps));
  }
  s.each = s.pieces != 0 ? s.units / s.pieces : 0;
  s.more = static_cast<std::uint32_t>(s.units - s.each * s.pieces);
  return s;
}

struct Place {
  std::uint32_t sequence, head, index; // the index-th unit of a row
};
// Where a unit lies.
__device__ __forceinline__ Place place_of(const Schedule &s, const DecodeParams &p, Count unit) {
  Place at{};
  bool found = false;
  Count before = s.before;
  for (std::uint32_t i = s.first; i < s.last && unit >= before && !found; ++i) {
    const std::uint32_t each = s.units_of(p, i);
    const Count end = before + static_cast<Count>(each) * p.a.caches.kv_heads;
    if (unit < end) {
      at.sequence = i;
      at.head = static_cast<std::uint32_t>((unit - before) / each);
      // a row has less than 2^31 units, so that wrapping leaves this right
      at.index = static_cast<std::uint32_t>(unit - before) - at.head * each;
      found = true;
    }
    before = end;
  }
  const std::uint32_t who = __ballot_sync(0xFFFFFFFFU, found);
  const int from = who != 0 ? __ffs(who) - 1 : 0;
  at.sequence = __shfl_sync(0xFFFFFFFFU, at.sequence, from);
  at.head = __shfl_sync(0xFFFFFFFFU, at.head, from);
  at.index = __shfl_sync(0xFFFFFFFFU, at.index, from);
  return at;
}
// Units of a row and the first of them.
__device__ __forceinline__ std::uint32_t units_of_row(const Schedule &s, const DecodeParams &p, std::uint32_t sequence,
                                                      std::uint32_t head, Count &first) {
  Count at = s.before;
  std::uint32_t each = 0;
  for (std::uint32_t i = s.first; i < s.last && i <= sequence; ++i) {
    each = s.units_of(p, i);
    at += i < sequence ? static_cast<Count>(each) * p.a.caches.kv_heads : static_cast<Count>(each) * head;
  }
  const int from = static_cast<int>(sequence / s.share);
  first = __shfl_sync(0xFFFFFFFFU, at, from);
  return __shfl_sync(0xFFFFFFFFU, each, from);
}

// ---- small pieces ----
__device__ __forceinline__ std::uint32_t smem_address(const void *p) {
  return static_cast<std::uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbarrier_init(std::uint32_t bar, std::uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbarrier_expect_tx(std::uint32_t bar, std::uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbarrier_try_wait(std::uint32_t bar, std::uint32_t parity) {
  std::uint32_t done;
  asm volatile("{\n"
               ".reg .pred p;\n"
               "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               "selp.u32 %0, 1, 0, p;\n"
               "}\n"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done != 0;
}
// a call reads each row once: they leave L2 first
__device__ __forceinline__ std::uint64_t evict_first_policy() {
  std::uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void bulk_copy_g2s(std::uint32_t dst, const void *src, std::uint32_t bytes, std::uint32_t bar,
                                              std::uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void ldmatrix_x4(std::uint32_t addr, std::uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(std::uint32_t addr, std::uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void lds128(std::uint32_t addr, std::uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint2 lds64(std::uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(std::uint32_t addr, uint2 v) {
  asm volatile("st.shared.v2.u32 [%0], {%1,%2};\n" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void sts128(std::uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float lds_float(std::uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts_float(std::uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(addr), "f"(v) : "memory");
}

template <bool Half>
__device__ __forceinline__ void mma(float (&c)[4], std::uint32_t a0, std::uint32_t a1, std::uint32_t a2, std::uint32_t a3,
                                    std::uint32_t b0, std::uint32_t b1) {
  if constexpr (Half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// the 16-bit parts of two values: the rounded ones (part 0) or what is left of them (part 1)
template <bool Half> __device__ __forceinline__ std::uint32_t split2(float x, float y, int part) {
  if constexpr (Half) {
    __half2 hi = __floats2half2_rn(x, y);
    if (part != 0) {
      const float2 back = __half22float2(hi);
      hi = __floats2half2_rn(x - back.x, y - back.y);
    }
    return *reinterpret_cast<const std::uint32_t *>(&hi);
  } else {
    __nv_bfloat162 hi = __floats2bfloat162_rn(x, y);
    if (part != 0) {
      const float2 back = __bfloat1622float2(hi);
      hi = __floats2bfloat162_rn(x - back.x, y - back.y);
    }
    return *reinterpret_cast<const std::uint32_t *>(&hi);
  }
}

// the two codes in the low or high half of a word as FP16, exactly
__device__ __forceinline__ std::uint32_t half2_of_low(std::uint32_t w) {
  std::uint32_t out;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(out) : "r"(w));
  return out;
}
__device__ __forceinline__ std::uint32_t half2_of_high(std::uint32_t w) {
  std::uint32_t out;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(out) : "r"(w));
  return out;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

template <bool F32> __device__ __forceinline__ void load8(const void *base, std::size_t index, float (&v)[8]) {
  if constexpr (F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + index);
    const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + index + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 raw = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(base) + index);
    const std::uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000U);
    }
  }
}
// x times a share or weight.  Over BF16 rows an infinity stays one where FP32 has only a zero left of a share that is more; 8-bit
// rows hold none.
template <bool EightBit> __device__ __forceinline__ float share_of(float x, float by) {
  return EightBit || fabsf(x) <= 3.4028234663852886e38F ? x * by : x;
}
template <bool EightBit> __device__ __forceinline__ float4 share_of(float4 v, float by) {
  return make_float4(share_of<EightBit>(v.x, by), share_of<EightBit>(v.y, by), share_of<EightBit>(v.z, by),
                     share_of<EightBit>(v.w, by));
}
template <bool F32> __device__ __forceinline__ float4 load4(const void *base, std::size_t index) {
  if constexpr (F32) {
    return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + index);
  } else {
    const uint2 raw = *reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(base) + index);
    return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xFFFF0000U), __uint_as_float(raw.y << 16),
                       __uint_as_float(raw.y & 0xFFFF0000U));
  }
}
template <bool F32> __device__ __forceinline__ void store4(void *base, std::size_t index, float4 v) {
  if constexpr (F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + index) = v;
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(base) + index) =
        make_uint2(*reinterpret_cast<const std::uint32_t *>(&a), *reinterpret_cast<const std::uint32_t *>(&b));
  }
}
__device__ __forceinline__ float4 gated(float4 v, float4 gate) {
  return make_float4(v.x / (1.0F + expf(-gate.x)), v.y / (1.0F + expf(-gate.y)), v.z / (1.0F + expf(-gate.z)),
                     v.w / (1.0F + expf(-gate.w)));
}

// Parts 0 and 1, 2 and 3 of two values in BF16: column parts `part` and `part` + 2.
__device__ __forceinline__ void split4(float x, float y, int part, std::uint32_t &first, std::uint32_t &second) {
  std::uint32_t parts[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 rounded = __floats2bfloat162_rn(x, y);
    const float2 back = __bfloat1622float2(rounded);
    parts[i] = *reinterpret_cast<const std::uint32_t *>(&rounded);
    x -= back.x;
    y -= back.y;
  }
  first = part != 0 ? parts[1] : parts[0];
  second = part != 0 ? parts[3] : parts[2];
}

// A lane's 16 dims of a step's matrix operand, as the fragments want them.
//   BF16: fragment ks, half: dims 16 ks + 8 half + 2 t, +1.   8 bit: fragment 4 s + w, half: dims 64 s + 16 t + 4 w + 2 half, +1.
// FP32 queries over BF16 rows have four parts of eight bits: columns take parts 0 and 1, and in a second product into the same
// sums parts 2 and 3 (two parts are off by 2^-17, ten times the error of FP32 sums).
template <bool F32, bool EightBit> struct Query {
  static constexpr bool kFourParts = F32 && !EightBit;
  std::uint32_t fragment[32];
  std::uint32_t rest[kFourParts ? 32 : 1];
  float scale; // of head t: logit (base 2) = product * scale (* the block's K scale)

  // column g of the lane (g, t): head g / 2, part g & 1
  __device__ __forceinline__ void load(const void *query, std::size_t base, std::uint32_t group, int g, int t) {
    const std::uint32_t head = static_cast<std::uint32_t>(g >> 1);
    const bool live = head < group;
    const std::size_t row = base + head * kKvHeadDim;
    const int part = g & 1;
    if constexpr (!EightBit) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const std::size_t index = row + 8 * i + 2 * t;
        float2 x = make_float2(0.0F, 0.0F);
        if (live) {
          if constexpr (F32) {
            x = *reinterpret_cast<const float2 *>(static_cast<const float *>(query) + index);
          } else {
            const std::uint32_t raw = *reinterpret_cast<const std::uint32_t *>(static_cast<const __nv_bfloat16 *>(query) + index);
            x = make_float2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xFFFF0000U));
          }
        }
        if constexpr (kFourParts) {
          split4(x.x, x.y, part, fragment[i], rest[i]);
        } else {
          fragment[i] = split2<false>(x.x, x.y, part);
        }
      }
      scale = 0.0625F * kLog2e;
    } else {
      float x[64];
      float amax = 0.0F;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[8] = {};
          if (live) {
            load8<F32>(query, row + 64 * s + 16 * t + 8 * half, v);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[16 * s + 8 * half + e] = v[e];
            amax = fmaxf(amax, kv8_finite_magnitude(v[e]));
          }
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFU, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFU, amax, 2));
      // largest magnitude to 2^7 .. 2^8: BF16 queries are then exact in FP16 down to 2^-24 of it, FP32 ones to 2^-22 in two parts
      const int e = max(-100, min(120, static_cast<int>(__float_as_uint(amax) >> 23) - 127));
      const float up = __uint_as_float(static_cast<std::uint32_t>(127 + 7 - e) << 23);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        fragment[i] = split2<true>(x[2 * i] * up, x[2 * i + 1] * up, part);
      }
      // of head t: held by the lanes of column 2 t
      const int e_t = __shfl_sync(0xFFFFFFFFU, e, 8 * t);
      scale = __uint_as_float(static_cast<std::uint32_t>(127 - 7 + e_t) << 23) * (0.0625F * kLog2e);
    }
  }
};

// A lane's eight dims of the new token's row, fetched when its piece begins.
template <bool F32> struct NewRow {
  uint4 raw[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *base, std::size_t index) {
    const uint4 *at = reinterpret_cast<const uint4 *>(static_cast<const unsigned char *>(base) + index * (F32 ? 4 : 2));
    raw[0] = at[0];
    if constexpr (F32) {
      raw[1] = at[1];
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const std::uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F32) {
        x[i] = __uint_as_float(w[i]);
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000U);
      }
    }
    if constexpr (F32) {
      x[4] = __uint_as_float(raw[1].x);
      x[5] = __uint_as_float(raw[1].y);
      x[6] = __uint_as_float(raw[1].z);
      x[7] = __uint_as_float(raw[1].w);
    }
  }
};

// The new token's row into the cache and into its slot, which holds the rows of its block: row r of the block whose first row
// is row r0 of the plane.  Not inlined: one step in many comes here.
template <bool EightBit>
__device__ __noinline__ void append_row(std::uint32_t slot, unsigned char *plane, std::uint32_t r0, std::uint32_t r, float x0,
                                        float x1, float x2, float x3, float x4, float x5, float x6, float x7) {
  using L = Slot<EightBit>;
  const std::uint32_t lane = threadIdx.x % 32;
  const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
  if constexpr (EightBit) {
    unsigned char *record = plane + static_cast<std::size_t>(r0 / kStep) * kKv8BlockBytes;
    float amax = 0.0F;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      amax = fmaxf(amax, kv8_finite_magnitude(x[e]));
    }
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFU, amax, step));
    }
    const float before = r > 0 ? lds_float(slot + kSlotScale) : 0.0F;
    const float scale = fmaxf(kv8_scale(amax), before);
    const float inverse = kv8_inverse(scale);
    __syncwarp(); // everyone has the scale in front
    if (lane == 0) {
      sts_float(slot + kSlotScale, scale);
      *reinterpret_cast<float *>(record + kKv8CodeBytes) = scale;
    }
    if (scale != before) {
      const float ratio = before * inverse;
#pragma unroll 1
      for (std::uint32_t i = 0; i < r; ++i) {
        const uint2 old = lds64(slot + L::row(i) + 8 * lane);
        std::uint32_t w[2] = {old.x, old.y};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 a = kv8_values2(w[k] & 0xFFFFU), b = kv8_values2(w[k] >> 16);
          w[k] = kv8_codes2(a.x * ratio, a.y * ratio) | (kv8_codes2(b.x * ratio, b.y * ratio) << 16);
        }
        sts64(slot + L::row(i) + 8 * lane, make_uint2(w[0], w[1]));
        *reinterpret_cast<uint2 *>(record + i * kKvHeadDim + 8 * lane) = make_uint2(w[0], w[1]);
      }
    }
    std::uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      w[k] = kv8_codes2(x[4 * k] * inverse, x[4 * k + 1] * inverse) |
             (kv8_codes2(x[4 * k + 2] * inverse, x[4 * k + 3] * inverse) << 16);
    }
    sts64(slot + L::row(r) + 8 * lane, make_uint2(w[0], w[1]));
    *reinterpret_cast<uint2 *>(record + r * kKvHeadDim + 8 * lane) = make_uint2(w[0], w[1]);
  } else {
    const uint4 raw = make_uint4(split2<false>(x[0], x[1], 0), split2<false>(x[2], x[3], 0), split2<false>(x[4], x[5], 0),
                                 split2<false>(x[6], x[7], 0));
    sts128(slot + L::row(r) + 16 * lane, raw);
    *reinterpret_cast<uint4 *>(plane + static_cast<std::size_t>(r0 + r) * 512 + 16 * lane) = raw;
  }
  __syncwarp();
}

// One warp's share of steps [begin, end) of a row over BF16 rows, value by value and without parts: for rows with infinities or
// not-a-numbers, where a part of a query or weight that is zero, or of the other sign, makes a not-a-number of what is none.
// A lane has eight dims of all heads.  16 sequences of 8192 tokens: 89 us without such rows, 480 where all parts come here.
template <bool F32>
__device__ __noinline__ void plain_part(const DecodeParams &p, std::uint32_t sequence, std::uint32_t head, std::uint32_t begin,
                                        std::uint32_t end, float *warp_max, float *warp_sum, float *warp_out) {
  constexpr std::uint32_t kWarps = Shape<false>::kWarps;
  const std::uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  std::uint32_t why;
  const Row row = row_of(p.a, sequence, why);
  float q[kGroup][8] = {}, out[kGroup][8] = {}, top[kGroup], sum[kGroup];
#pragma unroll
  for (std::uint32_t h = 0; h < kGroup; ++h) {
    top[h] = kLowest;
    sum[h] = 0.0F;
    if (h < p.group) {
      load8<F32>(p.a.query, (static_cast<std::size_t>(sequence) * p.a.query_heads + head * p.group + h) * kKvHeadDim + 8 * lane,
                 q[h]);
    }
  }
  for (std::uint32_t s = begin + warp; s < end; s += kWarps) {
    const std::uint32_t tok0 = (s < row.sink_steps ? s : row.window_step + (s - row.sink_steps)) * kStep;
    const unsigned char *keys = row.view.plane(0, head, tok0);
    const unsigned char *values = row.view.plane(1, head, tok0);
    if (keys == nullptr) {
      continue;
    }
    for (std::uint32_t token = tok0; token < tok0 + kStep; ++token) {
      if (token > row.pos || (token < row.low && token >= row.sinks)) {
        continue;
      }
      const std::size_t index = static_cast<std::size_t>(row.view.row_in_plane(token)) * kKvHeadDim + 8 * lane;
      float k[8], v[8];
      load8<false>(keys, index, k);
      load8<false>(values, index, v);
#pragma unroll
      for (std::uint32_t h = 0; h < kGroup; ++h) {
        float logit = 0.0F;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          logit = fmaf(q[h][e], k[e], logit);
        }
#pragma unroll
        for (int step = 16; step > 0; step /= 2) {
          logit += __shfl_xor_sync(0xFFFFFFFFU, logit, step);
        }
        logit *= 0.0625F * kLog2e;
        const float next = fmaxf(top[h], logit);
        const float keep = fast_exp2(top[h] - next), weight = fast_exp2(logit - next);
        top[h] = next;
        sum[h] = fmaf(sum[h], keep, weight);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float term = logit > -INFINITY ? share_of<false>(v[e], weight) : weight * v[e];
          out[h][e] = share_of<false>(out[h][e], keep) + term;
        }
      }
    }
  }
#pragma unroll
  for (std::uint32_t h = 0; h < kGroup; ++h) {
    const float normalise = sum[h] == 0.0F ? 0.0F : 1.0F / sum[h];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      warp_out[(warp * kGroup + h) * kMergePitch + 8 * lane + e] = out[h][e] * normalise;
    }
    if (lane == 0) {
      warp_max[warp * kGroup + h] = top[h];
      warp_sum[warp * kGroup + h] = sum[h];
    }
  }
}

template <bool F32, bool EightBit>
__global__ void __launch_bounds__(Shape<EightBit>::kWarps * 32, Shape<EightBit>::kCtasPerSm)
    kv_decode_kernel(const __grid_constant__ DecodeParams p) {
  using S = Shape<EightBit>;
  using L = Slot<EightBit>;
  constexpr std::uint32_t kWarps = S::kWarps;
  constexpr std::uint32_t kSlots = S::kSlots;
  extern __shared__ __align__(128) unsigned char smem[];
  const std::uint32_t warp = threadIdx.x / 32;
  const std::uint32_t lane = threadIdx.x % 32;
  const int g = static_cast<int>(lane >> 2);
  const int t = static_cast<int>(lane & 3U);
  const std::uint32_t ring = smem_address(smem) + warp * kSlots * L::kBytes;
  const std::uint32_t bars = smem_address(smem) + S::kRingBytes + warp * kSlots * 8;
  if (lane == 0) {
    for (std::uint32_t r = 0; r < kSlots; ++r) {
      mbarrier_init(bars + r * 8, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  grid_dependency_wait();
  grid_dependents_may_launch();

  const Schedule plan = make_schedule(p, blockIdx.x == 0 && warp == 0);
  if (blockIdx.x >= plan.pieces) {
    return;
  }
  const Place start = place_of(plan, p, plan.target != 0 ? static_cast<Count>(blockIdx.x) : plan.bound(blockIdx.x));
  const std::uint64_t policy = evict_first_policy();
  std::uint32_t sequence = start.sequence;
  std::uint32_t head = start.head;
  std::uint32_t step = plan.target != 0 ? start.index * plan.target : start.index;
  Count left = plan.target != 0 ? plan.target : plan.bound(blockIdx.x + 1) - plan.bound(blockIdx.x);
  bool first_row = true;
  std::uint32_t issued = 0, issue_at = 0;                  // slots of this warp that have been asked for
  std::uint32_t waited = 0, wait_at = 0, wait_parity = 0;  // ... that have arrived
  bool healthy = true;

  for (;;) {
    std::uint32_t why;
    const Row row = row_of(p.a, sequence, why);
    const std::uint32_t begin = step;
    const std::uint32_t end = static_cast<std::uint32_t>(min(static_cast<Count>(row.steps), begin + left));
    left -= end - begin;
    const KvView &view = row.view;
    const std::uint32_t my_steps = end - begin > warp ? (end - begin - warp + kWarps - 1) / kWarps : 0;
    const std::uint32_t my_slots = S::kHalves * my_steps;
    auto token_of = [&](std::uint32_t s) { return (s < row.sink_steps ? s : row.window_step + (s - row.sink_steps)) * kStep; };

    // What this lane copies of a step, from the start of the cache or page on: a KiB of the K or V rows (8 bit: lanes 0 to 3 and 4
    // to 7), two rows of the K plane (BF16).
    const std::size_t plane_bytes = view.plane_bytes();
    const std::size_t values_behind = view.kv_heads * plane_bytes; // V plane behind the K plane
    const unsigned char *lane_base = view.base + head * plane_bytes +
                                     (EightBit ? (lane & 3U) * 1024 + (lane & 4U ? values_behind : 0) : lane * 1024);
    // slot n of this row's part.  8 bit: K and V rows of the warp's step n; BF16: the K rows (n even) or V rows of step n / 2
    auto issue = [&](std::uint32_t n) {
      const std::uint32_t tok0 = token_of(begin + warp + n / S::kHalves * kWarps);
      const std::uint32_t slot = ring + issue_at * L::kBytes;
      const std::uint32_t bar = bars + issue_at * 8;
      issue_at = issue_at + 1 == kSlots ? 0 : issue_at + 1;
      ++issued;
      const unsigned char *src = lane_base;
      std::uint32_t row_in_plane = tok0;
      fence_proxy_async(); // earlier accesses to this slot are ordered before the copy
      if (view.table != nullptr) {
        const std::uint32_t page = __ldg(view.table + tok0 / kKvPageTokens);
        row_in_plane = tok0 % kKvPageTokens;
        src += page * (2 * values_behind);
        if (page >= view.pool_pages) {
          if (lane == 0) {
            atomicOr(p.status, static_cast<unsigned int>(RIB200_DEVICE_PAGE_OUT_OF_RANGE));
            mbarrier_expect_tx(bar, 0);
          }
          __syncwarp();
          return;
        }
      }
      if constexpr (EightBit) {
        if (lane == 0) {
          mbarrier_expect_tx(bar, 2 * kKv8BlockBytes);
        }
        __syncwarp();
        if (lane < 8) {
          bulk_copy_g2s(slot + (lane & 4U ? L::kValues : 0U) + (lane & 3U) * L::kPitch,
                        src + static_cast<std::size_t>(row_in_plane / kStep) * kKv8BlockBytes, (lane & 3U) == 3 ? 1040 : 1024,
                        bar, policy);
        }
      } else {
        const std::uint32_t rows = min(kStep, row.pos + 1 - tok0);
        if (lane == 0) {
          mbarrier_expect_tx(bar, rows * 512);
        }
        __syncwarp();
        if (2 * lane < rows) {
          bulk_copy_g2s(slot + lane * L::kPitch,
                        src + static_cast<std::size_t>(row_in_plane) * 512 + (n & 1U ? values_behind : 0),
                        min(2U, rows - 2 * lane) * 512, bar, policy);
        }
      }
    };
    // The next slot, when its rows are here; kNoSlot if they do not come.
    auto wait = [&] {
      const std::uint32_t bar = bars + wait_at * 8;
      if (!mbarrier_try_wait(bar, wait_parity)) {
        const long long started = clock64();
        while (!mbarrier_try_wait(bar, wait_parity)) {
          if (clock64() - started > kWaitLimitCycles) {
            healthy = false;
            break;
          }
        }
      }
      healthy = __all_sync(0xFFFFFFFFU, healthy);
      if (!healthy) {
        return kNoSlot;
      }
      const std::uint32_t slot = ring + wait_at * L::kBytes;
      ++waited;
      if (++wait_at == kSlots) {
        wait_at = 0;
        wait_parity ^= 1U;
      }
      return slot;
    };

    const std::uint32_t early = min(my_slots, kSlots - 1);
    for (std::uint32_t n = 0; n < early; ++n) {
      issue(n);
    }
    Query<F32, EightBit> q;
    const std::size_t q_base =
        (static_cast<std::size_t>(sequence) * p.a.query_heads + head * p.group) * kKvHeadDim;
    q.load(p.a.query, q_base, p.group, g, t);

    // The new token's row belongs to the row's last step.
    const bool appends = end == row.steps && my_steps != 0 && (end - 1 - begin) % kWarps == warp;
    NewRow<F32> fresh[2];
    if (appends) {
      const std::size_t index =
          (static_cast<std::size_t>(sequence) * p.a.caches.kv_heads + head) * kKvHeadDim + 8 * lane;
      fresh[0].load(p.a.key, index);
      fresh[1].load(p.a.value, index);
    }
    auto append = [&](std::uint32_t slot, std::uint32_t is_value, std::uint32_t tok0) {
      unsigned char *plane = view.plane(is_value, head, tok0);
      if (plane != nullptr) {
        float x[8];
        fresh[is_value].get(x);
        append_row<EightBit>(slot, plane, view.row_in_plane(tok0), row.pos - tok0, x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
      }
    };

    float oacc[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      oacc[i][0] = oacc[i][1] = oacc[i][2] = oacc[i][3] = 0.0F;
    }
    float run_max = kLowest;                 // of head t, base 2; 8 bit: rounded up to an integer
    float run_sum = 0.0F;                    // this lane's share of head t's sum
    // 8 bit, of head t: 2^unit is the unit of the sums of values.  The largest weight (relative to 2^run_max) times the V scale
    // of its block so far, rounded up to a power of two; from -100 to 119 once there is one.
    [[maybe_unused]] float unit = kLowest;

    for (std::uint32_t i = 0; i < my_steps; ++i) {
      const std::uint32_t tok0 = token_of(begin + warp + i * kWarps);
      const bool newest = appends && i + 1 == my_steps;
      const bool whole = tok0 + kStep <= row.pos + 1 && (tok0 >= row.low || tok0 + kStep <= row.sinks);
      auto seen = [&](std::uint32_t token) { return token <= row.pos && (token >= row.low || token < row.sinks); };

      // ---- K: logits and weights ----
      fence_proxy_async();
      __syncwarp(); // all lanes are done with the slot that is filled next
      if (S::kHalves * i + kSlots - 1 < my_slots) {
        issue(S::kHalves * i + kSlots - 1);
      }
      const std::uint32_t k_slot = wait();
      if (k_slot == kNoSlot) {
        break;
      }
      if (newest) {
        append(k_slot, 0, tok0);
      }
      float s[4][4] = {};
      float logit_scale = q.scale;
      std::uint32_t token_a, token_b; // of the lane's two rows
      if constexpr (EightBit) {
        // rows g and g + 8 are tokens a and a + 2; lanes of even and odd g read groups of rows two apart, whose pitch puts
        // them four bank groups apart, and t takes four neighbouring 16-byte pieces
        const std::uint32_t local = (g & 1) * 8 + ((g >> 2) & 1) * 4 + ((g >> 1) & 1);
        token_a = tok0 + local;
        token_b = token_a + 2;
        const std::uint32_t address = k_slot + L::row(local) + 16 * t;
        logit_scale *= lds_float(k_slot + kSlotScale);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          std::uint32_t a[4], b[4];
          lds128(address + 64 * part, a);
          lds128(address + 512 + 64 * part, b);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            mma<true>(s[w], half2_of_low(a[w]), half2_of_low(b[w]), half2_of_high(a[w]), half2_of_high(b[w]),
                      q.fragment[8 * part + 2 * w], q.fragment[8 * part + 2 * w + 1]);
          }
        }
      } else {
        token_a = tok0 + 2 * g;
        token_b = token_a + 1;
        const std::uint32_t mi = lane >> 3;
        const std::uint32_t address = k_slot + (lane & 7U) * L::kPitch + (mi & 1U) * 512 + (mi >> 1) * 16;
#pragma unroll
        for (int ks = 0; ks < 16; ++ks) {
          std::uint32_t a[4];
          ldmatrix_x4(address + ks * 32, a);
          mma<false>(s[ks & 3], a[0], a[1], a[2], a[3], q.fragment[2 * ks], q.fragment[2 * ks + 1]);
          if constexpr (q.kFourParts) {
            mma<false>(s[ks & 3], a[0], a[1], a[2], a[3], q.rest[2 * ks], q.rest[2 * ks + 1]);
          }
        }
      }
      // both parts of head t's logits
      float logit_a = (((s[0][0] + s[1][0]) + (s[2][0] + s[3][0])) + ((s[0][1] + s[1][1]) + (s[2][1] + s[3][1]))) * logit_scale;
      float logit_b = (((s[0][2] + s[1][2]) + (s[2][2] + s[3][2])) + ((s[0][3] + s[1][3]) + (s[2][3] + s[3][3]))) * logit_scale;
      if (!whole) {
        logit_a = seen(token_a) ? logit_a : -INFINITY;
        logit_b = seen(token_b) ? logit_b : -INFINITY;
      }
      float step_max = fmaxf(logit_a, logit_b);
      step_max = fmaxf(step_max, __shfl_xor_sync(0xFFFFFFFFU, step_max, 4));
      step_max = fmaxf(step_max, __shfl_xor_sync(0xFFFFFFFFU, step_max, 8));
      step_max = fmaxf(step_max, __shfl_xor_sync(0xFFFFFFFFU, step_max, 16));
      if constexpr (EightBit) {
        step_max = ceilf(step_max);
      }
      if (__any_sync(0xFFFFFFFFU, step_max > run_max)) {
        const float new_max = fmaxf(run_max, step_max);
        const float rescale = fast_exp2(run_max - new_max);
        run_sum *= rescale;
        if constexpr (EightBit) {
          unit -= new_max - run_max;
        } else {
#pragma unroll
          for (int m = 0; m < 16; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              oacc[m][e] *= rescale;
            }
          }
        }
        run_max = new_max;
      }
      float weight_a = fast_exp2(logit_a - run_max);
      float weight_b = fast_exp2(logit_b - run_max);
      run_sum += weight_a + weight_b;

      // ---- V ----
      std::uint32_t v_slot = k_slot + L::kValues;
      if constexpr (S::kHalves == 2) {
        fence_proxy_async();
        __syncwarp();
        if (2 * i + kSlots < my_slots) {
          issue(2 * i + kSlots);
        }
        v_slot = wait();
        if (v_slot == kNoSlot) {
          break;
        }
      }
      if (newest) {
        append(v_slot, 1, tok0);
      }
      if (!whole) { // what is not visible may be anything, a not-a-number too: zeros in its place
        for (std::uint32_t r = 0; r < kStep; ++r) {
          if (!seen(tok0 + r)) {
            if constexpr (EightBit) {
              sts64(v_slot + L::row(r) + 8 * lane, make_uint2(0U, 0U));
            } else {
              sts128(v_slot + L::row(r) + 16 * lane, make_uint4(0U, 0U, 0U, 0U));
            }
          }
        }
        __syncwarp();
      }
      // The weights as the other operand: lane (g, t) gives column g (head g / 2, part g & 1) for four tokens.
      const int part = g & 1;
      if constexpr (EightBit) {
        const float v_exponent =
            static_cast<float>(static_cast<int>(__float_as_uint(lds_float(v_slot + kSlotScale)) >> 23) - 127);
        const float step_unit = v_exponent + (step_max - run_max);
        if (__any_sync(0xFFFFFFFFU, step_unit > unit)) {
          const float new_unit = fmaxf(unit, step_unit);
          const float rescale = fast_exp2(unit - new_unit);
          unit = new_unit;
#pragma unroll
          for (int m = 0; m < 16; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              oacc[m][e] *= rescale;
            }
          }
        }
        // the weights times the block's scale in that unit: 2^15 at most
        weight_a = fast_exp2((logit_a - run_max) + (v_exponent - unit)) * kWeightUnit;
        weight_b = fast_exp2((logit_b - run_max) + (v_exponent - unit)) * kWeightUnit;
        // tokens 4 t .. 4 t + 3: token b3 b2 b1 b0 is row b1 ? b : a of the lane with g = b2 b0 b3
        const int from = (((t & 1) << 2) | (t >> 1)) * 4 + (g >> 1);
        const float w0 = __shfl_sync(0xFFFFFFFFU, weight_a, from);
        const float w1 = __shfl_sync(0xFFFFFFFFU, weight_a, from + 8);
        const float w2 = __shfl_sync(0xFFFFFFFFU, weight_b, from);
        const float w3 = __shfl_sync(0xFFFFFFFFU, weight_b, from + 8);
        const std::uint32_t b0 = split2<true>(w0, w1, part);
        const std::uint32_t b1 = split2<true>(w2, w3, part);
        const std::uint32_t address = v_slot + t * L::kPitch + 16 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          std::uint32_t c[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            lds128(address + e * 256 + u * 128, c[e]);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            // bytes of neighbouring tokens side by side; rows g and g + 8 of a product are neighbouring dims
            const std::uint32_t x = __byte_perm(c[0][w], c[1][w], 0x5140), y = __byte_perm(c[0][w], c[1][w], 0x7362);
            const std::uint32_t x2 = __byte_perm(c[2][w], c[3][w], 0x5140), y2 = __byte_perm(c[2][w], c[3][w], 0x7362);
            mma<true>(oacc[8 * u + 2 * w], half2_of_low(x), half2_of_high(x), half2_of_low(x2), half2_of_high(x2), b0, b1);
            mma<true>(oacc[8 * u + 2 * w + 1], half2_of_low(y), half2_of_high(y), half2_of_low(y2), half2_of_high(y2), b0, b1);
          }
        }
      } else {
        // tokens 2 m of rows m < 8 and 2 m + 1 of rows m + 8
        const int from = (2 * t) * 4 + (g >> 1);
        const float w0 = __shfl_sync(0xFFFFFFFFU, weight_a, from);
        const float w1 = __shfl_sync(0xFFFFFFFFU, weight_a, from + 4);
        const float w2 = __shfl_sync(0xFFFFFFFFU, weight_b, from);
        const float w3 = __shfl_sync(0xFFFFFFFFU, weight_b, from + 4);
        std::uint32_t b0, b1;
        [[maybe_unused]] std::uint32_t rest0, rest1;
        if constexpr (q.kFourParts) {
          split4(w0, w1, part, b0, rest0);
          split4(w2, w3, part, b1, rest1);
        } else {
          b0 = split2<false>(w0, w1, part);
          b1 = split2<false>(w2, w3, part);
        }
        const std::uint32_t mi = lane >> 3;
        const std::uint32_t address = v_slot + (lane & 7U) * L::kPitch + (mi >> 1) * 512 + (mi & 1U) * 16;
#pragma unroll
        for (int m = 0; m < 16; ++m) {
          std::uint32_t a[4];
          ldmatrix_x4_trans(address + m * 32, a);
          mma<false>(oacc[m], a[0], a[1], a[2], a[3], b0, b1);
          if constexpr (q.kFourParts) {
            mma<false>(oacc[m], a[0], a[1], a[2], a[3], rest0, rest1);
          }
        }
      }
    }
    if (!healthy) {
      // what has been asked for is on its way still: it has to be here before anything else happens to the ring
      const long long started = clock64();
      for (std::uint32_t at = waited; at < issued; ++at) {
        while (!mbarrier_try_wait(bars + at % kSlots * 8, (at / kSlots) & 1U) && clock64() - started <= kWaitLimitCycles) {
        }
      }
      if (lane == 0) {
        atomicOr(p.status, static_cast<unsigned int>(RIB200_DEVICE_WAIT_TIMED_OUT));
      }
    }

    run_sum += __shfl_xor_sync(0xFFFFFFFFU, run_sum, 4);
    run_sum += __shfl_xor_sync(0xFFFFFFFFU, run_sum, 8);
    run_sum += __shfl_xor_sync(0xFFFFFFFFU, run_sum, 16);

    // (not healthy: what is there is not used)
    bool odd = false;
    if constexpr (!EightBit) {
      float any[4] = {run_sum, 0.0F, 0.0F, 0.0F};
#pragma unroll
      for (int m = 0; m < 16; ++m) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          any[e] += oacc[m][e];
        }
      }
      const float all = (any[0] + any[1]) + (any[2] + any[3]); // a not-a-number stays one
      odd = __any_sync(0xFFFFFFFFU, all != all);
    }

    // ---- the warps' shares of this row's part come together ----
    const bool alone = begin == 0 && end == row.steps;
    float4 gate[2]; // of this thread's items
    if (alone) {
#pragma unroll
      for (std::uint32_t i = 0; i < 2; ++i) {
        const std::uint32_t item = threadIdx.x + i * kWarps * 32;
        if (item < p.group * 64) {
          gate[i] = load4<F32>(p.a.gate, q_base + item / 64 * kKvHeadDim + item % 64 * 4);
        }
      }
    }
    const bool stop = __syncthreads_or(!healthy ? 1 : 0) != 0; // every warp has left its ring: the merge area lies there
    float *merge = reinterpret_cast<float *>(smem);
    float *warp_max = merge;                      // [warp][head]
    float *warp_sum = merge + kWarps * kGroup;
    float *warp_out = merge + 2 * kWarps * kGroup; // [warp][head][kMergePitch], normalised
    if (odd && !stop) {
      if constexpr (!EightBit) {
        plain_part<F32>(p, sequence, head, begin, end, warp_max, warp_sum, warp_out);
      }
    } else {
      if (g == 0) {
        warp_max[warp * kGroup + t] = run_max;
        warp_sum[warp * kGroup + t] = run_sum;
      }
      const float normalise = run_sum == 0.0F ? 0.0F : (EightBit ? (1.0F / kWeightUnit) / run_sum : 1.0F / run_sum);
      {
        float *dst = warp_out + (warp * kGroup + t) * kMergePitch;
        if constexpr (EightBit) {
          const float scale = fast_exp2(unit);
          auto value = [&](int m, int e) { return (oacc[m][e] + oacc[m][e + 1]) * normalise * scale; };
#pragma unroll
          for (int m = 0; m < 16; m += 2) {
            *reinterpret_cast<float4 *>(dst + 128 * (m >> 3) + 16 * g + 2 * (m & 7)) =
                make_float4(value(m, 0), value(m, 2), value(m + 1, 0), value(m + 1, 2));
          }
        } else {
#pragma unroll
          for (int m = 0; m < 16; ++m) {
            dst[16 * m + g] = (oacc[m][0] + oacc[m][1]) * normalise;
            dst[16 * m + g + 8] = (oacc[m][2] + oacc[m][3]) * normalise;
          }
        }
      }
    }
    __syncthreads();
    float *part = p.parts + static_cast<std::size_t>(plan.target != 0 ? blockIdx.x : 2 * blockIdx.x + (first_row ? 0 : 1)) *
                                kPartFloats;
    static_assert(2 * kWarps * 32 >= kGroup * 64, "two items a thread at most");
#pragma unroll
    for (std::uint32_t i = 0; i < 2; ++i) {
      const std::uint32_t item = threadIdx.x + i * kWarps * 32;
      if (item >= p.group * 64) {
        break;
      }
      const std::uint32_t h = item / 64;
      const std::uint32_t dim0 = item % 64 * 4;
      float top = warp_max[h];
#pragma unroll
      for (std::uint32_t w = 1; w < kWarps; ++w) {
        top = fmaxf(top, warp_max[w * kGroup + h]);
      }
      float sum = 0.0F;
      float4 out = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
      for (std::uint32_t w = 0; w < kWarps; ++w) {
        const float share = warp_sum[w * kGroup + h] * fast_exp2(warp_max[w * kGroup + h] - top);
        const float4 v = share_of<EightBit>(
            *reinterpret_cast<const float4 *>(warp_out + (w * kGroup + h) * kMergePitch + dim0), share);
        sum += share;
        out.x += v.x; out.y += v.y; out.z += v.z; out.w += v.w;
      }
      const float inverse = 1.0F / sum;
      out = make_float4(out.x * inverse, out.y * inverse, out.z * inverse, out.w * inverse);
      if (alone) {
        const std::size_t index = q_base + h * kKvHeadDim + dim0;
        store4<F32>(p.a.output, index, gated(out, gate[i]));
      } else {
        *reinterpret_cast<float4 *>(part + h * kKvHeadDim + dim0) = out;
        if (dim0 == 0) {
          part[kGroup * kKvHeadDim + h] = top;
          part[kGroup * kKvHeadDim + kGroup + h] = sum;
        }
      }
    }
    if (left == 0 || plan.target != 0 || stop) {
      return;
    }
    first_row = false;
    step = 0;
    if (++head == p.a.caches.kv_heads) {
      head = 0;
      std::uint32_t ignored;
      do {
        ++sequence;
      } while (row_of(p.a, sequence, ignored).steps == 0);
    }
    fence_proxy_async(); // the merge area becomes ring again
    __syncthreads();
  }
}

// Puts the parts of a row together.  Where rows are cut by themselves there are few rows and many parts: grid = (rows, query
// heads of a KV head), eight groups of 64 threads take the parts in turn.  Else there are many rows of two or three parts: a
// block for every cut between two CTAs, which serves the row that the cut is the first one in, 64 threads a query head.  A
// thread has four dims.
constexpr std::uint32_t kCombineGroups = 8;
template <bool F32, bool EightBit>
__global__ void __launch_bounds__(kCombineGroups * 64) kv_combine_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float group_max[kCombineGroups], group_sum[kCombineGroups];
  __shared__ float4 group_out[kCombineGroups][64];
  grid_dependents_may_launch();
  // The first kernel lets this one in when everything in front of both has ended: positions, tables and gates are there, and
  // only the parts have to be waited for.
  const std::uint32_t lane = threadIdx.x % 64;
  // What is queued behind this kernel may rely on the first one having ended: one block at least stays until it has.
  auto leave = [] {
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      grid_dependency_wait();
    }
  };
  const Schedule plan = make_schedule(p, false);
  Place row;
  std::uint32_t count, first, first_slot;
  if (p.by_rows != 0) {
    row.sequence = blockIdx.x / p.a.caches.kv_heads;
    row.head = blockIdx.x % p.a.caches.kv_heads;
    Count unit;
    count = units_of_row(plan, p, row.sequence, row.head, unit);
    first = first_slot = static_cast<std::uint32_t>(unit);
    if (count <= 1) {
      leave();
      return;
    }
  } else {
    if (blockIdx.x + 1 >= plan.pieces) {
      leave();
      return;
    }
    const Count piece_begin = plan.bound(blockIdx.x), cut = plan.bound(blockIdx.x + 1);
    row = place_of(plan, p, cut - 1);
    std::uint32_t why;
    const Count row_begin = cut - 1 - row.index;
    const Count row_end = row_begin + row_of(p.a, row.sequence, why).steps;
    if (cut >= row_end || piece_begin > row_begin) {
      leave();
      return; // no cut inside a row, or not the first one
    }
    first = blockIdx.x;
    std::uint32_t last = first + 1; // the piece with the row's last step
    while (plan.bound(last + 1) < row_end) {
      ++last;
    }
    count = last - first + 1;
    first_slot = 2 * first + (piece_begin == row_begin ? 0U : 1U);
  }
  const std::uint32_t h = p.by_rows != 0 ? blockIdx.y : threadIdx.x / 64;
  const std::uint32_t group = p.by_rows != 0 ? threadIdx.x / 64 : 0;
  const std::uint32_t groups = p.by_rows != 0 ? kCombineGroups : 1;
  const std::size_t index =
      (static_cast<std::size_t>(row.sequence) * p.a.query_heads + row.head * p.group + h) * kKvHeadDim + lane * 4;
  float4 gate = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
  if (group == 0) {
    gate = load4<F32>(p.a.gate, index);
  }
  grid_dependency_wait();
  auto slot = [&](std::uint32_t i) {
    return p.parts + static_cast<std::size_t>(i == 0 ? first_slot : (first + i) * (p.by_rows != 0 ? 1U : 2U)) * kPartFloats;
  };
  float top = kLowest, sum = 0.0F;
  float4 out = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
  constexpr std::uint32_t kAtOnce = 8;
  for (std::uint32_t i = group; i < count; i += groups * kAtOnce) {
    float m[kAtOnce], l[kAtOnce];
    float4 v[kAtOnce];
#pragma unroll
    for (std::uint32_t j = 0; j < kAtOnce; ++j) {
      if (i + groups * j < count) {
        const float *part = slot(i + groups * j);
        m[j] = part[kGroup * kKvHeadDim + h];
        l[j] = part[kGroup * kKvHeadDim + kGroup + h];
        v[j] = *reinterpret_cast<const float4 *>(part + h * kKvHeadDim + lane * 4);
      }
    }
#pragma unroll
    for (std::uint32_t j = 0; j < kAtOnce; ++j) {
      if (i + groups * j < count) {
        const float next = fmaxf(top, m[j]);
        const float keep = fast_exp2(top - next), take = l[j] * fast_exp2(m[j] - next);
        sum = sum * keep + take;
        const float4 kept = share_of<EightBit>(out, keep), taken = share_of<EightBit>(v[j], take);
        out = make_float4(kept.x + taken.x, kept.y + taken.y, kept.z + taken.z, kept.w + taken.w);
        top = next;
      }
    }
  }
  if (p.by_rows != 0) {
    if (lane == 0) {
      group_max[group] = top;
      group_sum[group] = sum;
    }
    group_out[group][lane] = out;
    __syncthreads();
    if (group != 0) {
      return;
    }
#pragma unroll
    for (std::uint32_t i = 1; i < kCombineGroups; ++i) {
      top = fmaxf(top, group_max[i]);
    }
    sum = 0.0F;
    out = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
    for (std::uint32_t i = 0; i < kCombineGroups; ++i) {
      const float weight = fast_exp2(group_max[i] - top);
      sum += group_sum[i] * weight;
      const float4 v = share_of<EightBit>(group_out[i][lane], weight);
      out.x += v.x; out.y += v.y; out.z += v.z; out.w += v.w;
    }
  }
  const float inverse = 1.0F / sum;
  store4<F32>(p.a.output, index,
              gated(make_float4(out.x * inverse, out.y * inverse, out.z * inverse, out.w * inverse), gate));
}

template <bool F32, bool EightBit> void configure_once() {
  static std::once_flag flags[64];
  int device = 0;
  cuda_ok(cudaGetDevice(&device), "cudaGetDevice");
  require(device >= 0 && device < 64, "device ordinal out of range", RIB200_STATUS_INTERNAL);
  std::call_once(flags[device], [] {
    cuda_ok(cudaFuncSetAttribute(kv_decode_kernel<F32, EightBit>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(Shape<EightBit>::kSmemBytes)),
            "KV decode shared-memory opt-in");
  });
}

template <bool F32, bool EightBit> void launch(DecodeParams p, cudaStream_t stream) {
  using S = Shape<EightBit>;
  configure_once<F32, EightBit>();
  int device = 0, sms = 0;
  cuda_ok(cudaGetDevice(&device), "cudaGetDevice");
  cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "SM count query");
  p.ctas = std::min<std::uint32_t>(kMaxCtas, static_cast<std::uint32_t>(sms * S::kCtasPerSm));
  p.min_steps = S::kWarps;
  const std::uint32_t rows = p.a.batch * p.a.caches.kv_heads;
  p.by_rows = 8 * rows <= p.ctas ? 1U : 0U;
  launch_programmatic(kv_decode_kernel<F32, EightBit>, dim3(p.ctas), dim3(S::kWarps * 32), S::kSmemBytes, stream,
                      "KV decode launch", p);
  const dim3 grid = p.by_rows != 0 ? dim3(rows, p.group) : dim3(p.ctas - 1);
  launch_programmatic(kv_combine_kernel<F32, EightBit>, grid, dim3(64 * (p.by_rows != 0 ? kCombineGroups : p.group)), 0, stream,
                      "KV decode combine launch", p);
}

} // namespace

std::size_t kv_decode_workspace_bytes() { return static_cast<std::size_t>(2) * kMaxCtas * kPartFloats * sizeof(float); }

void launch_kv_decode(const KvDecodeArgs &a, cudaStream_t stream) {
  DecodeParams p{};
  p.a = a;
  p.parts = static_cast<float *>(a.workspace);
  p.status = device_status_word();
  p.group = a.query_heads / a.caches.kv_heads;
  if (a.caches.eight_bit) {
    a.activations_f32 ? launch<true, true>(p, stream) : launch<false, true>(p, stream);
  } else {
    a.activations_f32 ? launch<true, false>(p, stream) : launch<false, false>(p, stream);
  }
}

} // namespace rib200
