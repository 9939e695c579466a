// Device helpers shared by the two latent-attention kernels (latent.cu,
// latent_prefill.cu), beside those of prefill_common.cuh.
#pragma once

#include "prefill_common.cuh"

namespace nvb {

// A named stretch of memory, for the entry points' checks that what they write overlaps nothing else.
struct Stretch {
  const char* name;
  const void* at;  // null: not there
  long long bytes;
};
inline bool overlap(const Stretch& a, const Stretch& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at && b.at && x < y + uintptr_t(b.bytes) && y < x + uintptr_t(a.bytes);
}
// The first `written` of the stretches against all: -1 with the message where two overlap.
template <int N>
int check_apart(const Stretch (&s)[N], int written) {
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < N; ++j)
      if (overlap(s[i], s[j])) return api_detail::fail("%s overlaps %s", s[i].name, s[j].name);
  return 0;
}

namespace latent_common {

using namespace prefill_common;

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleLog2 = 8.0f;  // the maximum in use moves when it grew by 2^8 (P <= 2^8)

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, kErrLatentWait); }
// Every lane waits; the warp goes on only if all of them saw the phase complete.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(bar, parity));
}

// One thread of the warp, which the compiler knows to be one: the operands of its TMA and MMA instructions then stay in
// uniform registers. Under `lane == 0` every instruction moves them there again: an MMA takes 45 to 130 cycles to issue,
// 32 (M = N = 64) to 48 (M = 128, N = 64) this way, which is what it takes to read its operands.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// One arrival, and `bytes` to land. These take shared-memory addresses.
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                               int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// With an L2 eviction policy.
__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                               int c2, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

// Whether a pair of BF16 holds an infinity or NaN: an exponent of all ones carries into the sign's place.
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {  // such halves as 0
  return w & ~(((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u));
}

}  // namespace latent_common
}  // namespace nvb
