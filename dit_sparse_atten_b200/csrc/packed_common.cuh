// Shared device helpers of the packed-request kernels (residual_norm.cu,
// lora_*.cu, packed_attention.cu): several requests' tokens on one row axis,
// request s owning rows [starts[s], starts[s + 1]).  The offsets are device
// data, so every kernel checks what it reads and reports kErrBadRoute instead
// of following it out of range.
#pragma once

#include <stdint.h>

#include "bsa_common.cuh"

namespace bsa {

// Number of i in [1, n] with key(i) <= v, for a key that does not decrease
// with i: the request that owns row v when key(i) = starts[i].  All 32 lanes
// of the warp call it together; every round tests 32 evenly spaced keys, so
// up to 32 requests take one round of loads and 1,024 take two.  Keys in
// disorder give some value in [0, n].
template <typename Key>
__device__ __forceinline__ int warp_count_le(int n, int64_t v, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 32) {
    const int step = (n + 31) / 32;
    const int i = (lane + 1) * step;
    const bool le = i <= n && key(lo + i) <= v;
    const int k = __popc(__ballot_sync(0xffffffffu, le));
    lo += k * step;
    n = min(step - 1, n - k * step);
  }
  const bool le = lane < n && key(lo + lane + 1) <= v;
  return lo + __popc(__ballot_sync(0xffffffffu, le));
}

// The request that owns `row`, or -1 (starts do not cover the row).
__device__ __forceinline__ int request_of_row(const int32_t* __restrict__ starts, int requests,
                                              int64_t row) {
  const int s = warp_count_le(requests, row, [&](int i) {
    return static_cast<int64_t>(__ldg(starts + i));
  });
  if (s >= requests || row < __ldg(starts + s)) return -1;
  return s;
}

// A producer's ring of kSlots shared-memory slots.  Load j goes to slot j %
// kSlots and completes phase j / kSlots of the slot's "full" barrier.  `armed`
// counts the loads that have been issued: arm() stands behind each, and nowhere
// else, so that a producer which gives up knows what is still on its way.
template <int kSlots>
struct LoadRing {
  int armed = 0;
  __host__ __device__ int slot() const { return armed % kSlots; }
  // parity of the slot's "empty" barrier to wait for before the next load
  __host__ __device__ uint32_t empty_parity() const {
    return static_cast<uint32_t>(((armed / kSlots) & 1) ^ 1);
  }
  __host__ __device__ void arm() { ++armed; }
  // f(slot, parity of its "full" barrier) for the loads that may be in flight
  template <typename F>
  __host__ __device__ void for_each_open(F f) const {
    for (int j = armed > kSlots ? armed - kSlots : 0; j < armed; ++j)
      f(j % kSlots, static_cast<uint32_t>((j / kSlots) & 1));
  }
};

// Programmatic dependent launch: wait until the kernels this one depends on
// have completed and their writes are visible (returns at once when the
// launch carries no such dependency); let the next kernel's blocks start.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace bsa
