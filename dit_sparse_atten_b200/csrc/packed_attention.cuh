// Parts of packed_attention.cu: finding an item's request, the keys each of its
// rows sees, and the key-by-key way out for values that are not finite.
#pragma once

#include "attention_softmax.cuh"
#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace packed {

constexpr int kHeadDim = 128;
constexpr int kBlock = 128;             // keys a block
constexpr int kPanel = kBlock * 128;    // 64 columns x 128 rows, bf16
constexpr int kSlotBytes = 2 * kPanel;

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

// Queries q0 .. q0 + tokens of one request and its keys (uniform over the
// caller's warp).
struct Work {
  int64_t q0;          // first query row
  int64_t k0;          // first key row of the request
  int tokens;          // queries (0: nothing to do)
  int first_limit;     // keys that the first query sees, before clamping to [0, keys]
  int keys;            // keys of the request
};

// Query `token` of the item sees keys [0, limit).
__device__ __forceinline__ int row_limit(const Work& w, int token, bool causal) {
  if (token >= w.tokens) return 0;
  return causal ? max(0, min(w.keys, w.first_limit + token)) : w.keys;
}

// The item of slot `slot`, tt queries a slot.
__device__ __forceinline__ Work find_work(const PackedArgs& a, int64_t slot, int tt) {
  Work w{};
  const int s = warp_count_le(a.requests, slot, [&](int i) {
    return static_cast<int64_t>(__ldg(a.q_starts + i)) / tt + i;
  });
  if (s >= a.requests) return w;
  const int64_t qb = __ldg(a.q_starts + s), qe = __ldg(a.q_starts + s + 1);
  const int64_t kb = __ldg(a.k_starts + s), ke = __ldg(a.k_starts + s + 1);
  const bool bad = qb < 0 || qe < qb || qe > a.q_rows || kb < 0 || ke < kb || ke > a.k_rows ||
                   (s == 0 && qb != 0) || (s == a.requests - 1 && qe != a.q_rows);
  if (bad && (threadIdx.x & 31) == 0) atomicOr(a.err_word, kErrBadRoute);
  if (qb < 0 || qe > a.q_rows || kb < 0 || ke < kb || ke > a.k_rows) return w;
  w.q0 = qb + (slot - (qb / tt + s)) * tt;
  if (w.q0 < qb || w.q0 >= qe) return w;
  w.k0 = kb;
  w.tokens = static_cast<int>(min(static_cast<int64_t>(tt), qe - w.q0));
  w.keys = static_cast<int>(ke - kb);
  // int: q_rows, k_rows < 2^31 - 256
  w.first_limit = a.causal ? static_cast<int>(w.q0 - qb + 1 + (ke - kb) - (qe - qb)) : w.keys;
  return w;
}

// Key blocks that the item sees.
__device__ __forceinline__ int item_blocks(const Work& w, bool causal) {
  return (row_limit(w, w.tokens - 1, causal) + kBlock - 1) / kBlock;
}
// Parts of an item of `blocks` key blocks.
__device__ __forceinline__ int parts_of(int blocks, const PackedArgs& a) {
  return max(1, min(a.splits, blocks / a.part_blocks));
}
// Narrows `w` to one part of its keys (tokens = 0: there is no such part).
__device__ __forceinline__ void take_part(Work& w, int part, const PackedArgs& a) {
  if (w.tokens == 0) return;
  const int blocks = item_blocks(w, a.causal);
  const int parts = parts_of(blocks, a);
  if (part >= parts) {
    w.tokens = 0;
    return;
  }
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks) * part / parts);
  const int b1 = static_cast<int>(static_cast<int64_t>(blocks) * (part + 1) / parts);
  w.k0 += static_cast<int64_t>(b0) * kBlock;
  w.first_limit -= b0 * kBlock;
  w.keys = min(w.keys - b0 * kBlock, (b1 - b0) * kBlock);
}

// The masked end of a block of V in shared memory (a warp): rows [real, 128)
// lie past the request's end and are zeroed (0 * whatever another request
// holds there would reach O); rows [open, real) are hidden from part of the
// tile, and true is returned if one of them holds a value that is not finite.
__device__ __forceinline__ bool clean_masked_values(uint8_t* tile, int open, int real) {
  const int lane = threadIdx.x & 31;
  // a row is 8 chunks of 16 bytes in each panel; which of them is which (the
  // swizzle) does not matter for zeroing or scanning a whole row
  for (int i = lane + real * 8; i < kBlock * 8; i += 32) {
    *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(tile + kPanel + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  bool found = false;
  for (int i = lane + open * 8; i < real * 8; i += 32) {
#pragma unroll
    for (int panel = 0; panel < 2; ++panel) {
      const uint4 x = *reinterpret_cast<const uint4*>(tile + panel * kPanel + i * 16);
      const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int p = 0; p < 4; ++p)
        found |= (words[p] & 0x7f80u) == 0x7f80u || (words[p] & 0x7f800000u) == 0x7f800000u;
    }
  }
  fence_proxy_async_smem();
  return __any_sync(0xffffffffu, found);
}

// One query row key by key in float32 (a warp; lane owns 4 features): the way
// out when V holds non-finite values at masked keys.  Keys [0, end), of which
// `own` >= 0 takes blocks own, own + 2, ... only.  Returns the row's stabiliser
// (log2 domain) and sum; o is relative to the stabiliser.
static __device__ __noinline__ float2 exact_row(const PackedArgs& a, const __nv_bfloat16* q,
                                                int64_t k0, int head, int own, int end, float c,
                                                float4& o) {
  const int lane = threadIdx.x & 31;
  float qf[4], m = -INFINITY, l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int e = 0; e < 4; ++e) qf[e] = __bfloat162float(q[lane * 4 + e]);
  for (int j = 0; j < end; ++j) {
    if (own >= 0 && (j / kBlock & 1) != own) continue;
    const int64_t row = k0 + j;
    const __nv_bfloat16* k = a.k + row * a.k_stride_t + head * a.k_stride_h + lane * 4;
    const __nv_bfloat16* v = a.v + row * a.v_stride_t + head * a.v_stride_h + lane * 4;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(qf[e], __bfloat162float(k[e]), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= c;
    const float m_new = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
    const float p = m_new == -INFINITY && s == -INFINITY ? 0.f : ex2_approx(s - m_new);
    l = l * keep + p;
    o.x = fmaf(p, __bfloat162float(v[0]), m == -INFINITY ? 0.f : o.x * keep);
    o.y = fmaf(p, __bfloat162float(v[1]), m == -INFINITY ? 0.f : o.y * keep);
    o.z = fmaf(p, __bfloat162float(v[2]), m == -INFINITY ? 0.f : o.z * keep);
    o.w = fmaf(p, __bfloat162float(v[3]), m == -INFINITY ? 0.f : o.w * keep);
    m = m_new;
  }
  return make_float2(m, l);
}

}  // namespace packed
}  // namespace bsa
