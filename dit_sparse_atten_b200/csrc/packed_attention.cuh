// Parts of packed_attention.cu: finding an item's request, the keys each of its
// rows sees, and values that are not finite at keys that only some rows see.
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

// Keys of an item that some of its queries see and some do not: fewer than its
// queries, at most 256.  A bit each, from the first query's limit on.
constexpr int kHiddenWords = 8;

// The masked end of a block of V in shared memory (a warp): rows [real, 128)
// lie past the request's end and are zeroed (0 * whatever another request
// holds there would reach O).  Rows [first, real) are hidden from part of the
// item, `first` being the first query's limit: their elements that are not
// finite are zeroed too, and bit row - first of `odd` says that a row had one.
__device__ __forceinline__ void clean_masked_values(uint8_t* tile, int first, int real, uint32_t* odd) {
  const int lane = threadIdx.x & 31;
  // a row is 8 chunks of 16 bytes in each panel; which of them is which (the
  // swizzle) does not matter for a whole row
  for (int i = lane + real * 8; i < kBlock * 8; i += 32) {
    *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(tile + kPanel + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  // First a look, without a branch (with one a word: 16 causal prompts 80 us
  // instead of 68).  An exponent of ones, and only that, carries into the
  // sign's place when its lowest bit is added.
  const auto carries = [](uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; };
  uint32_t found = 0;
#pragma unroll 4
  for (int i = lane + max(0, first) * 8; i < real * 8; i += 32) {
    const uint4 x = *reinterpret_cast<const uint4*>(tile + i * 16);
    const uint4 y = *reinterpret_cast<const uint4*>(tile + kPanel + i * 16);
    found |= carries(x.x) | carries(x.y) | carries(x.z) | carries(x.w) | carries(y.x) | carries(y.y) |
             carries(y.z) | carries(y.w);
  }
  if (__any_sync(0xffffffffu, (found & 0x80008000u) != 0)) {
    for (int i = lane + max(0, first) * 8; i < real * 8; i += 32) {
      bool here = false;
      for (int p = 0; p < 8; ++p) {
        uint32_t* at = reinterpret_cast<uint32_t*>(tile + (p & 4 ? kPanel : 0) + i * 16) + (p & 3);
        const uint32_t bad = carries(*at) & 0x80008000u;
        if (bad == 0) continue;
        here = true;
        *at &= ~(bad | (bad - (bad >> 15)));     // 0xffff for each half that carries
      }
      const int h = i / 8 - first;
      if (here && h < 32 * kHiddenWords) atomicOr(odd + h / 32, 1u << (h & 31));   // past them: hidden from all
    }
  }
  fence_proxy_async_smem();
}

// The zeroed elements' part of the results: a warp adds p_j v_j of the keys j in
// `odd` (word w in lane w) to its 32 rows (a row's query sees keys [0, limit);
// the row's limit, stabiliser m and the factor of its results are in the lane of
// its number), for the elements that are not finite; the others went through
// the tensor cores.  A row that sees none of those keys is not touched.  `own`
// >= 0: keys of blocks own, own + 2, ... only.  The rows' results (float32
// `part`, or bf16 a.out) have been written by this warp; lane owns 4 features.
static __device__ __noinline__ void add_not_finite(const PackedArgs& a, uint32_t odd, int64_t q0,
                                                   int64_t k0, int head, int row0, int own, int first,
                                                   int limit, float m, float factor, float* part) {
  const int lane = threadIdx.x & 31;
  const float c = a.scale * attn::kLog2e;
  for (int x = 0; x < 32; ++x) {
    const int end = __shfl_sync(0xffffffffu, limit, x);
    const float m_row = __shfl_sync(0xffffffffu, m, x), f = __shfl_sync(0xffffffffu, factor, x);
    if (end <= first) continue;
    const int64_t q_row = q0 + (row0 + x) / a.group;
    const int h = head * a.group + (row0 + x) % a.group;
    const __nv_bfloat16* q = a.q + q_row * a.q_stride_t + h * a.q_stride_h + lane * 4;
    float add[4] = {0.f, 0.f, 0.f, 0.f};
    bool open = true;                              // an element that is not NaN yet
    for (int w = 0; w < kHiddenWords && open; ++w) {
      for (uint32_t bits = __shfl_sync(0xffffffffu, odd, w); bits != 0 && open; bits &= bits - 1) {
        const int j = first + w * 32 + __ffs(bits) - 1;
        if (j >= end) break;
        if (own >= 0 && (j / kBlock & 1) != own) continue;
        const __nv_bfloat16* k = a.k + (k0 + j) * a.k_stride_t + head * a.k_stride_h + lane * 4;
        const __nv_bfloat16* v = a.v + (k0 + j) * a.v_stride_t + head * a.v_stride_h + lane * 4;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(__bfloat162float(q[e]), __bfloat162float(k[e]), s);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        const float p = ex2_approx(fmaf(s, c, m_row == -INFINITY ? 0.f : -m_row));
        bool nan = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float t = __bfloat162float(v[e]);
          if (!(fabsf(t) < INFINITY)) add[e] = fmaf(p, t, add[e]);
          nan = nan && add[e] != add[e];
        }
        open = __any_sync(0xffffffffu, !nan);
      }
    }
    const int64_t at = (q_row * a.heads + h) * kHeadDim + lane * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (fabsf(add[e]) < INFINITY) continue;      // nothing was added
      if (part != nullptr)
        part[at + e] += add[e] * f;
      else
        a.out[at + e] = __float2bfloat16_rn(__bfloat162float(a.out[at + e]) + add[e] * f);
    }
  }
}

}  // namespace packed
}  // namespace bsa
