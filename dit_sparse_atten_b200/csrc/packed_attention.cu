// Attention over packed sequences where the query tiles alone leave SMs idle
// (a few new tokens over long keys): the keys of a tile are split over CTAs and
// joined.  The operator's definition and the larger form are in
// packed_attention_tiles.cu.
//
// One CTA takes one part of the key blocks of the 128 / G tokens x G heads of
// one key head, as the 128 rows of the MMA (row = token * G + head in group):
// all query heads that share a key head share its K and V loads, and a single
// new token still fills G rows.  Bound: HBM, K and V read once.
//   warp 8      TMA producer: K/V blocks of 128 keys into a ring of 32 KB
//               slots (K0, K1, V0, K2, V1, ...)
//   warp 9      TMEM owner; one thread loads Q and issues S_j = Q K_j^T
//   warp 10     one thread issues O += P_j V_j (P from tensor memory)
//   warp 11     cleans V of the masked blocks (clean_masked_values)
//   warps 0-7   softmax, two groups that take alternate key blocks, one row a
//               thread, log2 domain, a stabiliser that moves only past 2^8
// TMEM: three S (and P) buffers at [0, 384), O at [384, 512).
// Every mbarrier wait is bounded (bsa::mbar_wait); on a timeout the CTA sets
// kErrWaitTimeout, drains its copies and MMAs, frees TMEM and exits.
#include <algorithm>
#include <atomic>

#include "packed_attention.cuh"

namespace bsa {
namespace {

using namespace attn;
using namespace packed;

constexpr int kThreads = 384;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kPvWarp = 10;
constexpr int kCheckWarp = 11;
constexpr int kSBuffers = 3;
constexpr uint32_t kTmemO = 384;
constexpr int kSlots = 6;
constexpr int kQOff = 0;
constexpr int kRingOff = kQOff + 128 * 256;
constexpr int kXOff = kRingOff + kSlots * kSlotBytes;
constexpr int kBarOff = kXOff + 2 * 2 * 128 * 4;

struct Barriers {
  uint64_t q_full;
  uint64_t s_full[kSBuffers];
  uint64_t p_full[kSBuffers];
  uint64_t m_full[2];
  uint64_t o_done[kSBuffers];
  uint64_t drain[2];
  uint64_t masked_full[2];              // V of the masked blocks, before warp 11
  uint64_t slot_full[kSlots];
  uint64_t slot_empty[kSlots];
  uint32_t tmem_base;
  int abort;
  int exact_rows;                       // warp 11: recompute the rows key by key
};
constexpr int kUsed = kBarOff + static_cast<int>(sizeof(Barriers));

// Leaves O (relative to its stabiliser), the stabiliser and the sum of part
// `split` in the workspace for combine_kernel.
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_split_kernel(const __grid_constant__ CUtensorMap tm_q,
                            const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v, const PackedArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem + kQOff;
  uint8_t* sRing = smem + kRingOff;
  float* sX = reinterpret_cast<float*>(smem + kXOff);
  Barriers* bar = reinterpret_cast<Barriers*>(smem + kBarOff);
  volatile int* abort_flag = &bar->abort;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t slot = a.slots - 1 - blockIdx.x % a.slots;
  const int hk = static_cast<int>((blockIdx.x / a.slots) % a.kv_heads);
  const int split = static_cast<int>(blockIdx.x / (a.slots * a.kv_heads));
  const Work w = find_work(a, slot, a.tile_tokens);
  if (w.tokens == 0) return;
  const int G = a.group;
  const int all = (row_limit(w, w.tokens - 1, a.causal) + kBlock - 1) / kBlock;
  const int block0 = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
  const int n = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits) - block0;
  // The first block of this CTA that some row of the tile does not see whole.
  const int masked_from = max(0, min(n, max(0, row_limit(w, 0, a.causal)) / kBlock - block0));

  if (threadIdx.x == 0) {
    uint32_t dyn_bytes;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    const bool fits = (smem - smem_raw) + kUsed <= static_cast<int>(dyn_bytes);
    mbar_init(&bar->q_full, 1);
    for (int i = 0; i < kSBuffers; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_full[i], 128);
      mbar_init(&bar->o_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->m_full[i], 128);
      mbar_init(&bar->drain[i], 1);
      mbar_init(&bar->masked_full[i], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar->slot_full[s], 1);
      mbar_init(&bar->slot_empty[s], 1);
    }
    bar->exact_rows = 0;
    bar->abort = (prior_timeout(a.err_word) || !fits) ? 1 : 0;
    if (!fits) atomicOr(a.err_word, kErrSmemLayout);
    fence_mbar_init();
  }
  __syncthreads();
  if (bar->abort) return;  // uniform: set before the barrier, read after it
  if (warp == kMmaWarp) tmem_alloc(&bar->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;

  // Load sequence: K0, then K_{j+1}, V_j for every j.
  auto seq_k = [](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto seq_v = [n](int j) { return j + 1 < n ? 2 * j + 2 : 2 * j + 1; };

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    if (lane == 0 && n > 0) {
      uint32_t armed = 0, armed_phase = 0;
      int masked = 0;            // masked V blocks loaded
      bool ok = true;
      auto load = [&](const CUtensorMap* tm, int seq, int j, bool is_v) {
        const int s = seq % kSlots;
        const uint32_t ph = (seq / kSlots) & 1;
        if (!mbar_wait(&bar->slot_empty[s], ph ^ 1, abort_flag, a.err_word)) return false;
        uint8_t* dst = sRing + s * kSlotBytes;
        uint64_t* full = &bar->slot_full[s];
        if (is_v && j >= masked_from) {
          full = &bar->masked_full[masked++];     // at most two: the limits of a tile's rows
                                                  // span at most 127 keys
          armed &= ~(1u << s);   // an earlier load of this slot has long been consumed
        } else {
          armed |= 1u << s;
          armed_phase = (armed_phase & ~(1u << s)) | (ph << s);
        }
        const int row = static_cast<int>(w.k0 + static_cast<int64_t>(block0 + j) * kBlock);
        mbar_arrive_expect_tx(full, kSlotBytes);
        tma_load_3d(dst, tm, full, 0, hk, row);
        tma_load_3d(dst + kPanel, tm, full, 64, hk, row);
        return true;
      };
      ok = load(&tm_k, 0, 0, false);
      for (int j = 0; ok && j < n; ++j) {
        if (j + 1 < n) ok = load(&tm_k, seq_k(j + 1), j + 1, false);
        if (ok) ok = load(&tm_v, seq_v(j), j, true);
      }
      // Never leave a copy in flight into shared memory.
      int never = 0;
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (armed & (1u << s))
          mbar_wait(&bar->slot_full[s], (armed_phase >> s) & 1u, &never, a.err_word);
      for (int i = 0; i < masked; ++i) mbar_wait(&bar->masked_full[i], 0, &never, a.err_word);
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0 && n > 0) {
      const uint32_t idesc = idesc_bf16_f32(128, kBlock, false);
      const uint64_t kdesc0 = sdesc_sw128(smem_u32(sRing), 16, 1024);
      const uint64_t qdesc0 = sdesc_sw128(smem_u32(sQ), 16, 1024);
      // Rows past tile_tokens * G keep whatever the shared memory held: a row
      // of garbage reaches only its own row of S and O, which is not stored.
      mbar_arrive_expect_tx(&bar->q_full, static_cast<uint32_t>(a.tile_tokens * G) * 256u);
      tma_load_3d(sQ, &tm_q, &bar->q_full, 0, hk * G, static_cast<int>(w.q0));
      tma_load_3d(sQ + 16384, &tm_q, &bar->q_full, 64, hk * G, static_cast<int>(w.q0));
      int never = 0;
      bool ok = mbar_wait(&bar->q_full, 0, &never, a.err_word);
      for (int j = 0; ok && j < n; ++j) {
        const int sq = seq_k(j);
        const int s = sq % kSlots;
        ok = mbar_wait(&bar->slot_full[s], (sq / kSlots) & 1, abort_flag, a.err_word);
        // S_j overwrites P_{j-3} (same TMEM buffer): PV_{j-3} must be done.
        const int sb = j % kSBuffers;
        if (ok && j >= kSBuffers)
          ok = mbar_wait(&bar->o_done[sb], ((j - kSBuffers) / kSBuffers) & 1, abort_flag,
                         a.err_word);
        if (!ok) break;
        tc_fence_after();
        const uint64_t kd = kdesc0 + static_cast<uint64_t>((s * kSlotBytes) >> 4);
#pragma unroll
        for (int kk = 0; kk < kHeadDim / 16; ++kk) {
          const uint64_t db = kd + static_cast<uint64_t>(((kk >> 2) * kPanel + (kk & 3) * 32) >> 4);
          const uint64_t da = qdesc0 + static_cast<uint64_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
          umma_bf16_ss(tmem + sb * 128, da, db, idesc, kk > 0 ? 1u : 0u);
        }
        umma_commit(&bar->s_full[sb]);
        umma_commit(&bar->slot_empty[s]);
      }
      umma_commit(&bar->drain[0]);
      mbar_wait(&bar->drain[0], 0, &never, a.err_word);
    }
  } else if (warp == kPvWarp) {
    if (lane == 0 && n > 0) {
      const uint32_t idesc = idesc_bf16_f32(128, kHeadDim, true);
      const uint64_t vdesc0 = sdesc_sw128(smem_u32(sRing), kPanel, 1024);
      bool ok = true;
      for (int j = 0; ok && j < n; ++j) {
        const int sq = seq_v(j);
        const int s = sq % kSlots;
        ok = mbar_wait(&bar->slot_full[s], (sq / kSlots) & 1, abort_flag, a.err_word);
        const int sb = j % kSBuffers;
        if (ok) ok = mbar_wait(&bar->p_full[sb], (j / kSBuffers) & 1, abort_flag, a.err_word);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = vdesc0 + static_cast<uint64_t>((s * kSlotBytes) >> 4);
#pragma unroll
        for (int kk = 0; kk < kBlock / 16; ++kk)
          umma_bf16_ts(tmem + kTmemO, tmem + sb * 128 + kk * 8,
                       vd + static_cast<uint64_t>((kk * 16 * 128) >> 4), idesc,
                       (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&bar->o_done[sb]);
        umma_commit(&bar->slot_empty[s]);
      }
      int never = 0;
      umma_commit(&bar->drain[1]);
      mbar_wait(&bar->drain[1], 0, &never, a.err_word);
    }
  } else if (warp == kCheckWarp) {
    // ------------------------------------------------------ masked V blocks
    for (int j = masked_from; j < n; ++j) {
      const bool ok = mbar_wait(&bar->masked_full[j - masked_from], 0, abort_flag, a.err_word);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int s = seq_v(j) % kSlots;
      const int key0 = (block0 + j) * kBlock;
      if (clean_masked_values(sRing + s * kSlotBytes, max(0, row_limit(w, 0, a.causal) - key0),
                              min(kBlock, w.keys - key0)) &&
          lane == 0)
        *reinterpret_cast<volatile int*>(&bar->exact_rows) = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->slot_full[s]);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int grp = warp >> 2;
    const int wq = warp & 3;
    const int row = wq * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t pair_barrier = 1 + wq;
    const int token = row / G;
    const bool row_valid = token < w.tokens;
    const bool warp_active = wq * 32 < w.tokens * G;
    const int limit = row_limit(w, token, a.causal);

    float* m_buf = sX;
    const float c = a.scale * kLog2e;
    const float2 c2 = make_float2(c, c);
    float m_mine = -INFINITY;
    float l = 0.f;
    bool ok = true;
    for (int j = grp; ok && j < n; j += 2) {
      const int sb = j % kSBuffers;
      ok = mbar_wait(&bar->s_full[sb], (j / kSBuffers) & 1, abort_flag, a.err_word);
      if (!ok) break;
      tc_fence_after();
      const uint32_t sbuf = tmem + lane_addr + sb * 128;
      const bool partial = j >= masked_from;
      const int64_t valid = limit - (block0 + j) * kBlock;
      uint32_t keep[kKeptChunks<128>][32];
      const float mrow = warp_active ? row_max<128>(sbuf, partial, valid, keep) * c : -INFINITY;
      float m_prev = -INFINITY;
      if (j > 0) {
        ok = mbar_wait(&bar->m_full[(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, a.err_word);
        if (!ok) break;
        m_prev = m_buf[((j - 1) & 1) * 128 + row];
      }
      const bool need = mrow > m_prev + kRescaleThreshold;
      const float m_used = need ? mrow : m_prev;
      m_buf[(j & 1) * 128 + row] = m_used;
      mbar_arrive(&bar->m_full[j & 1]);
      if (warp_active) {
        // -inf stands for "no key yet": the sum is 0 and the row's exponents
        // (all -inf) are taken against 0.
        l = m_mine == -INFINITY ? 0.f : l * ex2_approx(m_mine - m_used);
        m_mine = m_used;
        const float neg = m_used == -INFINITY ? 0.f : -m_used;
        const float2 rs =
            row_exp<128, 0>(sbuf, partial, valid, c2, make_float2(neg, neg), keep);
        l += rs.x + rs.y;
      }
      if (j > 0 && __any_sync(0xffffffffu, need)) {
        ok = mbar_wait(&bar->o_done[(j - 1) % kSBuffers], ((j - 1) / kSBuffers) & 1, abort_flag,
                       a.err_word);
        if (!ok) break;
        tc_fence_after();
        if (warp_active) {
          const float p_scale = need ? ex2_approx(m_prev - m_used) : 1.f;
#pragma unroll 1
          for (int cc = 0; cc < kHeadDim / 32; ++cc) {
            uint32_t o[32];
            const uint32_t addr = tmem + lane_addr + kTmemO + cc * 32;
            tmem_ld_32x32b_x32(addr, o);
            tmem_wait_ld();
            reg_fence<32>(o);
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * p_scale);
            tmem_st_32x32b_x32(addr, o);
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar->p_full[sb]);
    }
    // ---------------------------------------------------------- epilogue
    float* xs = sX;
    named_bar_sync(pair_barrier, 64);
    xs[grp * 128 + row] = m_mine;
    xs[256 + grp * 128 + row] = l;
    named_bar_sync(pair_barrier, 64);
    const float m0 = xs[row], m1 = xs[128 + row];
    const float m_fin = fmaxf(m0, m1);
    float l_row = 0.f;
    if (m0 != -INFINITY) l_row += xs[256 + row] * ex2_approx(m0 - m_fin);
    if (m1 != -INFINITY) l_row += xs[384 + row] * ex2_approx(m1 - m_fin);
    if (ok && n > 0) {
      ok = mbar_wait(&bar->drain[1], 0, abort_flag, a.err_word);
      tc_fence_after();
    }
    const int head0 = hk * G;
    if (ok && n > 0 && *reinterpret_cast<volatile int*>(&bar->exact_rows)) {
      for (int r = warp; r < w.tokens * G; r += 8) {
        const int t = r / G, h = head0 + r % G;
        const int end = min(row_limit(w, t, a.causal), (block0 + n) * kBlock);
        float4 o;
        const float2 ml = exact_row(a, a.q + (w.q0 + t) * a.q_stride_t + h * a.q_stride_h, w.k0,
                                    hk, block0 * kBlock, end, c, o);
        const int64_t p = (split * a.q_rows + w.q0 + t) * a.heads + h;
        *reinterpret_cast<float4*>(a.part_o + p * kHeadDim + lane * 4) = o;
        if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = ml;
      }
    } else if (warp_active) {
      const int64_t p = (split * a.q_rows + w.q0 + token) * a.heads + head0 + (row - token * G);
#pragma unroll 1
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t o[32];
        if (ok && n > 0) {
          tmem_ld_32x32b_x32(tmem + lane_addr + kTmemO + grp * 64 + cc * 32, o);
          tmem_wait_ld();
          reg_fence<32>(o);
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0u;
        }
        if (!row_valid) continue;
        float4* dst = reinterpret_cast<float4*>(a.part_o + p * kHeadDim + grp * 64 + cc * 32);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          dst[x] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                               __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
      }
      if (row_valid && grp == 0)
        *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m_fin, l_row);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a split row: out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p -
// m) l_p, parts in order.  One warp a (query row, head).
__global__ void __launch_bounds__(256) combine_kernel(const PackedArgs a) {
  const int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int64_t rows = a.q_rows * a.heads;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY;
  for (int p = 0; p < a.splits; ++p) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (p * rows + row));
    if (ml.y != 0.f) m = fmaxf(m, ml.x);
  }
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p < a.splits; ++p) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (p * rows + row));
    if (ml.y == 0.f) continue;
    const float f = ex2_approx(ml.x - m);
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + (p * rows + row) * kHeadDim + lane * 4);
    l += ml.y * f;
    o.x = fmaf(v.x, f, o.x);
    o.y = fmaf(v.y, f, o.y);
    o.z = fmaf(v.z, f, o.z);
    o.w = fmaf(v.w, f, o.w);
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint2*>(a.out + row * kHeadDim + lane * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

cudaError_t launch_parts(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                         const PackedArgs& a, cudaStream_t stream) {
  static std::atomic<int> smem_bytes[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int bytes = (dev >= 0 && dev < 64) ? smem_bytes[dev].load(std::memory_order_acquire) : 0;
  if (bytes == 0) {
    int optin = 0;
    e = cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e != cudaSuccess) return e;
    bytes = optin < kUsed + 1024 ? optin : kUsed + 1024;
    if (bytes < kUsed) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(packed_attention_split_kernel,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) smem_bytes[dev].store(bytes, std::memory_order_release);
  }
  const int64_t grid = a.slots * a.kv_heads * a.splits;
  packed_attention_split_kernel<<<static_cast<unsigned>(grid), kThreads, bytes, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

}  // namespace

// Parts of a tile's keys: one where the tiles alone give every SM two CTAs;
// otherwise enough for four a SM, of 512 keys at least on the average request.
int32_t packed_splits(int64_t q_rows, int64_t k_rows, int32_t requests, int32_t heads,
                      int32_t kv_heads, int num_sms) {
  const int64_t ctas = (q_rows / (128 / (heads / kv_heads)) + requests) * kv_heads;
  if (ctas >= 2 * num_sms) return 1;
  const int64_t splits = std::min((4 * num_sms + ctas - 1) / ctas, k_rows / requests / 512);
  return static_cast<int32_t>(std::max<int64_t>(1, splits));
}

cudaError_t launch_packed_attention(const CUtensorMap& tq, const CUtensorMap& tk,
                                    const CUtensorMap& tv, const PackedArgs& a,
                                    cudaStream_t stream) {
  if (a.splits == 1) return launch_packed_tiles(tq, tk, tv, a, stream);
  const cudaError_t e = launch_parts(tq, tk, tv, a, stream);
  if (e != cudaSuccess) return e;
  const int64_t rows = a.q_rows * a.heads;
  combine_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace bsa
