// Softmax attention over packed sequences of different lengths, grouped heads,
// causal or full, for sm_100a:
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h / G]) v[j, h / G]
// over the keys j of query i's own request (causal: the first
// i + 1 + k_len - q_len of them, i counted within the request), in float32
// from bf16 inputs; a query that sees no key gives 0.
//
// One CTA takes the 128 / G tokens x G heads of one key head as the 128 rows
// of the MMA (row = token * G + head in group), so all query heads that share
// a key head share its K and V loads, and a single new token still fills G
// rows.  Tiles are found on the device: slot g belongs to request
// s = #{i >= 1: floor(q_starts[i] / tokens) + i <= g} (packed_common.cuh).
// Tiles late in their request see the most keys under the causal mask, so
// slots run from the last to the first; a key head's tiles run next to each
// other so that its K and V stay in L2.
//   warp 8      TMA producer: K/V blocks of 128 keys into a ring of 32 KB
//               slots (K0, K1, V0, K2, V1, ...)
//   warp 9      TMEM owner; one thread loads Q and issues S_j = Q K_j^T
//   warp 10     one thread issues O += P_j V_j (P from tensor memory)
//   warp 11     V of the masked blocks (the last one or two): rows past the
//               request's end are zeroed, since 0 * (whatever another request
//               holds there, NaN included) would reach O
//   warps 0-7   softmax, two groups that take alternate key blocks, one row a
//               thread, log2 domain, a stabiliser that moves only past 2^8
// TMEM: three S (and P) buffers at [0, 384), O at [384, 512).
//
// A value of V that is not finite at a key which part of the tile must not see
// (causal) cannot be kept out of those rows by P = 0; warp 11 looks for one
// and, if there is, the tile's rows are computed again key by key in float32.
//
// Every mbarrier wait is bounded (bsa::mbar_wait); on a timeout the CTA sets
// kErrWaitTimeout, drains its copies and MMAs, frees TMEM and exits.
#include <atomic>

#include "attention_softmax.cuh"
#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace {

using namespace attn;

constexpr int kThreads = 384;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kPvWarp = 10;
constexpr int kCheckWarp = 11;
constexpr int kHeadDim = 128;
constexpr int kBlock = 128;             // keys a block
constexpr int kSBuffers = 3;
constexpr uint32_t kTmemO = 384;
constexpr int kSlots = 6;
constexpr int kPanel = kBlock * 128;    // 64 columns x 128 rows, bf16
constexpr int kSlotBytes = 2 * kPanel;
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

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

// What a CTA works on (uniform over the CTA).
struct Work {
  int64_t q0;          // first query row
  int64_t k0;          // first key row of the request
  int tokens;          // queries of the tile (0: nothing to do)
  int first_limit;     // keys that the tile's first query sees, before clamping to [0, keys]
  int keys;            // keys of the request
  int block0, blocks;  // key blocks [block0, block0 + blocks)
};

// Query row `token` of the tile sees keys [0, limit).
__device__ __forceinline__ int row_limit(const Work& w, int token, bool causal) {
  if (token >= w.tokens) return 0;
  return causal ? max(0, min(w.keys, w.first_limit + token)) : w.keys;
}

__device__ __forceinline__ Work find_work(const PackedArgs& a, int64_t slot, int split) {
  Work w{};
  const int tt = a.tile_tokens;
  const int s = warp_count_le(a.requests, slot, [&](int i) {
    return static_cast<int64_t>(__ldg(a.q_starts + i)) / tt + i;
  });
  if (s >= a.requests) return w;
  const int64_t qb = __ldg(a.q_starts + s), qe = __ldg(a.q_starts + s + 1);
  const int64_t kb = __ldg(a.k_starts + s), ke = __ldg(a.k_starts + s + 1);
  const bool bad = qb < 0 || qe < qb || qe > a.q_rows || kb < 0 || ke < kb || ke > a.k_rows ||
                   (s == 0 && qb != 0) || (s == a.requests - 1 && qe != a.q_rows);
  if (bad && threadIdx.x == 0) atomicOr(a.err_word, kErrBadRoute);
  if (qb < 0 || qe > a.q_rows || kb < 0 || ke < kb || ke > a.k_rows) return w;
  w.q0 = qb + (slot - (qb / tt + s)) * tt;
  if (w.q0 < qb || w.q0 >= qe) return w;
  w.k0 = kb;
  w.tokens = static_cast<int>(min(static_cast<int64_t>(tt), qe - w.q0));
  w.keys = static_cast<int>(ke - kb);
  // int: |q_rows|, |k_rows| < 2^31 - 256
  w.first_limit = a.causal ? static_cast<int>(w.q0 - qb + 1 + (ke - kb) - (qe - qb)) : w.keys;
  const int visible = row_limit(w, w.tokens - 1, a.causal);
  const int n = (visible + kBlock - 1) / kBlock;
  w.block0 = static_cast<int>(static_cast<int64_t>(n) * split / a.splits);
  w.blocks = static_cast<int>(static_cast<int64_t>(n) * (split + 1) / a.splits) - w.block0;
  return w;
}

// One query row key by key in float32 (a warp; lane owns 4 features): the way
// out when V holds non-finite values at masked keys.  Returns the row's
// stabiliser (log2 domain) and sum; o is relative to the stabiliser.
__device__ __noinline__ float2 exact_row(const PackedArgs& a, const __nv_bfloat16* q,
                                         int64_t k0, int head, int begin, int end, float c,
                                         float4& o) {
  const int lane = threadIdx.x & 31;
  float qf[4], m = -INFINITY, l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int e = 0; e < 4; ++e) qf[e] = __bfloat162float(q[lane * 4 + e]);
  for (int j = begin; j < end; ++j) {
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
    const float p = m_new == -INFINITY ? 0.f : ex2_approx(s - m_new);
    l = l * keep + p;
    o.x = fmaf(p, __bfloat162float(v[0]), m == -INFINITY ? 0.f : o.x * keep);
    o.y = fmaf(p, __bfloat162float(v[1]), m == -INFINITY ? 0.f : o.y * keep);
    o.z = fmaf(p, __bfloat162float(v[2]), m == -INFINITY ? 0.f : o.z * keep);
    o.w = fmaf(p, __bfloat162float(v[3]), m == -INFINITY ? 0.f : o.w * keep);
    m = m_new;
  }
  return make_float2(m, l);
}

// kSplit: this CTA takes one of a.splits parts of the tile's key blocks and
// leaves O (relative to its stabiliser), the stabiliser and the sum in the
// workspace for combine_kernel.
template <bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tm_q,
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
  const int split = kSplit ? static_cast<int>(blockIdx.x / (a.slots * a.kv_heads)) : 0;
  const Work w = find_work(a, slot, split);
  if (w.tokens == 0) return;
  const int G = a.group;
  const int n = w.blocks;
  // The first block of this CTA that some row of the tile does not see whole.
  const int masked_from = max(0, min(n, max(0, row_limit(w, 0, a.causal)) / kBlock - w.block0));

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
        const int row = static_cast<int>(w.k0 + static_cast<int64_t>(w.block0 + j) * kBlock);
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
      uint8_t* tile = sRing + s * kSlotBytes;
      const int key0 = (w.block0 + j) * kBlock;
      const int real = min(kBlock, w.keys - key0);                    // rows of this request
      const int open = max(0, row_limit(w, 0, a.causal) - key0);      // rows that every query sees
      for (int i = lane + real * 8; i < kBlock * 8; i += 32) {
        // a row is 8 chunks of 16 bytes in each panel; which of them is which
        // (the swizzle) does not matter for zeroing or scanning a whole row
        *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(tile + kPanel + i * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      bool found = false;
      for (int i = lane + open * 8; i < real * 8; i += 32) {
#pragma unroll
        for (int panel = 0; panel < 2; ++panel) {
          const uint4 x = *reinterpret_cast<const uint4*>(tile + panel * kPanel + i * 16);
          const uint32_t e = 0x7f807f80u, words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int p = 0; p < 4; ++p)
            found |= (words[p] & e & 0xffffu) == (e & 0xffffu) || (words[p] & e) >> 16 == e >> 16;
        }
      }
      if (__any_sync(0xffffffffu, found) && lane == 0)
        *reinterpret_cast<volatile int*>(&bar->exact_rows) = 1;
      fence_proxy_async_smem();
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
      const int64_t valid = limit - (w.block0 + j) * kBlock;
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
        const int end = min(row_limit(w, t, a.causal), (w.block0 + n) * kBlock);
        float4 o;
        const float2 ml = exact_row(a, a.q + (w.q0 + t) * a.q_stride_t + h * a.q_stride_h, w.k0,
                                    hk, w.block0 * kBlock, end, c, o);
        const int64_t at = (w.q0 + t) * a.heads + h;
        if constexpr (kSplit) {
          const int64_t p = split * a.q_rows * a.heads + at;
          *reinterpret_cast<float4*>(a.part_o + p * kHeadDim + lane * 4) = o;
          if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = ml;
        } else {
          const float inv = ml.y != 0.f ? 1.f / ml.y : 0.f;
          *reinterpret_cast<uint2*>(a.out + at * kHeadDim + lane * 4) =
              make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        }
      }
    } else if (warp_active) {
      const int64_t at = (w.q0 + token) * a.heads + head0 + (row - token * G);
      const int64_t p = split * a.q_rows * a.heads + at;
      const float inv_l = kSplit ? 1.f : l_row != 0.f ? 1.f / l_row : 0.f;
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
        if constexpr (kSplit) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + p * kHeadDim + grp * 64 + cc * 32);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            dst[x] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                                 __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.out + at * kHeadDim + grp * 64 + cc * 32);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            dst[x] = make_uint4(
                pack_bf16x2(__uint_as_float(o[8 * x]) * inv_l, __uint_as_float(o[8 * x + 1]) * inv_l),
                pack_bf16x2(__uint_as_float(o[8 * x + 2]) * inv_l, __uint_as_float(o[8 * x + 3]) * inv_l),
                pack_bf16x2(__uint_as_float(o[8 * x + 4]) * inv_l, __uint_as_float(o[8 * x + 5]) * inv_l),
                pack_bf16x2(__uint_as_float(o[8 * x + 6]) * inv_l, __uint_as_float(o[8 * x + 7]) * inv_l));
        }
      }
      if constexpr (kSplit) {
        if (row_valid && grp == 0)
          *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m_fin, l_row);
      }
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

template <bool kSplit>
cudaError_t launch_main(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
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
    e = cudaFuncSetAttribute(packed_attention_kernel<kSplit>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) smem_bytes[dev].store(bytes, std::memory_order_release);
  }
  const int64_t grid = a.slots * a.kv_heads * a.splits;
  packed_attention_kernel<kSplit><<<static_cast<unsigned>(grid), kThreads, bytes, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

}  // namespace

// Parts of a tile's keys: one where the tiles alone give every SM two CTAs;
// otherwise enough for four a SM, of 512 keys at least on the average request.
int32_t packed_splits(int64_t q_rows, int64_t k_rows, int32_t requests, int32_t heads,
                      int32_t kv_heads, int num_sms) {
  const int64_t ctas = (q_rows / (128 / (heads / kv_heads)) + requests) * kv_heads;
  if (ctas >= 2 * num_sms) return 1;
  int64_t splits = (4 * num_sms + ctas - 1) / ctas;
  const int64_t most = k_rows / requests / 512;
  splits = splits < most ? splits : most;
  return static_cast<int32_t>(splits < 1 ? 1 : splits);
}

cudaError_t launch_packed_attention(const CUtensorMap& tq, const CUtensorMap& tk,
                                    const CUtensorMap& tv, const PackedArgs& a,
                                    cudaStream_t stream) {
  if (a.splits == 1) return launch_main<false>(tq, tk, tv, a, stream);
  const cudaError_t e = launch_main<true>(tq, tk, tv, a, stream);
  if (e != cudaSuccess) return e;
  const int64_t rows = a.q_rows * a.heads;
  combine_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace bsa
