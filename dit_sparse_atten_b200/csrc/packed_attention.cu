// Softmax attention over packed sequences of different lengths, grouped heads,
// causal or full, for sm_100a:
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h / G]) v[j, h / G]
// over the keys j of query i's own request (causal: the first
// i + 1 + k_len - q_len of them, i counted within the request), in float32
// from bf16 inputs; a query that sees no key gives 0.
//
// An item is 2 x (128 / G tokens) x G heads of one key head: two MMA tiles of
// 128 rows (row = token * G + head in group), so that all query heads of a key
// head, and both tiles, share its K and V loads.  While one tile's softmax
// runs, the tensor pipe works for the other.  CTAs are resident and take their
// next item from the grid's CTAs that have not started (cluster launch
// control), so an item's first loads and S run under the last softmax and the
// store of the item before.  Items are found on the device (packed_common.cuh),
// those late in their request first: under the causal mask they see the most
// keys.
//   warps 0-3, 4-7   softmax of tile 0, 1: 64 keys at a time, one row a thread,
//               log2 domain, a stabiliser that moves only past 2^8 (then O_t is
//               rescaled in TMEM); P is rounded to bf16, the tensor cores'
//               operand, its row sum is taken before the rounding
//   warps 8, 9  MMA issuers, one warp for each tile t: for each 64 keys u,
//               S_t(u + 1) = Q_t K(u + 1)^T, then O_t += P_t(u) V(u); warp 8
//               owns TMEM.  A tile has its own issuer so that it never waits
//               for the other's softmax.
//   warp 10     producer: asks for the next item, looks it up and publishes it;
//               loads Q, and K/V blocks of 128 keys into a ring of 32 KB slots
//               (K0, V0, K1, V1, ...)
//   warp 11     cleans V of the masked blocks (clean_masked_values)
// TMEM: tile t's S (64 columns) at 128 t, its two P buffers (32 columns each)
// behind it, O_t at 256 + 128 t.  P does not lie over S, so S(u + 1) is asked
// for as soon as the softmax has S(u) in registers, and the PV of the keys
// before has the time of a whole softmax; S of more than 64 keys leaves no room
// for two P.  Twelve warps leave a softmax thread 168 registers (thirteen: 128).
//
// Bound: the softmax warps.  64 keys of both tiles take 1,800 cycles: 1,024 of
// exponentials, the rest the latency of loading S, the row maxima and the
// hand-overs, which two warps a scheduler hide only in part; the products take
// 1,250 of tensor pipe (S of 64 keys 390 where 256 would be the full rate: Q is
// read from shared memory for every 64 keys).  Measured: 16,380 causal tokens,
// 16 / 4 heads, 975 to 995 us over several runs, 1,105 to 1,127 TFLOP/s; 21,967
// tokens x 40 heads against prompts of up to 512, 209 to 219 us; 16 causal
// prompts of 4,931 tokens, 68 us.  Earlier forms, in one run where this one took
// 840 / 184 / 69 us back to back: P over S's own columns with two S buffers of 64
// keys 940 / 200 / 71 us, one S of 128 keys 957 / 240 / 108, one issuer for both tiles 1,082 / 282; with
// the next block's S loaded ahead into registers the softmax spills (1,630 us);
// 16 softmax warps, tiles taking turns at the exponentials, and exponentials on
// the FMA pipe were slower too.
//
// Few items: the keys are cut into parts (kSplit), whose O, stabiliser and sum
// combine_kernel joins.  An item of at most one tile's tokens is `paired`:
// both tiles hold its queries and take alternate key blocks, each with a part of
// its own, since one tile's softmax is slower than the loads.  Measured: 16
// requests of one token over 250,000 keys, 40 / 8 heads, 205 to 212 us over
// several runs, 4.3 to 4.4 TB/s (the best: 180 us, 5.05 TB/s).
//
// A value of V that is not finite at a key which part of the item must not see
// (causal) cannot be kept out of those rows by P = 0; warp 11 zeroes such values
// and notes their keys, fewer than 256 an item, and the softmax warps add them
// to the results of the rows that see them (add_not_finite).  The cost does not
// grow with the keys' number: 8,192 causal tokens, 8 / 1 heads, 304 us; with one
// NaN 352, half of the values NaN 433, half of them +inf 1,282 (recomputing the
// item's rows key by key: 7,500 / 25,200 / 26,200).
//
// Every mbarrier wait is bounded (bsa::mbar_wait); on a timeout the CTA sets
// kErrWaitTimeout, drains its copies and MMAs, frees TMEM and exits.
#include <algorithm>
#include <atomic>

#include "packed_attention.cuh"

namespace bsa {
namespace {

using namespace attn;
using namespace packed;

constexpr int kSoftWarps = 8;
constexpr int kThreads = 384;
constexpr int kMmaWarp = 8;             // and 9
constexpr int kProducerWarp = 10;
constexpr int kCheckWarp = 11;
constexpr int kSub = 64;                // keys of S and of a P buffer
constexpr int kLate = 2;                // key blocks left to load of an item when the next is asked for
// Ring slots; parts of keys are bound by HBM and stage no output, which leaves
// room for one more.
constexpr int kMaxSlots = 5;
template <bool kSplit>
constexpr int kSlotsOf = kSplit ? 5 : 4;
constexpr int kMaskedRing = 4;          // masked V blocks between the producer and warp 11
constexpr int kWorkRing = 2;            // an item at work and the next
constexpr int kWorkReaders = kSoftWarps + 3;   // and both issuers, check
constexpr int kQOff = 0;
constexpr int kRingOff = 2 * kSlotBytes;
constexpr int kStageOff = kRingOff + kSlotsOf<false> * kSlotBytes;
constexpr int kStageBytes = 32 * 128;   // of each softmax warp: 64 features of its 32 rows
constexpr int kBarOff = std::max(kStageOff + kSoftWarps * kStageBytes, kRingOff + kSlotsOf<true> * kSlotBytes);

// An item as the scheduler publishes it.
struct Item {
  Work w;              // w.tokens < 0: no more items
  int hk;              // key head
  int n[2];            // 64-key sub-blocks of each tile
  int blocks;          // key blocks of the item
  int paired;          // the tiles hold the same queries, tile t key blocks t, t + 2, ...
  int part;            // of the keys
  uint32_t odd[kHiddenWords];   // hidden keys with values that are not finite; set by warp 11
};

struct Barriers {
  uint64_t q_full, q_empty;
  uint64_t s_full[2], s_empty[2], p_full[2][2], pv_done[2];   // [tile][P buffer]
  uint64_t o_full[2], o_empty[2];
  uint64_t slot_full[kMaxSlots], slot_empty[kMaxSlots];
  uint64_t masked_full[kMaskedRing];    // V of a masked block, before warp 11
  uint64_t work_full[kWorkRing], work_empty[kWorkRing];
  uint64_t next_full;                   // answer of the cluster launch control
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
  Item item[kWorkRing];
  uint4 next __attribute__((aligned(16)));
};
constexpr int kUsed = kBarOff + static_cast<int>(sizeof(Barriers));

// One lane of the (converged) warp, the same every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

// Cluster launch control: ask for a CTA of this grid that has not started to
// be cancelled, its index to be taken over by the caller.
__device__ __forceinline__ void request_next(uint4* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// blockIdx.x of the cancelled CTA, or -1 (all have started).
__device__ __forceinline__ int64_t answered_next(const uint4* answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return ok ? static_cast<int64_t>(x) : -1;
}

// kSplit: items are parts of the keys (take_part); O (relative to its
// stabiliser), the stabiliser and the sum go to the workspace for
// combine_kernel.
template <bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_tiles_kernel(const __grid_constant__ CUtensorMap tm_q,
                                  const __grid_constant__ CUtensorMap tm_k,
                                  const __grid_constant__ CUtensorMap tm_v, const PackedArgs a) {
  constexpr int kSlots = kSlotsOf<kSplit>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem + kQOff;
  uint8_t* sRing = smem + kRingOff;
  Barriers* bar = reinterpret_cast<Barriers*>(smem + kBarOff);
  volatile int* abort_flag = &bar->abort;

  // shuffled, so that the compiler knows it uniform over the warp
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int G = a.group;
  const int tt = a.tile_tokens;

  if (threadIdx.x == 0) {
    uint32_t dyn_bytes;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    const bool fits = (smem - smem_raw) + kUsed <= static_cast<int>(dyn_bytes);
    bar->abort = (prior_timeout(a.err_word) || !fits) ? 1 : 0;
    if (!fits) atomicOr(a.err_word, kErrSmemLayout);
    mbar_init(&bar->q_full, 1);
    mbar_init(&bar->q_empty, 2);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bar->s_full[t], 1);
      mbar_init(&bar->s_empty[t], 128);
      for (int b = 0; b < 2; ++b) mbar_init(&bar->p_full[t][b], 128);
      mbar_init(&bar->pv_done[t], 1);
      mbar_init(&bar->o_full[t], 1);
      mbar_init(&bar->o_empty[t], 128);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar->slot_full[s], 1);
      mbar_init(&bar->slot_empty[s], 2);
    }
    for (int i = 0; i < kMaskedRing; ++i) mbar_init(&bar->masked_full[i], 1);
    for (int i = 0; i < kWorkRing; ++i) {
      mbar_init(&bar->work_full[i], 1);
      mbar_init(&bar->work_empty[i], kWorkReaders);
    }
    mbar_init(&bar->next_full, 1);
    for (int t = 0; t < 2; ++t) mbar_init(&bar->drain[t], 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (bar->abort) return;  // uniform: set before the barrier, read after it
  if (warp == kMmaWarp) tmem_alloc(&bar->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;

  // Item number i of this CTA, or null (no more, or aborting).
  auto item_at = [&](int i) -> Item* {
    const int r = i % kWorkRing;
    if (!mbar_wait(&bar->work_full[r], (i / kWorkRing) & 1, abort_flag, a.err_word)) return nullptr;
    Item* it = &bar->item[r];
    return it->w.tokens < 0 ? nullptr : it;
  };
  auto done_with = [&](int i) { mbar_arrive(&bar->work_empty[i % kWorkRing]); };
  // First block of the item that some row of tile t does not see whole.
  auto masked_from = [&](const Work& w, int t) { return row_limit(w, t * tt, a.causal) / kBlock; };

  // Key blocks of an item: both tiles'.
  auto item_blocks = [&](const Item* it) { return it->blocks; };

  if (warp >= kSoftWarps) {
   if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    // The next item is asked for when an item's loads come to their last
    // blocks: asked for earlier, it would wait here while other CTAs run out
    // of work.
    int64_t cta = blockIdx.x;
    uint32_t asked = 0, answers = 0, armed = 0, armed_phase = 0;
    int seq = 0, masked = 0, loads = 0;        // of K/V, of masked V, of Q
    bool ok = true;
    for (int i = 0; ok;) {
      Item it{};
      it.w.tokens = -1;
      if (cta >= 0) {
        // late slots first; a key head's items next to each other
        it.hk = static_cast<int>(cta % a.kv_heads);
        const int64_t rest = cta / a.kv_heads;
        it.w = find_work(a, a.slots - 1 - rest % a.slots, 2 * tt);
        if constexpr (kSplit) {
          it.part = static_cast<int>(rest / a.slots);
          take_part(it.w, it.part, a);
        }
      }
      const Work& w = it.w;
      if (w.tokens != 0) {
        it.blocks = packed::item_blocks(w, a.causal);
        it.paired = kSplit && w.tokens > 0 && w.tokens <= tt;
        for (int t = 0; t < 2; ++t) {
          const int last = min(w.tokens, it.paired ? tt : (t + 1) * tt) - 1;
          const int keys = row_limit(w, last, a.causal);
          if (!it.paired) {
            it.n[t] = last < t * tt ? 0 : (keys + kSub - 1) / kSub;
          } else {
            const int before = (it.blocks - t - 1) / 2;       // blocks before this tile's last
            it.n[t] = it.blocks <= t ? 0 : 2 * before + min(2, (keys - (2 * before + t) * kBlock + kSub - 1) / kSub);
          }
        }
        if (lane == 0) {
          const int r = i % kWorkRing;
          ok = mbar_wait(&bar->work_empty[r], ((i / kWorkRing) & 1) ^ 1, abort_flag, a.err_word);
          if (ok) {
            bar->item[r] = it;
            mbar_arrive(&bar->work_full[r]);
          }
        }
        ++i;
      }
      if (cta < 0) break;
      if (lane == 0 && ok) {
        const int n = w.tokens == 0 ? 0 : item_blocks(&it);
        const int from = masked_from(w, 0);
        auto ask = [&] {
          mbar_arrive_expect_tx(&bar->next_full, 16);
          request_next(&bar->next, &bar->next_full);
          ++asked;
        };
        auto load = [&](const CUtensorMap* tm, int j, bool is_v) {
          const int s = seq % kSlots;
          const uint32_t ph = (seq / kSlots) & 1;
          if (!mbar_wait(&bar->slot_empty[s], ph ^ 1, abort_flag, a.err_word)) return false;
          uint8_t* dst = sRing + s * kSlotBytes;
          uint64_t* full = &bar->slot_full[s];
          if (is_v && j >= from) {
            full = &bar->masked_full[masked++ % kMaskedRing];
            armed &= ~(1u << s);   // an earlier load of this slot has long been consumed
          } else {
            armed |= 1u << s;
            armed_phase = (armed_phase & ~(1u << s)) | (ph << s);
          }
          const int row = static_cast<int>(w.k0 + static_cast<int64_t>(j) * kBlock);
          mbar_arrive_expect_tx(full, kSlotBytes);
          tma_load_3d(dst, tm, full, 0, it.hk, row);
          tma_load_3d(dst + kPanel, tm, full, 64, it.hk, row);
          ++seq;
          return true;
        };
        if (n <= kLate) ask();
        if (n > 0) {
          ok = load(&tm_k, 0, false);
          if (ok) ok = mbar_wait(&bar->q_empty, (loads & 1) ^ 1, abort_flag, a.err_word);
          if (ok) {
            // Rows past tt * G keep whatever the shared memory held: a row of
            // garbage reaches only its own row of S and O, which is not stored.
            mbar_arrive_expect_tx(&bar->q_full, static_cast<uint32_t>(tt * G) * 512u);
            for (int t = 0; t < 2; ++t)
              for (int p = 0; p < 2; ++p)
                tma_load_3d(sQ + t * kSlotBytes + p * kPanel, &tm_q, &bar->q_full, p * 64, it.hk * G,
                            static_cast<int>(w.q0) + (it.paired ? 0 : t * tt));
            ++loads;
          }
        }
        for (int j = 0; ok && j < n; ++j) {
          if (n > kLate && j == n - kLate) ask();
          if (j > 0) ok = load(&tm_k, j, false);
          if (ok) ok = load(&tm_v, j, true);
        }
        if (ok) ok = mbar_wait(&bar->next_full, answers & 1, abort_flag, a.err_word);
        if (ok) ++answers;
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      cta = answered_next(&bar->next);
      fence_proxy_async_smem();     // the answer is read before the next one is asked for
      __syncwarp();
    }
    if (lane == 0) {
      // Never leave a copy, or an answer, in flight into shared memory.
      int late = 0;
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (armed & (1u << s))
          mbar_drain(&bar->slot_full[s], (armed_phase >> s) & 1u, &late, a.err_word);
      for (int j = max(0, masked - kMaskedRing); j < masked; ++j)
        mbar_drain(&bar->masked_full[j % kMaskedRing], (j / kMaskedRing) & 1, &late, a.err_word);
      if (loads) mbar_drain(&bar->q_full, (loads - 1) & 1, &late, a.err_word);
      if (asked != answers) mbar_drain(&bar->next_full, answers & 1, &late, a.err_word);
    }
   } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ------------------------------------------------------------ MMA issuers
    {
      const int t = warp - kMmaWarp;
      const uint32_t idesc_s = idesc_bf16_f32(128, kSub, false);
      const uint32_t idesc_o = idesc_bf16_f32(128, kHeadDim, true);
      const uint64_t kdesc0 = sdesc_sw128(smem_u32(sRing), 16, 1024);
      const uint64_t vdesc0 = sdesc_sw128(smem_u32(sRing), kPanel, 1024);
      const uint64_t qdesc = sdesc_sw128(smem_u32(sQ + t * kSlotBytes), 16, 1024);
      const uint32_t s_tmem = tmem + t * 128, o_tmem = tmem + 256 + t * 128;
      int slot = 0, loads = 0;
      uint32_t ring_phase = 0;
      uint32_t scored = 0, used = 0, outs = 0;   // S issued, P consumed, O finished
      bool ok = true;
      // The whole warp goes through the loop, so that the descriptors stay in
      // uniform registers; one elected lane issues.
      auto wait = [&](uint64_t* b, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, a.err_word)) != 0;
      };
      auto commit = [&](uint64_t* b) {
        if (elect_one()) umma_commit(b);
      };
      // Next slot of the ring, once it is full.
      auto next_slot = [&]() -> int {
        const int s = slot;
        ok = wait(&bar->slot_full[s], ring_phase);
        if (++slot == kSlots) slot = 0, ring_phase ^= 1;
        return s;
      };
      // S of keys 64 half .. of the K block in slot s, once the softmax has read
      // the S before.
      auto issue_s = [&](int s, int half) {
        if (!(ok = wait(&bar->s_empty[t], (scored & 1) ^ 1))) return;
        ++scored;
        tc_fence_after();
        const uint64_t kd = kdesc0 + static_cast<uint64_t>((s * kSlotBytes + half * kSub * 128) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kHeadDim / 16; ++kk) {
            const uint64_t off = static_cast<uint64_t>(((kk >> 2) * kPanel + (kk & 3) * 32) >> 4);
            umma_bf16_ss(s_tmem, qdesc + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          umma_commit(&bar->s_full[t]);
        }
        __syncwarp();
      };
      // O += P V for sub-block u, half of the V block in slot s.
      auto issue_pv = [&](int s, int half, int u, bool last) {
        // the first PV of an item overwrites the O that the softmax group stores
        if (u == 0 && !(ok = wait(&bar->o_empty[t], (outs & 1) ^ 1))) return;
        const uint32_t b = used & 1;
        if (!(ok = wait(&bar->p_full[t][b], (used >> 1) & 1))) return;
        ++used;
        tc_fence_after();
        const uint64_t vd = vdesc0 + static_cast<uint64_t>((s * kSlotBytes + half * kSub * 128) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kSub / 16; ++kk)
            umma_bf16_ts(o_tmem, s_tmem + kSub + b * (kSub / 2) + kk * 8,
                         vd + static_cast<uint64_t>((kk * 16 * 128) >> 4), idesc_o, (u > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&bar->pv_done[t]);
          if (last) umma_commit(&bar->o_full[t]);
        }
        __syncwarp();
        if (last) ++outs;
      };
      for (int i = 0; ok; ++i) {
        const Item* it = item_at(i);
        if (!__all_sync(0xffffffffu, it != nullptr)) break;
        const int mine = __shfl_sync(0xffffffffu, it->n[t], 0);         // sub-blocks
        const int n = __shfl_sync(0xffffffffu, item_blocks(it), 0);
        const bool paired = __shfl_sync(0xffffffffu, it->paired, 0) != 0;
        __syncwarp();
        if (elect_one()) done_with(i);
        if (n == 0) continue;
        // Blocks past this tile's last are only passed on (the other tile reads
        // them): the slot is given back once it is full.
        int sk = next_slot();
        if (!ok || !(ok = wait(&bar->q_full, loads & 1))) break;
        ++loads;
        tc_fence_after();
        int u = 0;                             // this tile's next sub-block
        bool own = !paired || t == 0;          // block j is this tile's
        if (own && mine > 0) issue_s(sk, 0);
        if (!ok) break;
        if (mine == 0 || (own && mine == 1)) commit(&bar->q_empty);
        for (int j = 0; j < n; ++j) {
          // sub-block u's PV behind S of the next, whose softmax is first
          if (own && u + 1 < mine) issue_s(sk, 1);
          if (!ok) break;
          commit(&bar->slot_empty[sk]);
          if (own && u + 2 == mine) commit(&bar->q_empty);
          const int sv = next_slot();
          if (!ok) break;
          if (own && u < mine) issue_pv(sv, 0, u, u + 1 == mine);
          if (!ok) break;
          if (!paired && j + 1 < n) {
            sk = next_slot();
            if (!ok) break;
            if (u + 2 < mine) issue_s(sk, 0);
            if (!ok) break;
            if (u + 3 == mine) commit(&bar->q_empty);
          }
          if (own && u + 1 < mine) issue_pv(sv, 1, u + 1, u + 2 == mine);
          if (!ok) break;
          commit(&bar->slot_empty[sv]);
          if (own) u += 2;
          if (paired && j + 1 < n) {
            own = ((j + 1) & 1) == t;
            sk = next_slot();
            if (!ok) break;
            if (own && u < mine) issue_s(sk, 0);
            if (!ok) break;
            if (own && u + 1 == mine) commit(&bar->q_empty);
          }
        }
      }
      int late = 0;
      commit(&bar->drain[t]);
      mbar_drain(&bar->drain[t], 0, &late, a.err_word);
    }
   } else if (warp == kCheckWarp) {
    // ------------------------------------------------------ masked V blocks
    int seq = 0, masked = 0;
    for (int i = 0;; ++i) {
      Item* it = item_at(i);
      if (!__all_sync(0xffffffffu, it != nullptr)) break;
      const Work w = it->w;
      const int n = item_blocks(it);
      bool ok = true;
      for (int j = masked_from(w, 0); ok && j < n; ++j) {
        ok = mbar_wait(&bar->masked_full[masked % kMaskedRing], (masked / kMaskedRing) & 1, abort_flag,
                       a.err_word);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++masked;
        const int s = (seq + 2 * j + 1) % kSlots;
        const int key0 = j * kBlock;
        clean_masked_values(sRing + s * kSlotBytes, row_limit(w, 0, a.causal) - key0,
                            min(kBlock, w.keys - key0), it->odd);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->slot_full[s]);
      }
      if (!ok) break;
      seq += 2 * n;
      __syncwarp();
      if (lane == 0) done_with(i);
    }
   }
  } else {
    // ------------------------------------------------------------ softmax
    const int t = warp >> 2;                   // this group's tile
    const int wq = warp & 3;
    const int row = wq * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t sbuf = tmem + lane_addr + t * 128;
    const uint32_t obuf = tmem + lane_addr + 256 + t * 128;
    const int head_in_group = row - row / G * G;
    const float c = a.scale * kLog2e;
    const float2 c2 = make_float2(c, c);
    uint32_t seen = 0, outs = 0;               // sub-blocks, outputs
    bool ok = true;
    for (int i = 0; ok; ++i) {
      Item* it = item_at(i);
      if (!__all_sync(0xffffffffu, it != nullptr)) break;
      const Work w = it->w;
      const int n = t ? it->n[1] : it->n[0];
      const int head = it->hk * G + head_in_group;
      const int paired = kSplit ? it->paired : 0;
      const int t0 = paired ? 0 : t * tt;        // first query of the tile
      const int token = t0 + row / G;            // in the item
      const int from = row_limit(w, t0, a.causal);   // keys that every row sees
      // rows past the tile's tokens x heads (row / G >= tt) belong to no query
      const int limit = row < tt * G ? row_limit(w, token, a.causal) : 0;
      const bool warp_active = wq * 32 < min(tt, w.tokens - t0) * G;
      float m = -INFINITY, l = 0.f;
      for (int u = 0; u < n; ++u, ++seen) {
        ok = mbar_wait(&bar->s_full[t], seen & 1, abort_flag, a.err_word);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        if (warp_active) {
          uint32_t r[kSub];
          tmem_ld_32x32b_x32(sbuf, r);
          tmem_ld_32x32b_x32(sbuf + 32, r + 32);
          tmem_wait_ld();
          reg_fence<kSub>(r);
          tc_fence_before();
          mbar_arrive(&bar->s_empty[t]);
          const int key0 = paired ? (u & ~1) * kBlock + t * kBlock + (u & 1) * kSub : u * kSub;
          if (key0 + kSub > from) {
            const int valid = limit - key0;
#pragma unroll
            for (int x = 0; x < kSub; ++x)
              if (x >= valid) r[x] = __float_as_uint(-INFINITY);
          }
          float m8[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) m8[q] = fmaxf(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
#pragma unroll
          for (int x = 16; x < kSub; x += 16)
#pragma unroll
            for (int q = 0; q < 8; ++q)
              m8[q] = fmax3(m8[q], __uint_as_float(r[x + 2 * q]), __uint_as_float(r[x + 2 * q + 1]));
          const float mrow = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]),
                                   fmaxf(m8[6], m8[7])) * c;
          const bool need = mrow > m + kRescaleThreshold;
          if (u > 0 && __any_sync(0xffffffffu, need)) {
            ok = mbar_wait(&bar->pv_done[t], (seen - 1) & 1, abort_flag, a.err_word);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc_fence_after();
            const float f = need ? ex2_approx(m - mrow) : 1.f;
            l *= f;
#pragma unroll 1
            for (int cc = 0; cc < kHeadDim / 16; ++cc) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(obuf + cc * 16, o);
              tmem_wait_ld();
              reg_fence<16>(o);
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st_32x32b_x16(obuf + cc * 16, o);
            }
          }
          if (need) m = mrow;
          // -inf stands for "no key yet": the exponents (all -inf) are taken against 0.
          const float neg = m == -INFINITY ? 0.f : -m;
          const float2 neg_m = make_float2(neg, neg);
          float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                           make_float2(0.f, 0.f)};
          uint32_t pk[kSub / 2];
#pragma unroll
          for (int x = 0; x < kSub; x += 2) {
            const float2 e =
                __ffma2_rn(make_float2(__uint_as_float(r[x]), __uint_as_float(r[x + 1])), c2, neg_m);
            const float2 p = make_float2(ex2_approx(e.x), ex2_approx(e.y));
            acc[(x >> 1) & 3] = __fadd2_rn(acc[(x >> 1) & 3], p);
            pk[x >> 1] = pack_bf16x2(p.x, p.y);
          }
          tmem_st_32x32b_x32(sbuf + kSub + (seen & 1) * 32, pk);
          const float2 sum = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
          l += sum.x + sum.y;
          tmem_wait_st();
          tc_fence_before();
        } else {
          mbar_arrive(&bar->s_empty[t]);
        }
        mbar_arrive(&bar->p_full[t][seen & 1]);
      }
      if (!ok) break;
      // ---------------------------------------------------------- epilogue
      if (n > 0) {
        ok = mbar_wait(&bar->o_full[t], outs & 1, abort_flag, a.err_word);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        ++outs;
        tc_fence_after();
      }
      if constexpr (kSplit) {
        const int64_t p = ((it->part + paired * (it->part + t)) * a.q_rows + w.q0 + token) * a.heads + head;
        const bool row_valid = row < tt * G && token < w.tokens;
#pragma unroll 1
        for (int cc = 0; cc < kHeadDim / 32; ++cc) {
          uint32_t o[32];
          if (n > 0 && warp_active) {
            tmem_ld_32x32b_x32(obuf + cc * 32, o);
            tmem_wait_ld();
            reg_fence<32>(o);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0u;
          }
          if (row_valid) {
            uint4* dst = reinterpret_cast<uint4*>(a.part_o + p * kHeadDim + cc * 32);
#pragma unroll
            for (int x = 0; x < 8; ++x) dst[x] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        if (n > 0) {
          tc_fence_before();
          mbar_arrive(&bar->o_empty[t]);
        }
        if (row_valid) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m, l);
      } else {
        // O goes out through shared memory: a thread owns a row, whose 16-byte
        // pieces would each be a store of their own; staged, 8 lanes write 128
        // bytes of a row.  (16 16-byte stores a thread took 9,000 cycles an item.)
        const float inv_l = l != 0.f ? 1.f / l : 0.f;
        // this lane's rows of the stage (4 x + lane / 8): their offsets from the
        // item's first output
        const int own = ((token - t * tt) * a.heads + head_in_group) * kHeadDim;
        int at[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) at[x] = __shfl_sync(0xffffffffu, own, x * 4 + (lane >> 3));
        __nv_bfloat16* out = a.out + ((w.q0 + t * tt) * a.heads + it->hk * G) * kHeadDim + (lane & 7) * 8;
        const float2 inv2 = make_float2(inv_l, inv_l);
        const int rows = min(tt, w.tokens - t * tt) * G - wq * 32;   // of this warp
        uint8_t* stage = smem + kStageOff + warp * kStageBytes;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t o[2][32];
          if (n > 0 && warp_active) {
            tmem_ld_32x32b_x32(obuf + half * 64, o[0]);
            tmem_ld_32x32b_x32(obuf + half * 64 + 32, o[1]);
            tmem_wait_ld();
            reg_fence<32>(o[0]);
            reg_fence<32>(o[1]);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[0][x] = o[1][x] = 0u;
          }
          if (half == 1 && n > 0) {
            tc_fence_before();
            mbar_arrive(&bar->o_empty[t]);     // O_t is in registers: its buffer is free
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint32_t* v = &o[x >> 2][(x & 3) * 8];
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), inv2);
              pk[e] = pack_bf16x2(y.x, y.y);
            }
            *reinterpret_cast<uint4*>(stage + sw128_offset(lane, x)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
          __syncwarp();
          uint4 line[8];
#pragma unroll
          for (int x = 0; x < 8; ++x)
            line[x] = *reinterpret_cast<const uint4*>(stage + sw128_offset(x * 4 + (lane >> 3), lane & 7));
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (x * 4 + (lane >> 3) < rows) *reinterpret_cast<uint4*>(out + at[x] + half * 64) = line[x];
          __syncwarp();
        }
      }
      __syncwarp();
      if (a.causal && n > 0) {
        const uint32_t odd = lane < kHiddenWords ? *reinterpret_cast<volatile uint32_t*>(&it->odd[lane]) : 0u;
        if (__any_sync(0xffffffffu, odd != 0)) {
          float* part = nullptr;
          if constexpr (kSplit)
            part = a.part_o + (it->part + paired * (it->part + t)) * a.q_rows * a.heads * kHeadDim;
          add_not_finite(a, odd, w.q0 + t0, w.k0, it->hk, wq * 32, paired ? t : -1,
                         row_limit(w, 0, a.causal), limit, m, kSplit ? 1.f : l != 0.f ? 1.f / l : 0.f, part);
          __syncwarp();
        }
      }
      if (lane == 0) done_with(i);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a row: out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m)
// l_p, parts in order.  One warp a (query row, head).
__global__ void __launch_bounds__(256) combine_kernel(const PackedArgs a) {
  const int64_t rows = a.q_rows * a.heads;
  const int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int tt = 2 * a.tile_tokens;
  const int64_t q = row / a.heads;
  const int s = request_of_row(a.q_starts, a.requests, q);
  if (s < 0) return;                             // reported by the main kernel
  const int64_t begin = __ldg(a.q_starts + s);
  const Work w = find_work(a, begin / tt + s + (q - begin) / tt, tt);
  if (w.tokens == 0) return;
  const int parts = parts_of(item_blocks(w, a.causal), a) * (w.tokens <= a.tile_tokens ? 2 : 1);
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row;
  const float4* po = reinterpret_cast<const float4*>(a.part_o + row * kHeadDim) + lane;
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 32) {
    const float2 x = __ldg(ml + p * rows);
    if (x.y != 0.f) m = fmaxf(m, x.x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    const float2 x = __ldg(ml + p * rows);
    const float4 v = __ldg(po + p * rows * (kHeadDim / 4));
    const float f = x.y != 0.f ? ex2_approx(x.x - m) : 0.f;
    // a part without a key holds zeros
    l = fmaf(x.y, f, l);
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
cudaError_t launch_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
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
    e = cudaFuncSetAttribute(packed_attention_tiles_kernel<kSplit>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) smem_bytes[dev].store(bytes, std::memory_order_release);
  }
  packed_attention_tiles_kernel<kSplit>
      <<<static_cast<unsigned>(a.slots * a.kv_heads * a.splits), kThreads, bytes, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

}  // namespace

// Parts of an item's keys: one where the items alone give every SM two, or an
// average request has less than 1,024 keys; otherwise parts of part_blocks on
// the average request, up to sixteen parts an SM (a part costs about a
// microsecond beyond its loads).  Requests of a few tokens share a part between
// both tiles and take parts of twice the keys (in one run: 16
// requests of one token over 250,000 keys 180 us, with parts of 4 blocks 187; one request of one token
// over 16,384 keys: 33 us against 39), unless that leaves more than half of the
// SMs without one (25 tokens of 4 requests over 33,700 keys: 45 us, with parts
// of 4 blocks 33).
PackedPlan packed_plan(int64_t q_rows, int64_t k_rows, int32_t requests, int32_t heads,
                       int32_t kv_heads, int num_sms) {
  const int32_t tile_tokens = 128 / (heads / kv_heads);
  const int64_t items = (q_rows / (2 * tile_tokens) + requests) * kv_heads;
  const int64_t keys = requests > 0 ? k_rows / requests : 0;
  PackedPlan p{1, 4};
  if (items >= 2 * num_sms || keys < 8 * kBlock) return p;
  if (q_rows <= static_cast<int64_t>(requests) * tile_tokens && 2 * items * (keys / (8 * kBlock)) >= num_sms)
    p.part_blocks = 8;
  p.splits = static_cast<int32_t>(std::max<int64_t>(
      2, std::min((16 * num_sms + items - 1) / items, keys / (p.part_blocks * kBlock))));
  return p;
}

cudaError_t launch_packed_attention(const CUtensorMap& tq, const CUtensorMap& tk,
                                    const CUtensorMap& tv, const PackedArgs& a,
                                    cudaStream_t stream) {
  if (a.splits == 1) return launch_tiles<false>(tq, tk, tv, a, stream);
  const cudaError_t e = launch_tiles<true>(tq, tk, tv, a, stream);
  if (e != cudaSuccess) return e;
  const int64_t rows = a.q_rows * a.heads;
  combine_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace bsa
