// Low-rank adapters of many requests beside a shared projection, over a
// packed batch: for a row t of request s with adapter i = adapters[s] >= 0,
//   out[t] = y[t] + scales[i] * (x[t] A_i^T) B_i^T,   A_i [R, K], B_i [N, R],
// and out[t] = y[t] without an adapter (-1).  y is the shared projection's
// output (a plain library product).
//
// Two launches: the "shrink" leaves u = scales[i] * x A^T as bf16 [rows, R
// padded to 32] in the workspace, the "expand" adds u B^T to y.  Bound: HBM (x
// and y read once, out written once; 2 R (K + N) flops a row are far below the
// tensor rate for R <= 128).  u is rounded to bf16 as the tensor cores'
// operand: 2^-8 of each of its entries, as the final rounding of a delta that
// stands alone.
//
// K is cut into slices where the row tiles alone would leave SMs idle; the
// slices of a tile are one thread-block cluster, whose CTAs sum each other's
// float32 partial tiles through distributed shared memory in a fixed order.
//
// Measured over several runs: 57,600 rows, K = N = 5,120, rank 32, 312 to 320
// us, 5.5 to 5.7 TB/s (the best: 296); 10,007 ragged rows, N = 13,824,
// rank 64, 130 to 134 us (126); 1,859 rows of 8 prompts, K = 4,096, rank 128, 33
// us and 32 single rows, N = 30,720, rank 16, 19 us, which are the latency of
// the two launches.
//
// A row tile never spans two requests: tile slot g of M rows belongs to
// request s = #{i >= 1: floor(starts[i] / M) + i <= g} (floor(e/M) - floor(b/M)
// + 1 >= ceil((e - b) / M), so every request's slots hold its rows), found by
// one warp search; no list of tiles has to be made on the host.
#include <algorithm>
#include <atomic>

#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace {

constexpr int kFewRows = 8;        // rows a tile, requests of few rows
constexpr int kTileRows = 128;     // rows a tile, tensor-core shrink
constexpr int kExpandRows = 16;    // rows a tile, expand of requests of few rows
constexpr int kWarps = 8;
constexpr int kMaxSlices = 8;      // portable cluster size

struct Tile {
  int64_t row;      // first row
  int rows;         // rows of this tile (0: none)
  int adapter;      // -1: none
};

// Tile of slot g (uniform over the calling warp).
template <int M>
__device__ __forceinline__ Tile find_tile(const LoraArgs& a, int64_t g) {
  const int s = warp_count_le(a.requests, g, [&](int i) {
    return static_cast<int64_t>(__ldg(a.row_starts + i)) / M + i;
  });
  Tile t{0, 0, -1};
  if (s >= a.requests) return t;
  const int64_t begin = __ldg(a.row_starts + s), end = __ldg(a.row_starts + s + 1);
  const int id = __ldg(a.adapters + s);
  const bool bad = begin < 0 || end < begin || end > a.rows ||
                   (s == 0 && begin != 0) || (s == a.requests - 1 && end != a.rows);
  if ((bad || id < -1 || id >= a.count) && (threadIdx.x & 31) == 0) atomicOr(a.err_word, kErrBadRoute);
  if (begin < 0 || end > a.rows) return t;
  t.row = begin + (g - (begin / M + s)) * M;
  if (t.row < begin || t.row >= end) return t;
  t.rows = static_cast<int>(min(static_cast<int64_t>(M), end - t.row));
  t.adapter = id >= 0 && id < a.count ? id : -1;
  return t;
}

__device__ __forceinline__ float adapter_scale(const LoraArgs& a, int adapter) {
  return a.scales != nullptr ? __ldg(a.scales + adapter) : 1.f;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Cluster helpers: the K slices of a tile are the CTAs of a cluster.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// The float4 at `p` (this CTA's shared memory) in CTA `rank` of the cluster.
__device__ __forceinline__ float4 peer_float4(const float* p, int rank) {
  uint32_t addr;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Joins the slices' partial tiles `part` (rows `stride` floats apart, in
// the shared memory of each CTA of the cluster): this CTA takes every slices-th
// row, adds the slices in order, scales, rounds and writes u.  Columns past the
// rank are 0, not what the padded products left there: that is 0 times x and
// the scale, NaN where one of them is not finite, and would reach the whole row
// through the expand's 0 columns of B.
__device__ __forceinline__ void join_slices(const LoraArgs& a, const Tile& t, const float* part,
                                            int stride, float scale) {
  if (a.slices > 1) cluster_sync(); else __syncthreads();
  const int per_row = a.rank_pad / 4;
  const int mine = static_cast<int>(blockIdx.y);
  for (int i = threadIdx.x; ; i += blockDim.x) {
    const int row = mine + i / per_row * a.slices, c = i % per_row * 4;
    if (row >= t.rows) break;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.rank) {                            // rank % 8 == 0
      const float* at = part + row * stride + c;
      if (a.slices == 1) {
        v = *reinterpret_cast<const float4*>(at);
      } else {
        float4 p[kMaxSlices];                    // all on their way at once
#pragma unroll
        for (int s = 0; s < kMaxSlices; ++s)
          p[s] = s < a.slices ? peer_float4(at, s) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int s = 0; s < kMaxSlices; ++s) {
          v.x += p[s].x; v.y += p[s].y; v.z += p[s].z; v.w += p[s].w;
        }
      }
      v = make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
    }
    *reinterpret_cast<uint2*>(a.workspace + (t.row + row) * a.rank_pad + c) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
  __syncwarp();
  if (a.slices > 1) cluster_sync();   // peers may still read this CTA's tile
}

// Shrink for requests of few rows: up to 8 rows of one request.  The adapter
// is the M operand (16 ranks), the rows the N operand (8), so a few rows waste
// little and A is read once.  Lane (g, q) = (lane / 4, lane % 4) reads 16
// bytes, k = 8 q .. 8 q + 7 of each 32-column step: the four words serve two
// k16 products, for both operands in the same (permuted) order of k.
template <int RG>
__global__ void __launch_bounds__(kWarps * 32) lora_shrink_few_kernel(const LoraArgs a) {
  constexpr int kPad = RG * 16;
  __shared__ __align__(16) float part[kWarps][kFewRows][kPad];
  pdl_launch_dependents();
  const Tile t = find_tile<kFewRows>(a, blockIdx.x);
  if (t.rows == 0 || t.adapter < 0) return;      // uniform over the cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int steps = (a.k + 31) / 32;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / a.slices);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / a.slices);
  const __nv_bfloat16* la = a.lora_a + static_cast<int64_t>(t.adapter) * a.rank * a.k;
  const __nv_bfloat16* x = a.x + (t.row + (g < t.rows ? g : 0)) * a.x_stride;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float d[RG][4];
#pragma unroll
  for (int m = 0; m < RG; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[m][e] = 0.f;
#pragma unroll 2
  for (int s = s0 + warp; s < s1; s += kWarps) {
    const int k = s * 32 + q * 8;
    const bool in = k < a.k;
    const uint4 b = in && g < t.rows ? __ldg(reinterpret_cast<const uint4*>(x + k)) : zero;
#pragma unroll
    for (int m = 0; m < RG; ++m) {
      const int r = m * 16 + g;
      const uint4 lo = in && r < a.rank
          ? __ldg(reinterpret_cast<const uint4*>(la + static_cast<int64_t>(r) * a.k + k)) : zero;
      const uint4 hi = in && r + 8 < a.rank
          ? __ldg(reinterpret_cast<const uint4*>(la + static_cast<int64_t>(r + 8) * a.k + k)) : zero;
      mma_bf16(d[m], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
      mma_bf16(d[m], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
    }
  }
#pragma unroll
  for (int m = 0; m < RG; ++m) {
    part[warp][2 * q][m * 16 + g] = d[m][0];
    part[warp][2 * q + 1][m * 16 + g] = d[m][1];
    part[warp][2 * q][m * 16 + g + 8] = d[m][2];
    part[warp][2 * q + 1][m * 16 + g + 8] = d[m][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kFewRows * kPad; i += kWarps * 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += (&part[w][0][0])[i];
    (&part[0][0][0])[i] = sum;
  }
  join_slices(a, t, &part[0][0][0], kPad, adapter_scale(a, t.adapter));
}

// Shrink on the tensor cores (14,400 rows, K = 5,120, rank 32: 33 us for 148 MB,
// bound by HBM and the ramp of the first loads): 128 rows of one request (the
// box may reach into the next request's rows; they fill rows of the tile that
// are not stored) times the adapter's ranks as N, 64 of K a stage, both by TMA.
//   warp 0   TMA producer     warp 1   TMEM owner and MMA issuer
//   all      epilogue: a row a thread, float32 to shared memory, join_slices
struct ShrinkBarriers {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
};
constexpr int kShrinkThreads = 128;
// Two CTAs an SM; also holds the 128 x 128 float32 partial tile.
constexpr int kShrinkRing = 100 * 1024;
constexpr int kShrinkSmem = kShrinkRing + 1024 + static_cast<int>(sizeof(ShrinkBarriers));

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

template <int kPad>
__global__ void __launch_bounds__(kShrinkThreads)
    lora_shrink_kernel(const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_a, const LoraArgs a) {
  constexpr int kXBytes = kTileRows * 128;
  constexpr int kStage = kXBytes + kPad * 128;
  constexpr int kStages = kShrinkRing / kStage < 8 ? kShrinkRing / kStage : 8;
  constexpr int kCols = kPad < 32 ? 32 : kPad;
  constexpr int kPartStride = kPad + 4;   // a thread writes a row: 16 bytes off the bank period
  static_assert(kStages >= 3 && kTileRows * kPartStride * 4 <= kShrinkRing, "ring");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  ShrinkBarriers* bar = reinterpret_cast<ShrinkBarriers*>(ring + kShrinkRing);
  volatile int* abort_flag = &bar->abort;
  pdl_launch_dependents();
  const Tile t = find_tile<kTileRows>(a, blockIdx.x);
  if (t.rows == 0 || t.adapter < 0) return;      // uniform over the cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int steps = (a.k + 63) / 64;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / a.slices);
  const int n = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / a.slices) - s0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    mbar_init(&bar->done, 1);
    bar->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&bar->tmem_base, kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  if (warp == 0) {
    if (lane == 0) {
      LoadRing<kStages> loads;
      for (int i = 0; i < n; ++i) {
        const int s = loads.slot();
        if (!mbar_wait(&bar->empty[s], loads.empty_parity(), abort_flag, a.err_word)) break;
        uint8_t* dst = ring + s * kStage;
        mbar_arrive_expect_tx(&bar->full[s], kStage);
        tma_load_2d(dst, &tm_x, &bar->full[s], (s0 + i) * 64, static_cast<int>(t.row));
        tma_load_3d(dst + kXBytes, &tm_a, &bar->full[s], (s0 + i) * 64, 0, t.adapter);
        loads.arm();
      }
      // Never leave a copy in flight into shared memory.
      int late = 0;
      loads.for_each_open([&](int s, uint32_t parity) { mbar_drain(&bar->full[s], parity, &late, a.err_word); });
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_bf16_f32(128, kPad, false);
      const uint64_t x0 = sdesc_sw128(smem_u32(ring), 16, 1024);
      for (int i = 0; i < n; ++i) {
        const int s = i % kStages;
        if (!mbar_wait(&bar->full[s], (i / kStages) & 1, abort_flag, a.err_word)) break;
        tc_fence_after();
        const uint64_t xd = x0 + static_cast<uint64_t>((s * kStage) >> 4);
        const uint64_t ad = xd + static_cast<uint64_t>(kXBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_bf16_ss(tmem, xd + kk * 2, ad + kk * 2, idesc, (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&bar->empty[s]);
      }
      int late = 0;
      umma_commit(&bar->done);
      mbar_drain(&bar->done, 0, &late, a.err_word);
    }
  }
  __syncthreads();
  // A timed-out wait leaves wrong sums behind, reported in the error word; the
  // cluster still meets at its barriers below.
  tc_fence_after();
  float* part = reinterpret_cast<float*>(ring);
  const int row = threadIdx.x;
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    uint32_t v[32];
    tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, v);
    tmem_wait_ld();
    reg_fence<32>(v);
#pragma unroll
    for (int e = 0; e < 32; e += 4)
      if (c + e < kPad)
        *reinterpret_cast<uint4*>(part + row * kPartStride + c + e) =
            make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
  join_slices(a, t, part, kPartStride, adapter_scale(a, t.adapter));
}

// Expand for requests of few rows: out = y + u B^T for 16 rows of one request
// and kGroups x 32 columns a warp.  Product column n of n-tile j stands for
// column 8 (n / 2) + 2 j + n % 2 of the 32, so that a thread's 4 x 2 results
// are 8 consecutive columns: y and out move as 16-byte accesses, and u's rows
// are the A fragments as they lie (k permuted as in lora_shrink_few_kernel).
// All loads of y and B are requested before the wait for u: a CTA lives for
// little more than one memory latency, which is what bounds this kernel.
template <int KB, int kGroups>
__global__ void __launch_bounds__(kWarps * 32) lora_expand_few_kernel(const LoraArgs a) {
  const int64_t slot = blockIdx.x / a.col_ctas;
  const Tile t = find_tile<kExpandRows>(a, slot);
  if (t.rows == 0) {
    pdl_wait();     // no block ends before the shrink has: what follows may reuse its workspace
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const bool has = t.adapter >= 0;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const __nv_bfloat16* lb = a.lora_b + (has ? static_cast<int64_t>(t.adapter) * a.n * a.rank : 0);
  const int c0 = (static_cast<int>(blockIdx.x % a.col_ctas) * kWarps + warp) * 32 * kGroups;
  uint4 y[kGroups][2], b[kGroups][KB][4];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int col = c0 + i * 32 + 8 * q;         // this thread's 8 columns
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = g + 8 * half;
      y[i][half] = row < t.rows && col < a.n
          ? *reinterpret_cast<const uint4*>(a.y + (t.row + row) * a.y_stride + col) : zero;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + i * 32 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int k = kb * 32 + q * 8;
        b[i][kb][j] = has && c < a.n && k < a.rank
            ? __ldg(reinterpret_cast<const uint4*>(lb + static_cast<int64_t>(c) * a.rank + k)) : zero;
      }
    }
  }
  pdl_wait();                                    // u
  uint4 w[KB][2];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = g + 8 * half;
      w[kb][half] = has && row < t.rows
          ? *reinterpret_cast<const uint4*>(a.workspace + (t.row + row) * a.rank_pad + kb * 32 + q * 8)
          : zero;
    }
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    float d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) d[j][e] = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        mma_bf16(d[j], w[kb][0].x, w[kb][1].x, w[kb][0].y, w[kb][1].y, b[i][kb][j].x, b[i][kb][j].y);
        mma_bf16(d[j], w[kb][0].z, w[kb][1].z, w[kb][0].w, w[kb][1].w, b[i][kb][j].z, b[i][kb][j].w);
      }
    }
    const int col = c0 + i * 32 + 8 * q;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = g + 8 * half;
      if (row >= t.rows || col >= a.n) continue;
      uint32_t v[4] = {y[i][half].x, y[i][half].y, y[i][half].z, y[i][half].w};
      if (has) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = pack_bf16x2(__uint_as_float(v[j] << 16) + d[j][2 * half],
                             __uint_as_float(v[j] & 0xffff0000u) + d[j][2 * half + 1]);
      }
      *reinterpret_cast<uint4*>(a.out + (t.row + row) * a.out_stride + col) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// Expand on the tensor cores: resident CTAs take (128 rows x 128 columns)
// tiles of out, columns first, and stream y through a ring of shared-memory
// stages; D = u B^T goes through two TMEM buffers, and out is written over y's
// stage and stored by TMA (a tile that ends inside 128 rows: by the threads,
// since a box would reach into the next request).  Every copy is asynchronous,
// so HBM stays busy while the small products and sums go on.
//   warp 0     TMA producer: y and B of a tile; u when the row tile changes
//   warp 1     TMEM owner and MMA issuer
//   warps 2-9  y + D: two groups of four warps take alternate tiles (and TMEM
//              buffers), a row a thread, 32 columns at a time
template <int KP>   // 64-column panels of the rank
struct ExpandLayout {
  static constexpr int kYBytes = kTileRows * 256;
  static constexpr int kBBytes = KP * 128 * 128;
  static constexpr int kStage = kYBytes + kBBytes;
  static constexpr int kStages = KP == 1 ? 4 : 3;
  static constexpr int kUBytes = KP * kTileRows * 128;
  static constexpr int kUBuffers = KP == 1 ? 2 : 1;
  static constexpr int kUOff = kStages * kStage;
  static constexpr int kBarOff = kUOff + kUBuffers * kUBytes;
};
struct ExpandBarriers {
  uint64_t full[4], empty[4];
  uint64_t u_full[2], u_empty[2];
  uint64_t d_full[2], d_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
constexpr int kExpandThreads = 320;

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(smem_u32(src))
               : "memory");
}

// Walks this CTA's tiles; each warp has its own copy.  Items are runs of
// `run` column tiles of one row tile; CTA b takes runs b, b + grid, ...
struct ExpandWalk {
  int64_t slot;        // row tile of the run
  int part;            // run within the row tile
  int col, end;        // next column tile of the run, and its end
  int cols, run, parts;
  int step_slots, step_parts;
  int64_t slots;
  bool fresh = true;   // `slot` has not been looked up
  Tile tile{0, 0, -1};
  __device__ ExpandWalk(int64_t slots_, int cols_, int run_)
      : cols(cols_), run(run_), parts((cols_ + run_ - 1) / run_), slots(slots_) {
    slot = blockIdx.x / parts;
    part = static_cast<int>(blockIdx.x % parts);
    step_slots = static_cast<int>(gridDim.x / parts);
    step_parts = static_cast<int>(gridDim.x % parts);
    col = part * run;
    end = min(col + run, cols);
  }
  // Column tile of the next item with rows, or -1; `changed`: another row tile.
  __device__ __forceinline__ int next(const LoraArgs& a, bool& changed) {
    changed = false;
    while (slot < slots) {
      if (fresh) {
        tile = find_tile<kTileRows>(a, slot);
        fresh = false;
        changed = true;
      }
      if (tile.rows > 0 && col < end) return col++;
      const int64_t before = slot;
      slot += step_slots;
      part += step_parts;
      if (part >= parts) {
        part -= parts;
        ++slot;
      }
      fresh = slot != before;
      col = part * run;
      end = min(col + run, cols);
    }
    return -1;
  }
};

template <int KP>
__global__ void __launch_bounds__(kExpandThreads, 1)
    lora_expand_tiles_kernel(const __grid_constant__ CUtensorMap tm_y,
                             const __grid_constant__ CUtensorMap tm_out,
                             const __grid_constant__ CUtensorMap tm_b,
                             const __grid_constant__ CUtensorMap tm_u, const LoraArgs a) {
  using L = ExpandLayout<KP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  ExpandBarriers* bar = reinterpret_cast<ExpandBarriers*>(smem + L::kBarOff);
  volatile int* abort_flag = &bar->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t slots = a.rows / kTileRows + a.requests;
  const int cols = (a.n + 127) / 128;
  ExpandWalk walk(slots, cols, a.run);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->u_full[i], 1);
      mbar_init(&bar->u_empty[i], 1);
      mbar_init(&bar->d_full[i], 1);
      mbar_init(&bar->d_empty[i], 128);
    }
    mbar_init(&bar->drain, 1);
    bar->abort = prior_timeout(a.err_word) ? 1 : 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (bar->abort) {           // uniform
    pdl_wait();               // never end before the shrink has
    return;
  }
  if (warp == 1) tmem_alloc(&bar->tmem_base, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  bool changed;
  if (warp == 0) {
    // -------------------------------------------------------------- producer
    LoadRing<L::kStages> tiles;
    LoadRing<L::kUBuffers> us;      // u of row tiles with an adapter
    bool ok = true, waited = false;
    for (int c; ok && (c = walk.next(a, changed)) >= 0;) {
      const bool has = walk.tile.adapter >= 0;
      const int s = tiles.slot();
      uint8_t* dst = smem + s * L::kStage;
      const int row = static_cast<int>(walk.tile.row);
      if (lane == 0) {
        ok = mbar_wait(&bar->empty[s], tiles.empty_parity(), abort_flag, a.err_word);
        if (ok) {
          mbar_arrive_expect_tx(&bar->full[s], L::kYBytes + (has ? L::kBBytes : 0));
          tma_load_2d(dst, &tm_y, &bar->full[s], c * 128, row);
          tma_load_2d(dst + 16384, &tm_y, &bar->full[s], c * 128 + 64, row);
          if (has)
#pragma unroll
            for (int p = 0; p < KP; ++p)
              tma_load_3d(dst + L::kYBytes + p * 16384, &tm_b, &bar->full[s], p * 64, c * 128,
                          walk.tile.adapter);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok) tiles.arm();
      if (ok && changed && has) {
        if (!waited) pdl_wait();               // u comes from the shrink
        waited = true;
        const int ub = us.slot();
        if (lane == 0) {
          ok = mbar_wait(&bar->u_empty[ub], us.empty_parity(), abort_flag, a.err_word);
          if (ok) {
            mbar_arrive_expect_tx(&bar->u_full[ub], L::kUBytes);
#pragma unroll
            for (int p = 0; p < KP; ++p)
              tma_load_2d(smem + L::kUOff + ub * L::kUBytes + p * 16384, &tm_u, &bar->u_full[ub], p * 64, row);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (ok) us.arm();
      }
    }
    if (!waited) pdl_wait();    // never end before the shrink has
    // Never leave a copy in flight into shared memory: the readers may have
    // given up, or give up after this.
    if (lane == 0) {
      int late = 0;
      tiles.for_each_open([&](int s, uint32_t parity) { mbar_drain(&bar->full[s], parity, &late, a.err_word); });
      us.for_each_open([&](int s, uint32_t parity) { mbar_drain(&bar->u_full[s], parity, &late, a.err_word); });
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t idesc = idesc_bf16_f32(128, 128, false);
    const int ksteps = (a.rank + 15) / 16;
    int i = 0, u = 0, uses[2] = {0, 0};        // uses of each TMEM buffer
    bool ok = true, open = false;              // open: a row tile's u is in use
    for (int c; ok && (c = walk.next(a, changed)) >= 0; ++i) {
      const bool has = walk.tile.adapter >= 0;
      if (lane == 0) {
        if (changed && open) umma_commit(&bar->u_empty[(u - 1) % L::kUBuffers]);
        if (has) {
          const int s = i % L::kStages, db = i & 1;
          const int use = db ? uses[1]++ : uses[0]++;
          if (changed) {
            ok = mbar_wait(&bar->u_full[u % L::kUBuffers], (u / L::kUBuffers) & 1, abort_flag, a.err_word);
            ++u;
          }
          const int ub = (u - 1) % L::kUBuffers;
          if (ok) ok = mbar_wait(&bar->full[s], (i / L::kStages) & 1, abort_flag, a.err_word);
          if (ok) ok = mbar_wait(&bar->d_empty[db], (use & 1) ^ 1, abort_flag, a.err_word);
          if (ok) {
            tc_fence_after();
            const uint64_t ud = sdesc_sw128(smem_u32(smem + L::kUOff + ub * L::kUBytes), 16, 1024);
            const uint64_t bd = sdesc_sw128(smem_u32(smem + s * L::kStage + L::kYBytes), 16, 1024);
            for (int kk = 0; kk < ksteps; ++kk) {
              const uint64_t off = static_cast<uint64_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
              umma_bf16_ss(tmem + db * 128, ud + off, bd + off, idesc, kk > 0 ? 1u : 0u);
            }
            umma_commit(&bar->d_full[db]);
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (changed) open = has;
    }
    if (lane == 0) {
      int late = 0;
      umma_commit(&bar->drain);
      mbar_drain(&bar->drain, 0, &late, a.err_word);
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int wq = warp & 3;                   // TMEM lanes 32 wq ..
    const int row = wq * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    const int db = (warp - 2) >> 2;            // this group's TMEM buffer and tile parity
    const bool leader = ((warp - 2) & 3) == 0 && lane == 0;
    int i = 0, use = 0;
    bool ok = true;
    for (int c; (c = walk.next(a, changed)) >= 0; ++i) {
      if ((i & 1) != db) continue;
      const bool has = walk.tile.adapter >= 0;
      const int s = i % L::kStages;
      ok = mbar_wait(&bar->full[s], (i / L::kStages) & 1, abort_flag, a.err_word);
      if (ok && has) ok = mbar_wait(&bar->d_full[db], use & 1, abort_flag, a.err_word);
      ok = __all_sync(0xffffffffu, ok);
      uint8_t* y = smem + s * L::kStage;
      const bool whole = walk.tile.rows == kTileRows;
      if (ok) {
        tc_fence_after();
        __nv_bfloat16* out = a.out + (walk.tile.row + row) * a.out_stride + c * 128;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t v[32];
          if (has) {
            tmem_ld_32x32b_x32(tmem + lane_addr + db * 128 + cc * 32, v);
            tmem_wait_ld();
            reg_fence<32>(v);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4* at = reinterpret_cast<uint4*>(y + (cc >> 1) * 16384 + sw128_offset(row, (cc & 1) * 4 + j));
            const uint4 in = *at;
            uint32_t w[4] = {in.x, in.y, in.z, in.w};
            if (has) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(__uint_as_float(w[e] << 16) + __uint_as_float(v[8 * j + 2 * e]),
                                   __uint_as_float(w[e] & 0xffff0000u) + __uint_as_float(v[8 * j + 2 * e + 1]));
            }
            const uint4 res = make_uint4(w[0], w[1], w[2], w[3]);
            if (whole)
              *at = res;
            else if (row < walk.tile.rows && c * 128 + cc * 32 + j * 8 < a.n)
              *reinterpret_cast<uint4*>(out + cc * 32 + j * 8) = res;
          }
        }
        if (has) {
          tc_fence_before();
          mbar_arrive(&bar->d_empty[db]);
          ++use;
        }
        if (whole) fence_proxy_async_smem();
      }
      // A warp that has given up comes here too, and the group leaves together:
      // one that left alone would be waited for without a limit.  (An mbarrier
      // that only the leader waits on: 320 us for the 57,600 rows against 315.)
      ok = named_bar_and(1 + db, 128, ok);
      if (!ok) break;
      if (leader) {
        if (whole) {
          tma_store_2d(&tm_out, y, c * 128, static_cast<int>(walk.tile.row));
          if (c * 128 + 64 < a.n)
            tma_store_2d(&tm_out, y + 16384, c * 128 + 64, static_cast<int>(walk.tile.row));
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        mbar_arrive(&bar->empty[s]);
      }
    }
    if (leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// Launch with a cluster of (1, slices, 1) CTAs.
template <typename... Params, typename... Args>
cudaError_t launch_sliced(void (*kernel)(Params...), dim3 grid, int threads, int smem, int slices,
                          cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = static_cast<unsigned>(slices);
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

// Launch whose blocks may start while the previous kernel of the stream still
// runs (griddepcontrol).
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem,
                             cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

// Raises a kernel's dynamic shared memory limit, once a device.
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, std::atomic<bool> (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  return e;
}

template <int kPad>
cudaError_t launch_shrink(const CUtensorMap& tx, const CUtensorMap& ta, const LoraArgs& a, dim3 grid,
                          cudaStream_t stream) {
  static std::atomic<bool> ready[64] = {};
  const cudaError_t e = allow_smem(lora_shrink_kernel<kPad>, kShrinkSmem, ready);
  if (e != cudaSuccess) return e;
  return launch_sliced(lora_shrink_kernel<kPad>, grid, kShrinkThreads, kShrinkSmem, a.slices, stream,
                       tx, ta, a);
}

template <int KP>
cudaError_t launch_tiles(const LoraMaps& m, LoraArgs a, cudaStream_t stream, int num_sms) {
  // Two column tiles of a row tile in a row share its u; longer runs move a
  // CTA's rows apart from its neighbours' in DRAM (57,600 x 5,120, rank 32:
  // 235 us for runs of 1, 217 of 2, 233 of 4, 246 and more of whole rows).
  a.run = 2;
  static std::atomic<bool> ready[64] = {};
  const int smem = ExpandLayout<KP>::kBarOff + static_cast<int>(sizeof(ExpandBarriers)) + 1024;
  const cudaError_t e = allow_smem(lora_expand_tiles_kernel<KP>, smem, ready);
  if (e != cudaSuccess) return e;
  const int64_t cols = (a.n + 127) / 128;
  const int64_t items = (a.rows / kTileRows + a.requests) * ((cols + a.run - 1) / a.run);
  return launch_dependent(lora_expand_tiles_kernel<KP>,
                          dim3(static_cast<unsigned>(std::min<int64_t>(items, num_sms))),
                          kExpandThreads, smem, stream, m.y, m.out, m.b, m.u, a);
}

}  // namespace

// The tensor-core shrink takes requests of more than 16 rows on average; fewer
// rows would leave most of its 128-row tiles empty and go 8 to a tile.  Slices
// of K: two CTAs an SM (eight of the small ones), at least 4 steps of 64 each.
LoraPlan lora_plan(int64_t rows, int32_t requests, int32_t k, int32_t rank, int num_sms) {
  LoraPlan p{};
  p.rank_pad = (rank + 31) / 32 * 32;
  p.few_rows = rows <= 16ll * requests;
  const int64_t slots = rows / (p.few_rows ? kFewRows : kTileRows) + requests;
  const int64_t want = static_cast<int64_t>(num_sms) * (p.few_rows ? 8 : 2) / slots;
  const int64_t most = std::min<int64_t>(kMaxSlices, (k + 255) / 256);
  p.slices = static_cast<int32_t>(std::max<int64_t>(1, std::min(want, most)));
  p.workspace_bytes = rows * p.rank_pad * 2;
  return p;
}

cudaError_t launch_lora_add(const LoraMaps& maps, LoraArgs a, cudaStream_t stream, int num_sms) {
  if (a.rows == 0 || a.n == 0) return cudaSuccess;
  const int groups = (a.rank + 15) / 16;
  const dim3 grid(static_cast<unsigned>(a.rows / (a.few_rows ? kFewRows : kTileRows) + a.requests),
                  static_cast<unsigned>(a.slices));
  cudaError_t e;
  if (a.few_rows) {
    const int threads = kWarps * 32;
    if (groups <= 1) e = launch_sliced(lora_shrink_few_kernel<1>, grid, threads, 0, a.slices, stream, a);
    else if (groups <= 2) e = launch_sliced(lora_shrink_few_kernel<2>, grid, threads, 0, a.slices, stream, a);
    else if (groups <= 4) e = launch_sliced(lora_shrink_few_kernel<4>, grid, threads, 0, a.slices, stream, a);
    else e = launch_sliced(lora_shrink_few_kernel<8>, grid, threads, 0, a.slices, stream, a);
    if (e != cudaSuccess) return e;
    const int kb = a.rank_pad / 32;
    auto expand = [&](auto kernel, int columns) {
      a.col_ctas = (a.n + kWarps * columns - 1) / (kWarps * columns);
      const int64_t ctas = (a.rows / kExpandRows + a.requests) * a.col_ctas;
      return launch_dependent(kernel, dim3(static_cast<unsigned>(ctas)), threads, 0, stream, a);
    };
    if (kb == 1) return expand(lora_expand_few_kernel<1, 4>, 128);
    if (kb == 2) return expand(lora_expand_few_kernel<2, 2>, 64);
    if (kb == 3) return expand(lora_expand_few_kernel<3, 1>, 32);
    return expand(lora_expand_few_kernel<4, 1>, 32);
  }
  if (groups <= 1) e = launch_shrink<16>(maps.x, maps.a, a, grid, stream);
  else if (groups <= 2) e = launch_shrink<32>(maps.x, maps.a, a, grid, stream);
  else if (groups <= 4) e = launch_shrink<64>(maps.x, maps.a, a, grid, stream);
  else e = launch_shrink<128>(maps.x, maps.a, a, grid, stream);
  if (e != cudaSuccess) return e;
  return a.rank <= 64 ? launch_tiles<1>(maps, a, stream, num_sms)
                      : launch_tiles<2>(maps, a, stream, num_sms);
}

// Ranks that a box of lora_a's tensor map covers.
int lora_rank_box(int32_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

}  // namespace bsa
