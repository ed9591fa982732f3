// Low-rank adapters of many requests beside a shared projection, over a
// packed batch: for a row t of request s with adapter i = adapters[s] >= 0,
//   out[t] = y[t] + scales[i] * (x[t] A_i^T) B_i^T,   A_i [R, K], B_i [N, R],
// and out[t] = y[t] without an adapter (-1).  y is the shared projection's
// output (a plain library product).
//
// Two launches: the "shrink" x A^T leaves u [rows, R] (float32 partial sums
// over slices of K), the "expand" adds the slices, scales and multiplies by
// B^T.  Bound: HBM (x and y read once, out written once; 2 R (K + N) flops a
// row are far below the tensor rate for R <= 128).
//
// A row tile never spans two requests: tile slot g of M rows belongs to
// request s = #{i >= 1: floor(starts[i] / M) + i <= g} (floor(e/M) - floor(b/M)
// + 1 >= ceil((e - b) / M), so every request's slots hold its rows), found by
// one warp search; no list of tiles has to be made on the host.
#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace {

constexpr int kShrinkRows = 8;
constexpr int kExpandRows = 64;
constexpr int kExpandCols = 256;
constexpr int kWarps = 8;

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
  const bool bad = begin < 0 || end < begin || end > a.rows ||
                   (s == 0 && begin != 0) || (s == a.requests - 1 && end != a.rows);
  int id = __ldg(a.adapters + s);
  if ((bad || id < -1 || id >= a.count) && (threadIdx.x & 31) == 0) atomicOr(a.err_word, kErrBadRoute);
  if (begin < 0 || end > a.rows) return t;
  t.row = begin + (g - (begin / M + s)) * M;
  if (t.row < begin || t.row >= end) return t;
  t.rows = static_cast<int>(min(static_cast<int64_t>(M), end - t.row));
  t.adapter = id >= 0 && id < a.count ? id : -1;
  return t;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// u[slice][row][r] = x[row][k in slice] . A[r][k in slice] for up to 8 rows of
// one request.  The adapter is the M operand (16 ranks), the rows the N
// operand (8), so a few rows waste little and A is read once.  Lane (g, q) =
// (lane / 4, lane % 4) reads 16 bytes, k = 8 q .. 8 q + 7 of each 32-column
// step: the four words serve two k16 products, for both operands in the same
// (permuted) order of k.
template <int RG>
__global__ void __launch_bounds__(kWarps * 32) lora_shrink_kernel(const LoraArgs a) {
  __shared__ float part[kWarps][RG * 16][kShrinkRows];
  const Tile t = find_tile<kShrinkRows>(a, blockIdx.x);
  if (t.rows == 0 || t.adapter < 0) return;      // uniform over the block
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int slice = blockIdx.y;
  const int steps = (a.k + 31) / 32;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * slice / a.slices);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (slice + 1) / a.slices);
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
    part[warp][m * 16 + g][2 * q] = d[m][0];
    part[warp][m * 16 + g][2 * q + 1] = d[m][1];
    part[warp][m * 16 + g + 8][2 * q] = d[m][2];
    part[warp][m * 16 + g + 8][2 * q + 1] = d[m][3];
  }
  __syncthreads();
  float* u = a.workspace + (static_cast<int64_t>(slice) * a.rows + t.row) * a.rank_pad;
  for (int i = threadIdx.x; i < t.rows * a.rank_pad; i += kWarps * 32) {
    const int row = i / a.rank_pad, r = i % a.rank_pad;
    float sum = 0.f;
    if (r < RG * 16)
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += part[w][r][row];
    u[i] = sum;
  }
}

// out = y + (scale * sum of u's slices) B^T: each warp owns 32 columns, holds
// their B fragments in registers and goes down the tile's rows 16 at a time.
// Product column n of n-tile j stands for column 8 (n / 2) + 2 j + n % 2 of
// the 32, so that a thread's 4 x 2 results are 8 consecutive columns: y and
// out move as 16-byte accesses without a detour through shared memory.  The
// scaled u is rounded to bf16 (the tensor cores' operand; 2^-9 of the delta,
// as large as the final rounding of a delta that stands alone).
template <int KB>
__global__ void __launch_bounds__(kWarps * 32) lora_expand_kernel(const LoraArgs a) {
  const Tile t = find_tile<kExpandRows>(a, blockIdx.x);
  if (t.rows == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int c0 = blockIdx.y * kExpandCols + warp * 32;
  if (c0 >= a.n) return;
  const int col = c0 + 8 * q;                    // this thread's 8 columns
  const bool has = t.adapter >= 0;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 b[KB][4];
  if (has) {
    const __nv_bfloat16* lb = a.lora_b + static_cast<int64_t>(t.adapter) * a.n * a.rank;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int k = kb * 32 + q * 8;
        b[kb][j] = c < a.n && k < a.rank
            ? __ldg(reinterpret_cast<const uint4*>(lb + static_cast<int64_t>(c) * a.rank + k)) : zero;
      }
    }
  }
  const float scale = has ? (a.scales != nullptr ? __ldg(a.scales + t.adapter) : 1.f) : 0.f;
  for (int r0 = 0; r0 < t.rows; r0 += 16) {
    float d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[j][e] = 0.f;
    if (has) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int k = kb * 32 + q * 8;
        uint32_t w[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = r0 + g + 8 * half;
          float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (row < t.rows && k < a.rank) {
            const float* u = a.workspace + (t.row + row) * a.rank_pad + k;
            for (int s = 0; s < a.slices; ++s) {
              const float4 p0 = __ldg(reinterpret_cast<const float4*>(u));
              const float4 p1 = __ldg(reinterpret_cast<const float4*>(u) + 1);
              v[0] += p0.x; v[1] += p0.y; v[2] += p0.z; v[3] += p0.w;
              v[4] += p1.x; v[5] += p1.y; v[6] += p1.z; v[7] += p1.w;
              u += a.rows * a.rank_pad;
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) w[half][e] = pack_bf16x2(v[2 * e] * scale, v[2 * e + 1] * scale);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma_bf16(d[j], w[0][0], w[1][0], w[0][1], w[1][1], b[kb][j].x, b[kb][j].y);
          mma_bf16(d[j], w[0][2], w[1][2], w[0][3], w[1][3], b[kb][j].z, b[kb][j].w);
        }
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = r0 + g + 8 * half;
      if (row < t.rows && col < a.n) {
        const uint4 in = *reinterpret_cast<const uint4*>(a.y + (t.row + row) * a.y_stride + col);
        uint32_t w[4] = {in.x, in.y, in.z, in.w};
        if (has) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = pack_bf16x2(__uint_as_float(w[j] << 16) + d[j][2 * half],
                               __uint_as_float(w[j] & 0xffff0000u) + d[j][2 * half + 1]);
        }
        *reinterpret_cast<uint4*>(a.out + (t.row + row) * a.out_stride + col) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

}  // namespace

// Slices of K: enough CTAs for two waves of eight a SM, at least 512 of K each.
LoraPlan lora_plan(int64_t rows, int32_t requests, int32_t k, int32_t rank, int num_sms) {
  LoraPlan p{};
  p.rank_pad = (rank + 15) / 16 * 16;
  const int64_t slots = rows / kShrinkRows + requests;
  int64_t slices = (static_cast<int64_t>(num_sms) * 8 + slots - 1) / slots;
  const int64_t most = (k + 511) / 512;
  p.slices = static_cast<int32_t>(slices < 1 ? 1 : slices > most ? most : slices);
  p.workspace_bytes = rows * p.rank_pad * p.slices * 4;
  return p;
}

cudaError_t launch_lora_add(const LoraArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.n == 0) return cudaSuccess;
  const int groups = (a.rank + 15) / 16;
  const dim3 sg(static_cast<unsigned>(a.rows / kShrinkRows + a.requests),
                static_cast<unsigned>(a.slices));
  if (groups <= 1) lora_shrink_kernel<1><<<sg, kWarps * 32, 0, stream>>>(a);
  else if (groups <= 2) lora_shrink_kernel<2><<<sg, kWarps * 32, 0, stream>>>(a);
  else if (groups <= 4) lora_shrink_kernel<4><<<sg, kWarps * 32, 0, stream>>>(a);
  else lora_shrink_kernel<8><<<sg, kWarps * 32, 0, stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const dim3 eg(static_cast<unsigned>(a.rows / kExpandRows + a.requests),
                static_cast<unsigned>((a.n + kExpandCols - 1) / kExpandCols));
  const int kb = (a.rank + 31) / 32;
  if (kb <= 1) lora_expand_kernel<1><<<eg, kWarps * 32, 0, stream>>>(a);
  else if (kb <= 2) lora_expand_kernel<2><<<eg, kWarps * 32, 0, stream>>>(a);
  else lora_expand_kernel<4><<<eg, kWarps * 32, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace bsa
