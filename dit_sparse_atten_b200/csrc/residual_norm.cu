// Norms before and after a block, fused with its gate and residual, over a
// packed batch.  Row t belongs to request s (row_starts); in float32:
//   p = y[t], or post_norm(y[t]) * post_weight + post_bias
//   r = x[t] + gate[s] * p                                    -> residual[t]
//   h = norm(r) * weight + bias                (r before its rounding)
//   h = h * (1 + scale[s]) + shift[s]                         -> normed[t]
// norm(v) = (v - mean) / sqrt(var + eps) ("layer") or v / sqrt(mean(v^2) + eps)
// ("rms").  Unfused, this is the modulated LayerNorm, the gated residual and
// their float32 round trips of wan_diffusers.py:75-117.
//
// Bound: HBM.  A row is read once and stays in registers (8 columns to a
// 16-byte chunk, kChunks chunks a thread), so x and y are read once and r and
// h written once.  The variance is taken around the mean in a second register
// pass, not as E[v^2] - mean^2, which loses the variance of rows with a large
// mean.  Measured: 57,600 x 5,120 bf16 rows with y and three modulations in 402
// to 415 us over several runs, 5.7 to 5.9 TB/s (the best: 367 us, 6.43 TB/s, the
// rate of a plain copy; the other times in this file are from that run).  Before
// the resident kernel the float32 modulation rows went through L1 for every row
// and the sums' fixed instructions (380 a warp and row) filled the issue slots.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace {

constexpr int kNormStages = 16;                  // rows in flight a block, at most
constexpr int kNormRingBytes = 200 * 1024;       // of all blocks of an SM

// Untiled bulk copy; both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void widen2(uint32_t w, float& a, float& b, __nv_bfloat16) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void widen2(uint32_t w, float& a, float& b, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) {
  return pack_bf16x2(a, b);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float v, float* p) { *p = v; }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(float v, __half* p) { *p = __float2half_rn(v); }

// A thread's eight values of a chunk.  kVec: consecutive, all there, 16-byte
// aligned.  Otherwise (a width that is not a multiple of 8, or rows off the
// 16-byte grid) `es` apart, so that the block's threads read neighbouring
// columns, and there where e * es < left (20,000 x 1,777 bf16 rows with three
// modulations: 150 us, eight consecutive columns a thread 213).
template <bool kVec, bool kStream, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int left, int es, float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {              // a column past the width reads the last one: no branches
      const float t = widen(p[min(e * es, left - 1)]);
      v[e] = e * es < left ? t : 0.f;
    }
  } else if constexpr (sizeof(T) == 4) {
    const float4* q = reinterpret_cast<const float4*>(p);
    const float4 a = kStream ? __ldcs(q) : __ldg(q);
    const float4 b = kStream ? __ldcs(q + 1) : __ldg(q + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    const uint4 a = kStream ? __ldcs(q) : __ldg(q);
    widen2(a.x, v[0], v[1], T());
    widen2(a.y, v[2], v[3], T());
    widen2(a.z, v[4], v[5], T());
    widen2(a.w, v[6], v[7], T());
  }
}

// Eight values from shared memory (16-byte aligned) as four pairs, and back to
// global memory: pairs feed the packed float32 instructions.
template <typename T>
__device__ __forceinline__ void shared_pairs(const T* p, float2 (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    widen2(a.x, v[0].x, v[0].y, T());
    widen2(a.y, v[1].x, v[1].y, T());
    widen2(a.z, v[2].x, v[2].y, T());
    widen2(a.w, v[3].x, v[3].y, T());
  }
}
template <typename T>
__device__ __forceinline__ void store_pairs(T* p, const float2 (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow2(v[0].x, v[0].y, T()), narrow2(v[1].x, v[1].y, T()),
                                              narrow2(v[2].x, v[2].y, T()), narrow2(v[3].x, v[3].y, T()));
  }
}

template <bool kVec, typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int left, int es, const float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e * es < left) narrow(v[e], p + e * es);
  } else if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow2(v[0], v[1], T()), narrow2(v[2], v[3], T()),
                                              narrow2(v[4], v[5], T()), narrow2(v[6], v[7], T()));
  }
}

// A parameter vector of any of the three types (NormParam::dtype), the same
// for the whole launch.
template <bool kVec>
__device__ __forceinline__ void load_param(const NormParam& p, int64_t offset, int left, int es,
                                           float (&v)[8]) {
  if (p.dtype == kDtypeF32)
    load8<kVec, false>(static_cast<const float*>(p.ptr) + offset, left, es, v);
  else if (p.dtype == kDtypeBf16)
    load8<kVec, false>(static_cast<const __nv_bfloat16*>(p.ptr) + offset, left, es, v);
  else
    load8<kVec, false>(static_cast<const __half*>(p.ptr) + offset, left, es, v);
}

// Sum over the block, in a fixed order.  `slot` alternates between two arrays
// so that one barrier a sum is enough; entries past the block's warps are 0.
__device__ __forceinline__ float block_sum(float v, float* slot) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int warps = blockDim.x >> 5;
  if (warps == 1) {
    __syncwarp();
    return v;
  }
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < warps; w += 4) {
    const float4 p = *reinterpret_cast<const float4*>(slot + w);
    t.x += p.x; t.y += p.y; t.z += p.z; t.w += p.w;
  }
  return (t.x + t.y) + (t.z + t.w);
}

// v -> norm(v) in place (columns past the width stay 0).
template <int kChunks>
__device__ __forceinline__ void normalise(float (&v)[kChunks][8], int first, int es, int width, int kind,
                                          float eps, float (*slots)[32], int& turn) {
  const float inv_n = 1.f / static_cast<float>(width);
  const int stride = blockDim.x * 8;
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[c][e];
    mean = block_sum(s, slots[turn++ & 1]) * inv_n;
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int left = width - (first + c * stride);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] = e * es < left ? v[c][e] - mean : 0.f;
      s += v[c][e] * v[c][e];
    }
  }
  const float r = rsqrtf(fmaf(block_sum(s, slots[turn++ & 1]), inv_n, eps));
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] *= r;
}

// v = v * weight + bias for the parameters that are there.
template <bool kVec, int kChunks>
__device__ __forceinline__ void affine(float (&v)[kChunks][8], int first, int es, int width,
                                       const NormParam& weight, const NormParam& bias) {
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * blockDim.x * 8;
    if (col >= width) break;
    float w[8];
    if (weight.ptr != nullptr) {
      load_param<kVec>(weight, col, width - col, es, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] *= w[e];
    }
    if (bias.ptr != nullptr) {
      load_param<kVec>(bias, col, width - col, es, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] += w[e];
    }
  }
}

template <typename TX, typename TY, typename TN, bool kVec, int kChunks, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const NormArgs a) {
  __shared__ __align__(16) float slots[2][32];
  if (threadIdx.x < 64) (&slots[0][0])[threadIdx.x] = 0.f;
  __syncthreads();
  int turn = 0;
  const int64_t row = blockIdx.x;
  const int first = kVec ? threadIdx.x * 8 : threadIdx.x;
  const int es = kVec ? 1 : blockDim.x;
  const int stride = blockDim.x * 8;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  const TY* y = static_cast<const TY*>(a.y) + row * a.y_stride;
  float v[kChunks][8], p[kChunks][8];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * stride;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] = p[c][e] = 0.f;
    if (col >= a.width) continue;
    load8<kVec, true>(x + col, a.width - col, es, v[c]);
    if (a.y != nullptr) load8<kVec, true>(y + col, a.width - col, es, p[c]);
  }
  int64_t s = a.requests == 1 ? 0 : row;       // no row_starts: one request, or one for each row
  if (a.row_starts != nullptr) {
    s = request_of_row(a.row_starts, a.requests, row);
    if (s < 0) {                               // uniform over the block
      if (threadIdx.x == 0) atomicOr(a.err_word, kErrBadRoute);
      return;
    }
  }
  if (a.y != nullptr) {
    if (a.post_kind != kNormNone) {
      normalise<kChunks>(p, first, es, a.width, a.post_kind, a.eps, slots, turn);
      affine<kVec, kChunks>(p, first, es, a.width, a.post_weight, a.post_bias);
    }
    TX* r = static_cast<TX*>(a.residual) + row * a.width;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = first + c * stride;
      if (col >= a.width) break;
      float g[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
      if (a.gate.ptr != nullptr) load_param<kVec>(a.gate, s * a.gate_stride + col, a.width - col, es, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = fmaf(g[e], p[c][e], v[c][e]);
      store8<kVec>(r + col, a.width - col, es, v[c]);
    }
  }
  normalise<kChunks>(v, first, es, a.width, a.norm_kind, a.eps, slots, turn);
  affine<kVec, kChunks>(v, first, es, a.width, a.weight, a.bias);
  TN* h = static_cast<TN*>(a.normed) + row * a.width;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * stride;
    if (col >= a.width) break;
    float m[8];
    if (a.scale.ptr != nullptr) {
      load_param<kVec>(a.scale, s * a.scale_stride + col, a.width - col, es, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = fmaf(v[c][e], m[e], v[c][e]);
    }
    if (a.shift.ptr != nullptr) {
      load_param<kVec>(a.shift, s * a.shift_stride + col, a.width - col, es, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] += m[e];
    }
    store8<kVec>(h + col, a.width - col, es, v[c]);
  }
}

// A parameter's values for this thread's columns as pairs, `absent` where
// there is none.
__device__ __forceinline__ void param_pairs(const NormParam& p, int64_t offset, float absent,
                                            float2 (&v)[4]) {
  float t[8] = {absent, absent, absent, absent, absent, absent, absent, absent};
  if (p.ptr != nullptr) load_param<true>(p, offset, 8, 1, t);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = make_float2(t[2 * e], t[2 * e + 1]);
}

// v -> v - mean in place, returns 1 / sqrt(var + eps) ("layer"), or the same
// with mean 0 ("rms").  Chunks past the width are 0 and stay 0.
template <int kChunks>
__device__ __forceinline__ float centre(float2 (&v)[kChunks][4], const bool (&mine)[kChunks], int kind,
                                        float inv_n, float eps, float (*slots)[32], int& turn) {
  if (kind == kNormLayer) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      s = __fadd2_rn(s, __fadd2_rn(__fadd2_rn(v[c][0], v[c][1]), __fadd2_rn(v[c][2], v[c][3])));
    const float mean = block_sum(s.x + s.y, slots[turn]) * inv_n;
    turn ^= 1;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const float m = mine[c] ? -mean : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[c][e] = __fadd2_rn(v[c][e], make_float2(m, m));
    }
  }
  float2 s = make_float2(0.f, 0.f), t = s;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    s = __ffma2_rn(v[c][0], v[c][0], s);
    t = __ffma2_rn(v[c][1], v[c][1], t);
    s = __ffma2_rn(v[c][2], v[c][2], s);
    t = __ffma2_rn(v[c][3], v[c][3], t);
  }
  s = __fadd2_rn(s, t);
  const float sum = block_sum(s.x + s.y, slots[turn]);
  turn ^= 1;
  return rsqrtf(fmaf(sum, inv_n, eps));
}

// Many rows: a resident block takes rows blockIdx.x, + gridDim.x, ... (a run
// of rows a block instead: 407 us for 57,600 x 5,120 bf16, against 367) and a
// thread keeps its columns for all of them, so the modulation stays in
// registers, folded with the affine parameters into
//   r = x + g * post_norm(y),   h = a * norm(r) + b,
// and is loaded again only where the rows pass into another request.  x and y
// rows come through a ring of bulk copies that run `stages` rows ahead.
// (A post_bias would take 8 more registers a chunk: the kernel above has it.)
template <typename TX, typename TY, typename TN, int kChunks, int kMaxThreads, int kMinBlocks>
__global__ void __launch_bounds__(kMaxThreads, kMinBlocks)
    residual_norm_rows_kernel(const NormArgs a, int stages) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(16) float slots[2][32];
  __shared__ uint64_t full[kNormStages];
  __shared__ int abort_flag;
  const int x_bytes = a.width * static_cast<int>(sizeof(TX));
  const int y_bytes = a.y != nullptr ? a.width * static_cast<int>(sizeof(TY)) : 0;
  const int y_at = (x_bytes + 127) / 128 * 128;
  const int stage_bytes = y_at + (y_bytes + 127) / 128 * 128;
  for (int i = threadIdx.x; i < 64; i += blockDim.x) (&slots[0][0])[i] = 0.f;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
    abort_flag = prior_timeout(a.err_word) ? 1 : 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (abort_flag) return;                          // uniform
  auto load = [&](int64_t row, int stage) {
    uint8_t* dst = ring + stage * stage_bytes;
    mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(x_bytes + y_bytes));
    bulk_load(dst, static_cast<const TX*>(a.x) + row * a.x_stride, x_bytes, &full[stage]);
    if (y_bytes)
      bulk_load(dst + y_at, static_cast<const TY*>(a.y) + row * a.y_stride, y_bytes, &full[stage]);
  };
  const int64_t step = gridDim.x;
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && blockIdx.x + i * step < a.rows; ++i) load(blockIdx.x + i * step, i);
  const float inv_n = 1.f / static_cast<float>(a.width);
  const int first = threadIdx.x * 8;
  const int stride = blockDim.x * 8;
  bool mine[kChunks];
  float2 g[kChunks][4], ma[kChunks][4], mb[kChunks][4];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) mine[c] = first + c * stride < a.width;
  int64_t end = 0;                                 // first row that needs other modulation
  int turn = 0, stage = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += step) {
    bool known = true;
    if (row >= end) {
      int64_t s = 0;
      end = a.rows;
      if (a.row_starts != nullptr) {
        s = request_of_row(a.row_starts, a.requests, row);
        end = s >= 0 ? static_cast<int64_t>(__ldg(a.row_starts + s + 1)) : row;
      } else if (a.requests != 1) {
        s = row;
        end = row + 1;
      }
      known = s >= 0;
      if (!known && threadIdx.x == 0) atomicOr(a.err_word, kErrBadRoute);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (!known || !mine[c]) continue;
        const int col = first + c * stride;
        float2 t[4];
        param_pairs(a.gate, s * a.gate_stride + col, 1.f, g[c]);
        param_pairs(a.post_weight, col, 1.f, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) g[c][e] = __fmul2_rn(g[c][e], t[e]);
        param_pairs(a.weight, col, 1.f, ma[c]);
        param_pairs(a.bias, col, 0.f, mb[c]);
        param_pairs(a.scale, s * a.scale_stride + col, 0.f, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ma[c][e] = __ffma2_rn(ma[c][e], t[e], ma[c][e]);
          mb[c][e] = __ffma2_rn(mb[c][e], t[e], mb[c][e]);
        }
        param_pairs(a.shift, s * a.shift_stride + col, 0.f, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) mb[c][e] = __fadd2_rn(mb[c][e], t[e]);
      }
    }
    if (!mbar_wait(&full[stage], phase, &abort_flag, a.err_word)) {
      // Never leave a copy in flight into shared memory.
      int late = 0;
      if (threadIdx.x == 0)
        for (int i = 0; i < stages && row + i * step < a.rows; ++i)
          mbar_drain(&full[(stage + i) % stages], stage + i < stages ? phase : phase ^ 1, &late,
                    a.err_word);
      break;
    }
    const TX* xs = reinterpret_cast<const TX*>(ring + stage * stage_bytes) + first;
    const TY* ys = reinterpret_cast<const TY*>(ring + stage * stage_bytes + y_at) + first;
    float2 v[kChunks][4];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[c][e] = make_float2(0.f, 0.f);
      if (mine[c]) shared_pairs(xs + c * stride, v[c]);
    }
    if (a.y != nullptr) {
      float2 p[kChunks][4];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[c][e] = make_float2(0.f, 0.f);
        if (mine[c]) shared_pairs(ys + c * stride, p[c]);
      }
      if (a.post_kind != kNormNone) {
        const float r = centre<kChunks>(p, mine, a.post_kind, inv_n, a.eps, slots, turn);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[c][e] = __fmul2_rn(p[c][e], make_float2(r, r));
      }
      TX* dst = static_cast<TX*>(a.residual) + row * a.width + first;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (!mine[c]) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c][e] = __ffma2_rn(g[c][e], p[c][e], v[c][e]);
        if (known) store_pairs(dst + c * stride, v[c]);
      }
    }
    const float r = centre<kChunks>(v, mine, a.norm_kind, inv_n, a.eps, slots, turn);
    // every thread has read the stage (the sums' barriers are behind it)
    if (threadIdx.x == 0 && row + stages * step < a.rows) load(row + stages * step, stage);
    TN* dst = static_cast<TN*>(a.normed) + row * a.width + first;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (!known || !mine[c]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[c][e] = __ffma2_rn(__fmul2_rn(v[c][e], make_float2(r, r)), ma[c][e], mb[c][e]);
      store_pairs(dst + c * stride, v[c]);
    }
    if (++stage == stages) stage = 0, phase ^= 1;
  }
}

template <typename TX, typename TY, typename TN, int kChunks, int kMaxThreads, int kMinBlocks>
cudaError_t start_rows(const NormArgs& a, int threads, int blocks, cudaStream_t stream, int num_sms) {
  auto kernel = residual_norm_rows_kernel<TX, TY, TN, kChunks, kMaxThreads, kMinBlocks>;
  const int stage = (a.width * static_cast<int>(sizeof(TX)) + 127) / 128 * 128 +
                    (a.y != nullptr ? (a.width * static_cast<int>(sizeof(TY)) + 127) / 128 * 128 : 0);
  int stages = kNormRingBytes / blocks / stage;
  stages = stages > kNormStages ? kNormStages : stages;
  static std::atomic<bool> ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormRingBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const int64_t grid = std::min<int64_t>(a.rows, static_cast<int64_t>(num_sms) * blocks);
  kernel<<<static_cast<unsigned>(grid), threads, stages * stage, stream>>>(a, stages);
  return cudaGetLastError();
}

template <typename TX, typename TY, typename TN, bool kVec, int kChunks, int kMaxThreads>
void start(const NormArgs& a, int threads, cudaStream_t stream) {
  residual_norm_kernel<TX, TY, TN, kVec, kChunks, kMaxThreads>
      <<<static_cast<unsigned>(a.rows), threads, 0, stream>>>(a);
}

template <typename TX, typename TY, typename TN, bool kVec>
cudaError_t launch_typed(const NormArgs& a, cudaStream_t stream, int num_sms) {
  const int chunks = (a.width + 7) / 8;
  auto round = [](int n) { return (n + 31) / 32 * 32; };
  // Resident blocks from four rows an SM on (57,600 x 5,120 bf16 rows: 367 us,
  // one CTA a row 650; 8,190 x 1,536: 26 against 38); fewer rows do not repay
  // the ring.  Two chunks a thread halve the per-thread work of the sums; up
  // to 256 chunks one a thread leaves more rows in flight (8,190 x 1,536: 27.5
  // against 29.3 us).
  if constexpr (kVec) {
    if (a.rows >= 4 * num_sms && chunks <= 1280 && a.post_bias.ptr == nullptr) {
      if (chunks <= 256) {
        const int threads = round(chunks);
        return start_rows<TX, TY, TN, 1, 256, 3>(a, threads, std::min(768 / threads, 16), stream, num_sms);
      }
      const int threads = round((chunks + 1) / 2);
      if (threads <= 320)
        return start_rows<TX, TY, TN, 2, 320, 2>(a, threads, std::min(640 / threads, 16), stream, num_sms);
      return start_rows<TX, TY, TN, 2, 640, 1>(a, threads, 1, stream, num_sms);
    }
  }
  // one CTA a row: few rows get a thread for every chunk, more rows fewer
  // threads with more loads in flight each; odd widths no thread without a
  // column (20,000 x 100: 21 us, with 128 threads 72)
  int threads = a.rows <= 2 * num_sms && chunks <= 1024 ? std::max(128, round(chunks))
                : kVec                                  ? 128
                                                        : std::min(128, round(chunks));
  while (threads < 1024 && threads * (threads <= 256 ? 5 : 4) < chunks) threads *= 2;
  const int per = (chunks + threads - 1) / threads;
  if (per <= 1) start<TX, TY, TN, kVec, 1, 1024>(a, threads, stream);
  else if (per <= 2) start<TX, TY, TN, kVec, 2, 1024>(a, threads, stream);
  else if (threads > 256) start<TX, TY, TN, kVec, 4, 1024>(a, threads, stream);
  else if (per <= 3) start<TX, TY, TN, kVec, 3, 256>(a, threads, stream);
  else if (per <= 4) start<TX, TY, TN, kVec, 4, 256>(a, threads, stream);
  else start<TX, TY, TN, kVec, 5, 256>(a, threads, stream);
  return cudaGetLastError();
}

template <typename TX, typename TY, typename TN>
cudaError_t launch_vec(const NormArgs& a, cudaStream_t stream, int num_sms) {
  return a.vectorised ? launch_typed<TX, TY, TN, true>(a, stream, num_sms)
                      : launch_typed<TX, TY, TN, false>(a, stream, num_sms);
}

}  // namespace

cudaError_t launch_residual_norm(const NormArgs& a, cudaStream_t stream, int num_sms) {
  if (a.rows == 0 || a.width == 0) return cudaSuccess;
  if (a.x_dtype == kDtypeBf16) return launch_vec<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(a, stream, num_sms);
  if (a.x_dtype == kDtypeF16) return launch_vec<__half, __half, __half>(a, stream, num_sms);
  if (a.y_dtype == kDtypeBf16) return launch_vec<float, __nv_bfloat16, __nv_bfloat16>(a, stream, num_sms);
  if (a.y_dtype == kDtypeF16) return launch_vec<float, __half, __half>(a, stream, num_sms);
  return launch_vec<float, float, float>(a, stream, num_sms);
}

}  // namespace bsa
