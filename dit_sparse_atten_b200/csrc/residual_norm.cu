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
// h written once; the modulation rows come from L1/L2.  The variance is taken
// around the mean in a second register pass, not as E[v^2] - mean^2, which
// loses the variance of rows with a large mean.
#include <cuda_fp16.h>

#include "bsa_kernels.h"
#include "packed_common.cuh"

namespace bsa {
namespace {

// Eight consecutive values starting at p, of which the first `left` exist.
// kVec: all eight exist and p is 16-byte aligned.
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

template <bool kVec, bool kStream, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int left, float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? widen(p[e]) : 0.f;
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

template <bool kVec, typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int left, const float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) narrow(v[e], p + e);
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
__device__ __forceinline__ void load_param(const NormParam& p, int64_t offset, int left,
                                           float (&v)[8]) {
  if (p.dtype == kDtypeF32)
    load8<kVec, false>(static_cast<const float*>(p.ptr) + offset, left, v);
  else if (p.dtype == kDtypeBf16)
    load8<kVec, false>(static_cast<const __nv_bfloat16*>(p.ptr) + offset, left, v);
  else
    load8<kVec, false>(static_cast<const __half*>(p.ptr) + offset, left, v);
}

// Sum over the block; `slot` alternates so that one barrier a sum is enough.
__device__ __forceinline__ float block_sum(float v, float* slot) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float total = 0.f;
  for (int w = 0; w < warps; ++w) total += slot[w];
  return total;
}

// v -> norm(v) in place (columns past the width stay 0).
template <int kChunks>
__device__ __forceinline__ void normalise(float (&v)[kChunks][8], int first, int width, int kind,
                                          float eps, float (*slots)[32], int& turn) {
  const float n = static_cast<float>(width);
  const int stride = blockDim.x * 8;
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[c][e];
    mean = block_sum(s, slots[turn++ & 1]) / n;
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int left = width - (first + c * stride);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] = e < left ? v[c][e] - mean : 0.f;
      s += v[c][e] * v[c][e];
    }
  }
  const float r = 1.f / sqrtf(block_sum(s, slots[turn++ & 1]) / n + eps);
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] *= r;
}

// v = v * weight + bias for the parameters that are there.
template <bool kVec, int kChunks>
__device__ __forceinline__ void affine(float (&v)[kChunks][8], int first, int width,
                                       const NormParam& weight, const NormParam& bias) {
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * blockDim.x * 8;
    if (col >= width) break;
    float w[8];
    if (weight.ptr != nullptr) {
      load_param<kVec>(weight, col, width - col, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] *= w[e];
    }
    if (bias.ptr != nullptr) {
      load_param<kVec>(bias, col, width - col, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] += w[e];
    }
  }
}

template <typename TX, typename TY, typename TN, bool kVec, int kChunks>
__global__ void __launch_bounds__(kChunks == 1 ? 640 : 1024) residual_norm_kernel(const NormArgs a) {
  __shared__ float slots[2][32];
  int turn = 0;
  const int64_t row = blockIdx.x;
  int64_t s = a.requests == 1 ? 0 : row;       // no row_starts: one request, or one for each row
  if (a.row_starts != nullptr) {
    s = request_of_row(a.row_starts, a.requests, row);
    if (s < 0) {                               // uniform over the block
      if (threadIdx.x == 0) atomicOr(a.err_word, kErrBadRoute);
      return;
    }
  }
  const int first = threadIdx.x * 8;
  const int stride = blockDim.x * 8;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  float v[kChunks][8];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * stride;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    if (col < a.width) load8<kVec, true>(x + col, a.width - col, v[c]);
  }
  if (a.y != nullptr) {
    const TY* y = static_cast<const TY*>(a.y) + row * a.y_stride;
    float p[kChunks][8];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = first + c * stride;
#pragma unroll
      for (int e = 0; e < 8; ++e) p[c][e] = 0.f;
      if (col < a.width) load8<kVec, true>(y + col, a.width - col, p[c]);
    }
    if (a.post_kind != kNormNone) {
      normalise<kChunks>(p, first, a.width, a.post_kind, a.eps, slots, turn);
      affine<kVec, kChunks>(p, first, a.width, a.post_weight, a.post_bias);
    }
    TX* r = static_cast<TX*>(a.residual) + row * a.width;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = first + c * stride;
      if (col >= a.width) break;
      float g[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
      if (a.gate.ptr != nullptr) load_param<kVec>(a.gate, s * a.gate_stride + col, a.width - col, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = fmaf(g[e], p[c][e], v[c][e]);
      store8<kVec>(r + col, a.width - col, v[c]);
    }
  }
  normalise<kChunks>(v, first, a.width, a.norm_kind, a.eps, slots, turn);
  affine<kVec, kChunks>(v, first, a.width, a.weight, a.bias);
  TN* h = static_cast<TN*>(a.normed) + row * a.width;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = first + c * stride;
    if (col >= a.width) break;
    float m[8];
    if (a.scale.ptr != nullptr) {
      load_param<kVec>(a.scale, s * a.scale_stride + col, a.width - col, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = fmaf(v[c][e], m[e], v[c][e]);
    }
    if (a.shift.ptr != nullptr) {
      load_param<kVec>(a.shift, s * a.shift_stride + col, a.width - col, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] += m[e];
    }
    store8<kVec>(h + col, a.width - col, v[c]);
  }
}

template <typename TX, typename TY, typename TN, bool kVec>
cudaError_t launch_typed(const NormArgs& a, cudaStream_t stream) {
  const int chunks = (a.width + 7) / 8;
  const unsigned grid = static_cast<unsigned>(a.rows);
  auto threads = [&](int per) { return ((chunks + per - 1) / per + 31) / 32 * 32; };
  if (chunks <= 640)
    residual_norm_kernel<TX, TY, TN, kVec, 1><<<grid, threads(1), 0, stream>>>(a);
  else if (chunks <= 2048)
    residual_norm_kernel<TX, TY, TN, kVec, 2><<<grid, threads(2), 0, stream>>>(a);
  else
    residual_norm_kernel<TX, TY, TN, kVec, 4><<<grid, threads(4), 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename TX, typename TY, typename TN>
cudaError_t launch_vec(const NormArgs& a, cudaStream_t stream) {
  return a.vectorised ? launch_typed<TX, TY, TN, true>(a, stream)
                      : launch_typed<TX, TY, TN, false>(a, stream);
}

}  // namespace

cudaError_t launch_residual_norm(const NormArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.width == 0) return cudaSuccess;
  if (a.x_dtype == kDtypeBf16) return launch_vec<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(a, stream);
  if (a.x_dtype == kDtypeF16) return launch_vec<__half, __half, __half>(a, stream);
  if (a.y_dtype == kDtypeBf16) return launch_vec<float, __nv_bfloat16, __nv_bfloat16>(a, stream);
  if (a.y_dtype == kDtypeF16) return launch_vec<float, __half, __half>(a, stream);
  return launch_vec<float, float, float>(a, stream);
}

}  // namespace bsa
