// RMS norm of query and key heads, split-half rotation and the store into cache pages, one pass.
//
// Per row x of d elements (one token, one head), in fp32:
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w          (skipped without a weight)
//   z[i] = y[i] c[i] - y[i + d/2] s[i],  z[i + d/2] = y[i + d/2] c[i] + y[i] s[i]
// with (c, s) the table row of the token's position, the rotation of
// nexusquant/core/rope_utils.py:106-123; rounded once to the tensor's type.  Rotated keys and
// the values go either to dense outputs or to slot = page * page_size + offset of the pages.
//
// Bound by memory: every element is read and written once (2 bytes in, 2 bytes out at fp16).
// Eight lanes (four at d = 64) share a row: lane i holds elements 8i..8i+7 of each half, so both
// halves of a rotation pair are in one thread and the mean is three (two) shuffles.  A group
// takes kRows consecutive heads of one token at once: their loads are all in flight before the
// first is used, and the token's table row is read once for them.
#include <cstring>

#include "../../include/nexusquant_b200.h"
#include "nq_common.cuh"
#include "nq_internal.h"

namespace nq {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRows = 4;  // heads of one token per lane group

template <typename T>
struct Vec8 {
  uint4 u[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Vec8<T> ld8(const T* p) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void st8(T* p, const Vec8<T>& v) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v.u[i];
}

__device__ __forceinline__ void narrow8(const float* o, Vec8<__half>& v) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(o[2 * i], o[2 * i + 1]);
  memcpy(&v, h, 16);
}
__device__ __forceinline__ void narrow8(const float* o, Vec8<__nv_bfloat16>& v) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
  memcpy(&v, h, 16);
}
__device__ __forceinline__ void narrow8(const float* o, Vec8<float>& v) { memcpy(&v, o, 32); }

template <typename T>
__device__ __forceinline__ void widen8(const Vec8<T>& v, float* o) {
  load8(reinterpret_cast<const T*>(&v), o);
}

// 8 norm weights from element i of a vector in the tensors' type or fp32
template <typename T>
__device__ __forceinline__ void weights8(const void* w, int f32, int i, float* o) {
  if (f32) load8(static_cast<const float*>(w) + i, o);
  else widen8(ld8(static_cast<const T*>(w) + i), o);
}

template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LPR = D == 64 ? 4 : 8;  // lanes per row (two of eight idle at d = 96)
  constexpr int HALF = D / 2;
  const int lane = threadIdx.x % LPR;
  const int64_t unit = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) / LPR;
  const int rows = a.q_heads + a.heads + (a.v ? a.heads : 0);
  const int upt = (rows + kRows - 1) / kRows;  // units per token
  const int64_t t = unit / upt;
  const bool live = t < a.tokens;
  const bool on = live && lane < HALF / 8;
  const int r0 = (int)(unit - t * upt) * kRows, e = lane * 8;

  const T* src[kRows];
  Vec8<T> lo[kRows], hi[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = r0 + i;
    src[i] = nullptr;
    if (on && r < rows) {
      if (r < a.q_heads)
        src[i] = static_cast<const T*>(a.q) + t * a.q_stride_t + r * a.q_stride_h;
      else if (r < a.q_heads + a.heads)
        src[i] = static_cast<const T*>(a.k) + t * a.k_stride_t + (r - a.q_heads) * a.k_stride_h;
      else
        src[i] = static_cast<const T*>(a.v) + t * a.v_stride_t + (r - a.q_heads - a.heads) * a.v_stride_h;
      lo[i] = ld8(src[i] + e);
      hi[i] = ld8(src[i] + HALF + e);
    }
  }
  // the token's rotation and its place in the pages
  float c[8], s[8];
  int64_t slot = -1;
  if (on) {
    const int pos = min(max(a.positions[t], 0), a.rope_rows - 1);
    load8(a.rope_cos + (int64_t)pos * HALF + e, c);
    load8(a.rope_sin + (int64_t)pos * HALF + e, s);
    if (a.slots) {
      slot = a.slots[t];
      if (slot >= (int64_t)a.n_pages << a.page_shift) slot = -1;
    }
  }
  const int64_t page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = r0 + i;
    const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + a.heads;
    const void* w = is_v ? nullptr : (is_q ? a.q_weight : a.k_weight);
    float x[16], sum = 0.0f;
    if (src[i]) {
      widen8(lo[i], x);
      widen8(hi[i], x + 8);
#pragma unroll
      for (int j = 0; j < 16; ++j) sum = __fmaf_rn(x[j], x[j], sum);
    }
    if (a.q_weight || a.k_weight) {  // uniform: every lane of the warp takes the shuffles
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (!src[i]) continue;
    T* dst = nullptr;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + t * a.qo_stride_t + r * a.qo_stride_h;
    } else if (a.k_pages) {
      const int h = is_v ? r - a.q_heads - a.heads : r - a.q_heads;
      if (slot >= 0)
        dst = static_cast<T*>(is_v ? a.v_pages : a.k_pages) +
              ((((page * a.heads + h) << a.page_shift) + off) * (int64_t)D);
    } else if (!is_v) {
      dst = static_cast<T*>(a.k_out) + t * a.ko_stride_t + (r - a.q_heads) * a.ko_stride_h;
    }
    if (!dst) continue;
    if (!is_v) {
      if (w) {
        const float inv = 1.0f / sqrtf(__fmaf_rn(sum, 1.0f / D, a.eps));
        float g[16];
        weights8<T>(w, a.weight_f32, e, g);
        weights8<T>(w, a.weight_f32, HALF + e, g + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = x[j] * inv * g[j];
      }
      float y[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = __fmaf_rn(x[j], c[j], -(x[8 + j] * s[j]));
        y[8 + j] = __fmaf_rn(x[8 + j], c[j], x[j] * s[j]);
      }
      narrow8(y, lo[i]);
      narrow8(y + 8, hi[i]);
    }
    st8(dst + e, lo[i]);
    st8(dst + HALF + e, hi[i]);
  }
}

template <typename T>
cudaError_t run_norm_rope(const NormRopeArgs& a, cudaStream_t s) {
  const int rows = a.q_heads + a.heads + (a.v ? a.heads : 0);
  const int64_t units = (int64_t)a.tokens * ((rows + kRows - 1) / kRows);
  const int lpr = a.head_dim == 64 ? 4 : 8;
  const int64_t blocks = (units * lpr + kRopeThreads - 1) / kRopeThreads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const unsigned g = (unsigned)blocks;
  if (a.head_dim == 128) norm_rope_kernel<T, 128><<<g, kRopeThreads, 0, s>>>(a);
  else if (a.head_dim == 96) norm_rope_kernel<T, 96><<<g, kRopeThreads, 0, s>>>(a);
  else norm_rope_kernel<T, 64><<<g, kRopeThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeArgs& a, int dtype, cudaStream_t s) {
  if (dtype == NQ_F16) return run_norm_rope<__half>(a, s);
  if (dtype == NQ_BF16) return run_norm_rope<__nv_bfloat16>(a, s);
  return run_norm_rope<float>(a, s);
}

}  // namespace nq
