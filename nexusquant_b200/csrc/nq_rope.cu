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
// takes kRows heads of one token and one kind at once: their loads are all in flight before the
// first is used, and the products of weights and rotation (w c, w s) are formed once for them:
//   z[i] = (x[i] (w c)[i] - x[i + d/2] (w' s)[i]) / rms,  with w' the second half's weights.
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

// 8 norm weights from element i of a vector in the tensors' type or fp32; ones without a vector
template <typename T>
__device__ __forceinline__ void weights8(const void* w, int f32, int i, float* o) {
  if (!w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 1.0f;
  } else if (f32) {
    load8(static_cast<const float*>(w) + i, o);
  } else {
    widen8(ld8(static_cast<const T*>(w) + i), o);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LPR = D == 64 ? 4 : 8;  // lanes per row (two of eight idle at d = 96)
  constexpr int HALF = D / 2;
  const int lane = threadIdx.x % LPR, e = lane * 8;
  const int64_t unit = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) / LPR;
  // units of a token: its queries, its keys, its values
  const int uq = (a.q_heads + kRows - 1) / kRows, uk = (a.heads + kRows - 1) / kRows;
  const int upt = uq + (a.v ? 2 : 1) * uk;
  const int64_t t = unit / upt;
  const int u = (int)(unit - t * upt);
  const int kind = u < uq ? 0 : (u < uq + uk ? 1 : 2);  // queries, keys, values
  const int h0 = (kind == 0 ? u : kind == 1 ? u - uq : u - uq - uk) * kRows;
  const bool on = t < a.tokens && lane < HALF / 8;
  const int n = on ? min(kRows, (kind == 0 ? a.q_heads : a.heads) - h0) : 0;

  const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + e +
                 t * (kind == 0 ? a.q_stride_t : kind == 1 ? a.k_stride_t : a.v_stride_t);
  const int64_t step = kind == 0 ? a.q_stride_h : kind == 1 ? a.k_stride_h : a.v_stride_h;
  Vec8<T> lo[kRows], hi[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (i < n) {
      lo[i] = ld8(src + (h0 + i) * step);
      hi[i] = ld8(src + (h0 + i) * step + HALF);
    }
  // where the rows go
  T* dst = nullptr;
  int64_t dstep = 0;
  if (n > 0) {
    if (kind == 0) {
      dst = static_cast<T*>(a.q_out) + t * a.qo_stride_t;
      dstep = a.qo_stride_h;
    } else if (!a.k_pages) {
      dst = static_cast<T*>(a.k_out) + t * a.ko_stride_t;
      dstep = a.ko_stride_h;
    } else {
      const int64_t slot = a.slots[t], page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
      if (slot >= 0 && page < a.n_pages)
        dst = static_cast<T*>(kind == 2 ? a.v_pages : a.k_pages) + (((page * a.heads) << a.page_shift) + off) * (int64_t)D;
      dstep = (int64_t)D << a.page_shift;
    }
    if (dst) dst += e + h0 * dstep;
  }
  const void* w = kind == 0 ? a.q_weight : a.k_weight;
  const bool norm = kind < 2 && w;
  u64 lc[4], hs[4], hc[4], ls[4];  // (w c), (w' s), (w' c), (w s) of the 8 pairs, packed
  if (kind < 2 && dst) {
    const int pos = min(max(a.positions[t], 0), a.rope_rows - 1);
    float c[8], s[8], wl[8], wh[8];
    load8(a.rope_cos + (int64_t)pos * HALF + e, c);
    load8(a.rope_sin + (int64_t)pos * HALF + e, s);
    weights8<T>(w, a.weight_f32, e, wl);
    weights8<T>(w, a.weight_f32, HALF + e, wh);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 c2 = pk(c[2 * j], c[2 * j + 1]), s2 = pk(s[2 * j], s[2 * j + 1]);
      const u64 l2 = pk(wl[2 * j], wl[2 * j + 1]), h2 = pk(wh[2 * j], wh[2 * j + 1]);
      lc[j] = mul2(l2, c2);
      hs[j] = mul2(h2, pk(-s[2 * j], -s[2 * j + 1]));
      hc[j] = mul2(h2, c2);
      ls[j] = mul2(l2, s2);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float x[16];
    u64 sum2 = 0ull;
    if (kind < 2 && i < n) {
      widen8(lo[i], x);
      widen8(hi[i], x + 8);
      if (norm) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum2 = fma2(pk(x[2 * j], x[2 * j + 1]), pk(x[2 * j], x[2 * j + 1]), sum2);
      }
    }
    float inv = 1.0f;
    if (a.q_weight || a.k_weight) {  // uniform: every lane of the warp takes the shuffles
      float s0, s1;
      upk(sum2, s0, s1);
      float sum = s0 + s1;
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (norm) inv = 1.0f / sqrtf(__fmaf_rn(sum, 1.0f / D, a.eps));
    }
    if (i >= n || !dst) continue;
    if (kind < 2) {
      float y[16];
      const u64 inv2 = pk(inv, inv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 x0 = pk(x[2 * j], x[2 * j + 1]), x1 = pk(x[8 + 2 * j], x[9 + 2 * j]);
        upk(mul2(fma2(x0, lc[j], mul2(x1, hs[j])), inv2), y[2 * j], y[2 * j + 1]);
        upk(mul2(fma2(x1, hc[j], mul2(x0, ls[j])), inv2), y[8 + 2 * j], y[9 + 2 * j]);
      }
      narrow8(y, lo[i]);
      narrow8(y + 8, hi[i]);
    }
    st8(dst + i * dstep, lo[i]);
    st8(dst + i * dstep + HALF, hi[i]);
  }
}

template <typename T>
cudaError_t run_norm_rope(const NormRopeArgs& a, cudaStream_t s) {
  const int64_t units = (int64_t)a.tokens * ((a.q_heads + kRows - 1) / kRows +
                                             (a.v ? 2 : 1) * ((a.heads + kRows - 1) / kRows));
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
