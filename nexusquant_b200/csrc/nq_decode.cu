// Decode attention over pages: one query token per sequence attends to a prefix that the whole
// batch shares and then to its own pages, in one pass with a running maximum and sum.  One warp
// per (sequence, head).
#include "../../include/nexusquant_b200.h"
#include "nq_common.cuh"
#include "nq_internal.h"

namespace nq {
namespace {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float x, __half* p) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

template <typename T, int D>
__global__ void __launch_bounds__(32) decode_kernel(const DecodeArgs a) {
  const int lane = threadIdx.x, head = blockIdx.x, b = blockIdx.y;
  const int kh = head / (a.q_heads / a.heads);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride_b + head * a.q_stride_h;
  T* out = static_cast<T*>(a.out) + b * a.o_stride_b + head * a.o_stride_h;
  const int own = a.max_len ? min(max(a.lens[b], 0), a.max_len) : 0;
  float qv[D / 32], acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { qv[i] = to_f(q[lane + 32 * i]) * a.scale; acc[i] = 0.0f; }
  float m = -INFINITY, l = 0.0f;
  for (int part = 0; part < 2; ++part) {
    const int32_t* table = part ? a.tables + (int64_t)b * a.width : a.prefix_table;
    const int n = part ? own : a.prefix_len;
    for (int j = 0; j < n; ++j) {
      const int page = min(max(table[j >> a.page_shift], 0), a.n_pages - 1);
      const int64_t row = ((((int64_t)page * a.heads + kh) << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * D;
      const T* k = static_cast<const T*>(a.k_pages) + row;
      const T* v = static_cast<const T*>(a.v_pages) + row;
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) x = fmaf(qv[i], to_f(k[lane + 32 * i]), x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      const float mn = fmaxf(m, x), f = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(x - mn);
      m = mn;
      l = fmaf(l, f, p);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(acc[i], f, p * to_f(v[lane + 32 * i]));
    }
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) from_f(own + a.prefix_len > 0 ? acc[i] / l : 0.0f, out + lane + 32 * i);
}

template <typename T>
cudaError_t run_decode(const DecodeArgs& a, cudaStream_t s) {
  const dim3 g(a.q_heads, a.batch);
  if (a.head_dim == 128) decode_kernel<T, 128><<<g, 32, 0, s>>>(a);
  else if (a.head_dim == 96) decode_kernel<T, 96><<<g, 32, 0, s>>>(a);
  else decode_kernel<T, 64><<<g, 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t decode_workspace_bytes(const DecodeArgs&) { return 0; }

cudaError_t launch_decode(const DecodeArgs& a, int dtype, void*, cudaStream_t s) {
  return dtype == NQ_F16 ? run_decode<__half>(a, s) : run_decode<__nv_bfloat16>(a, s);
}

}  // namespace nq
