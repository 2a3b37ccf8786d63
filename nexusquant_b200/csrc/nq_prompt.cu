// Causal attention of packed prompts: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j
// that query i sees, in one pass with a running maximum and sum.  One warp per (query, head).
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
__global__ void __launch_bounds__(128) prompt_kernel(const PromptArgs a) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, head = blockIdx.y;
  if (t >= a.q_tokens) return;
  int s = 0;
  while (s < a.n_seqs && t >= a.starts[s + 1]) ++s;
  T* out = static_cast<T*>(a.out) + t * a.o_stride_t + head * a.o_stride_h;
  if (s == a.n_seqs || t < a.starts[s]) return;
  const int k0 = min(max(a.k_starts[s], 0), a.k_tokens), k1 = min(max(a.k_starts[s + 1], k0), a.k_tokens);
  const int nq = a.starts[s + 1] - a.starts[s];
  const int seen = k1 - k0 - nq + (t - a.starts[s]) + 1;  // keys that this query sees
  const int kh = head / (a.q_heads / a.heads);
  const T* q = static_cast<const T*>(a.q) + t * a.q_stride_t + head * a.q_stride_h;
  float qv[D / 32], acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { qv[i] = to_f(q[lane + 32 * i]) * a.scale; acc[i] = 0.0f; }
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < seen; ++j) {
    const T* k = static_cast<const T*>(a.k) + (int64_t)(k0 + j) * a.k_stride_t + kh * a.k_stride_h;
    const T* v = static_cast<const T*>(a.v) + (int64_t)(k0 + j) * a.v_stride_t + kh * a.v_stride_h;
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
#pragma unroll
  for (int i = 0; i < D / 32; ++i) from_f(seen > 0 ? acc[i] / l : 0.0f, out + lane + 32 * i);
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.q_heads + head] = seen > 0 ? m + logf(l) : -INFINITY;
}

template <typename T>
cudaError_t run_prompt(const PromptArgs& a, cudaStream_t s) {
  const dim3 g((a.q_tokens + 3) / 4, a.q_heads);
  if (a.head_dim == 128) prompt_kernel<T, 128><<<g, 128, 0, s>>>(a);
  else if (a.head_dim == 96) prompt_kernel<T, 96><<<g, 128, 0, s>>>(a);
  else prompt_kernel<T, 64><<<g, 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prompt(const PromptArgs& a, int dtype, cudaStream_t s) {
  return dtype == NQ_F16 ? run_prompt<__half>(a, s) : run_prompt<__nv_bfloat16>(a, s);
}

}  // namespace nq
