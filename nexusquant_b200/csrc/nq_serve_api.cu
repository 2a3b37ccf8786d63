// extern "C" entry points of the serving operators (declared in include/nexusquant_b200.h): host
// checks, then stream-ordered launches.  Nothing throws, nothing allocates device memory.
#include <cmath>
#include <cstring>

#include "../../include/nexusquant_b200.h"
#include "nq_internal.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int elem_bytes(int dtype) { return dtype == NQ_F32 ? 4 : 2; }
bool head_dim_ok(int d) { return d == 64 || d == 96 || d == 128; }
nq_status_t cuda_status(cudaError_t e) { return e == cudaSuccess ? NQ_OK : NQ_ERR_CUDA; }

// log2 of a page size, -1 for one the kernels do not take
int page_shift(int page_size) {
  return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

// 0 (the default) or a positive, finite logit scale
bool scale_ok(float s) { return s >= 0.0f && s <= 3.0e38f; }

template <typename... S>
bool rows16(int eb, S... strides) {
  return (... && (strides * eb % 16 == 0));
}

nq_status_t pool_args(const nq_pool_t* p, nq::PoolArgs& a) {
  if (!p || !p->k_pages || !p->v_pages || p->layers < 0 || p->n_pages < 0 || p->heads <= 0) return NQ_ERR_INVALID_ARG;
  const int sh = page_shift(p->page_size);
  if (sh < 0) return NQ_ERR_UNSUPPORTED;
  if (p->row_bytes <= 0) return NQ_ERR_INVALID_ARG;
  if (p->row_bytes % 16 || !aligned16(p->k_pages) || !aligned16(p->v_pages)) return NQ_ERR_ALIGNMENT;
  const int64_t page_vecs = (int64_t)p->heads * p->page_size * (p->row_bytes / 16);
  if (page_vecs > (1 << 30) || p->layers > 16384) return NQ_ERR_UNSUPPORTED;
  a.k = p->k_pages; a.v = p->v_pages;
  a.layers = p->layers; a.n_pages = p->n_pages; a.heads = p->heads; a.page_shift = sh;
  a.row_vecs = p->row_bytes / 16; a.page_vecs = (int32_t)page_vecs;
  return NQ_OK;
}

// checks of nq_attend_pages that need no workspace; fills `a`
nq_status_t decode_args(const nq_attend_pages_params_t* p, nq::DecodeArgs& a) {
  if (!p) return NQ_ERR_INVALID_ARG;
  if (p->batch < 0 || p->q_heads <= 0 || p->heads <= 0 || p->n_pages < 0 || p->table_width < 0 || p->max_len < 0 ||
      p->prefix_len < 0)
    return NQ_ERR_INVALID_ARG;
  if (p->dtype != NQ_F16 && p->dtype != NQ_BF16) return NQ_ERR_UNSUPPORTED;
  if (!head_dim_ok(p->head_dim) || p->q_heads % p->heads) return NQ_ERR_UNSUPPORTED;
  const int sh = page_shift(p->page_size);
  if (sh < 0) return NQ_ERR_UNSUPPORTED;
  if (!scale_ok(p->scale)) return NQ_ERR_INVALID_ARG;
  if (p->max_len > (int64_t)p->table_width << sh) return NQ_ERR_INVALID_ARG;
  if ((p->max_len || p->prefix_len) && p->n_pages == 0) return NQ_ERR_INVALID_ARG;
  std::memset(&a, 0, sizeof(a));
  a.q = p->q; a.k_pages = p->k_pages; a.v_pages = p->v_pages; a.out = p->out;
  a.batch = p->batch; a.q_heads = p->q_heads; a.heads = p->heads; a.head_dim = p->head_dim;
  a.n_pages = p->n_pages; a.page_shift = sh;
  a.tables = p->tables; a.lens = p->lens; a.width = p->table_width; a.max_len = p->max_len;
  a.prefix_table = p->prefix_table; a.prefix_len = p->prefix_len;
  a.q_stride_b = p->q_stride_b; a.q_stride_h = p->q_stride_h;
  a.o_stride_b = p->o_stride_b; a.o_stride_h = p->o_stride_h;
  a.scale = p->scale == 0.0f ? 1.0f / sqrtf((float)p->head_dim) : p->scale;
  return NQ_OK;
}

}  // namespace

extern "C" {

nq_status_t nq_norm_rope_qk(const nq_norm_rope_params_t* p, nq_stream_t stream) {
  if (!p || p->tokens < 0 || p->q_heads <= 0 || p->heads <= 0) return NQ_ERR_INVALID_ARG;
  if (p->dtype < 0 || p->dtype > 2) return NQ_ERR_INVALID_ARG;
  if (!head_dim_ok(p->head_dim)) return NQ_ERR_UNSUPPORTED;
  const bool pages = p->k_pages || p->v_pages;
  int sh = 0;
  if (pages) {
    if (!p->k_pages || !p->v_pages || p->n_pages < 0) return NQ_ERR_INVALID_ARG;
    sh = page_shift(p->page_size);
    if (sh < 0) return NQ_ERR_UNSUPPORTED;
  }
  if (p->tokens == 0) return NQ_OK;
  if (!p->q || !p->k || !p->q_out || !p->positions || !p->rope_cos || !p->rope_sin || p->rope_rows <= 0)
    return NQ_ERR_INVALID_ARG;
  if (pages ? (!p->v || !p->slots) : !p->k_out) return NQ_ERR_INVALID_ARG;
  const int eb = elem_bytes(p->dtype);
  const void* al[] = {p->q, p->k, p->v, p->q_weight, p->k_weight, p->rope_cos, p->rope_sin, p->q_out, p->k_out,
                      p->k_pages, p->v_pages};
  for (const void* x : al)
    if (!aligned16(x)) return NQ_ERR_ALIGNMENT;
  if (!rows16(eb, p->q_stride_t, p->q_stride_h, p->k_stride_t, p->k_stride_h, p->qo_stride_t, p->qo_stride_h))
    return NQ_ERR_ALIGNMENT;
  if (pages ? !rows16(eb, p->v_stride_t, p->v_stride_h) : !rows16(eb, p->ko_stride_t, p->ko_stride_h))
    return NQ_ERR_ALIGNMENT;
  nq::NormRopeArgs a;
  std::memset(&a, 0, sizeof(a));
  a.tokens = p->tokens; a.q_heads = p->q_heads; a.heads = p->heads; a.head_dim = p->head_dim;
  a.q = p->q; a.k = p->k; a.v = pages ? p->v : nullptr;
  a.q_stride_t = p->q_stride_t; a.q_stride_h = p->q_stride_h;
  a.k_stride_t = p->k_stride_t; a.k_stride_h = p->k_stride_h;
  a.v_stride_t = p->v_stride_t; a.v_stride_h = p->v_stride_h;
  a.q_weight = p->q_weight; a.k_weight = p->k_weight; a.weight_f32 = p->weight_f32; a.eps = p->eps;
  a.positions = p->positions; a.rope_cos = p->rope_cos; a.rope_sin = p->rope_sin; a.rope_rows = p->rope_rows;
  a.q_out = p->q_out; a.k_out = p->k_out;
  a.qo_stride_t = p->qo_stride_t; a.qo_stride_h = p->qo_stride_h;
  a.ko_stride_t = p->ko_stride_t; a.ko_stride_h = p->ko_stride_h;
  if (pages) {
    a.k_pages = p->k_pages; a.v_pages = p->v_pages; a.n_pages = p->n_pages; a.page_shift = sh; a.slots = p->slots;
  }
  return cuda_status(nq::launch_norm_rope(a, p->dtype, static_cast<cudaStream_t>(stream)));
}

nq_status_t nq_attend_prompt(const nq_attend_prompt_params_t* p, nq_stream_t stream) {
  if (!p || p->n_seqs < 0 || p->q_tokens < 0 || p->k_tokens < 0 || p->q_heads <= 0 || p->heads <= 0)
    return NQ_ERR_INVALID_ARG;
  if (p->dtype != NQ_F16 && p->dtype != NQ_BF16) return NQ_ERR_UNSUPPORTED;
  if (!head_dim_ok(p->head_dim) || p->q_heads % p->heads) return NQ_ERR_UNSUPPORTED;
  if (!scale_ok(p->scale)) return NQ_ERR_INVALID_ARG;
  if (p->n_seqs == 0 || p->q_tokens == 0) return NQ_OK;
  if (!p->q || !p->out || !p->seq_starts || !p->k_starts || (p->k_tokens && (!p->k || !p->v)))
    return NQ_ERR_INVALID_ARG;
  const void* al[] = {p->q, p->k, p->v, p->out};
  for (const void* x : al)
    if (!aligned16(x)) return NQ_ERR_ALIGNMENT;
  if (!rows16(2, p->q_stride_t, p->q_stride_h, p->k_stride_t, p->k_stride_h, p->v_stride_t, p->v_stride_h,
              p->o_stride_t, p->o_stride_h))
    return NQ_ERR_ALIGNMENT;
  nq::PromptArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.lse = p->lse;
  a.n_seqs = p->n_seqs; a.q_tokens = p->q_tokens; a.k_tokens = p->k_tokens;
  a.q_heads = p->q_heads; a.heads = p->heads; a.head_dim = p->head_dim;
  a.starts = p->seq_starts; a.k_starts = p->k_starts;
  a.q_stride_t = p->q_stride_t; a.q_stride_h = p->q_stride_h;
  a.k_stride_t = p->k_stride_t; a.k_stride_h = p->k_stride_h;
  a.v_stride_t = p->v_stride_t; a.v_stride_h = p->v_stride_h;
  a.o_stride_t = p->o_stride_t; a.o_stride_h = p->o_stride_h;
  a.scale = p->scale == 0.0f ? 1.0f / sqrtf((float)p->head_dim) : p->scale;
  return cuda_status(nq::launch_prompt(a, p->dtype, static_cast<cudaStream_t>(stream)));
}

size_t nq_attend_pages_workspace_size(const nq_attend_pages_params_t* p) {
  nq::DecodeArgs a;
  if (decode_args(p, a) != NQ_OK || a.batch == 0) return 0;
  return nq::decode_workspace_bytes(a);
}

nq_status_t nq_attend_pages(const nq_attend_pages_params_t* p, void* workspace, size_t workspace_bytes,
                            nq_stream_t stream) {
  nq::DecodeArgs a;
  const nq_status_t st = decode_args(p, a);
  if (st != NQ_OK) return st;
  if (a.batch == 0) return NQ_OK;
  if (!a.q || !a.out || ((a.max_len || a.prefix_len) && (!a.k_pages || !a.v_pages)) ||
      (a.max_len && (!a.tables || !a.lens)) || (a.prefix_len && !a.prefix_table))
    return NQ_ERR_INVALID_ARG;
  const void* al[] = {a.q, a.k_pages, a.v_pages, a.out};
  for (const void* x : al)
    if (!aligned16(x)) return NQ_ERR_ALIGNMENT;
  if (!rows16(2, a.q_stride_b, a.q_stride_h, a.o_stride_b, a.o_stride_h)) return NQ_ERR_ALIGNMENT;
  const size_t need = nq::decode_workspace_bytes(a);
  if (need && (!workspace || workspace_bytes < need)) return NQ_ERR_WORKSPACE;
  return cuda_status(nq::launch_decode(a, p->dtype, workspace, static_cast<cudaStream_t>(stream)));
}

nq_status_t nq_copy_pages(const nq_pool_t* pool, const int32_t* src, const int32_t* dst, int32_t n,
                          nq_stream_t stream) {
  nq::PoolArgs a;
  const nq_status_t st = pool_args(pool, a);
  if (st != NQ_OK) return st;
  if (n < 0) return NQ_ERR_INVALID_ARG;
  if (n == 0 || a.layers == 0) return NQ_OK;
  if (!src || !dst) return NQ_ERR_INVALID_ARG;
  return cuda_status(nq::launch_copy_pages(a, src, dst, n, static_cast<cudaStream_t>(stream)));
}

nq_status_t nq_compact_pages(const nq_pool_t* pool, int32_t batch, const int32_t* tables, int32_t table_width,
                             const int32_t* kept_idx, int64_t idx_stride, const int32_t* kept_count,
                             int32_t max_kept, const int32_t* dst_tables, int32_t dst_width, nq_stream_t stream) {
  nq::PoolArgs a;
  const nq_status_t st = pool_args(pool, a);
  if (st != NQ_OK) return st;
  if (batch < 0 || table_width < 0 || max_kept < 0 || dst_width < 0 || idx_stride < 0) return NQ_ERR_INVALID_ARG;
  if (batch > 65535 || (int64_t)a.layers * a.heads > 65535 || (int64_t)table_width << a.page_shift > 0x7fffffff ||
      (int64_t)dst_width << a.page_shift > 0x7fffffff)
    return NQ_ERR_UNSUPPORTED;
  if (max_kept > dst_width << a.page_shift || (batch > 1 && max_kept > idx_stride)) return NQ_ERR_INVALID_ARG;
  if (batch == 0 || max_kept == 0 || a.layers == 0) return NQ_OK;
  if (!tables || !kept_idx || !dst_tables) return NQ_ERR_INVALID_ARG;
  nq::CompactArgs c;
  c.tables = tables; c.kept_idx = kept_idx; c.kept_count = kept_count; c.dst_tables = dst_tables;
  c.batch = batch; c.width = table_width; c.dst_width = dst_width; c.max_kept = max_kept; c.idx_stride = idx_stride;
  return cuda_status(nq::launch_compact_pages(a, c, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
