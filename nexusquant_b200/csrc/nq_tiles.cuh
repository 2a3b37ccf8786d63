// Attention over tiles of 128 rows x 128 keys on the 5th-generation tensor cores: the kernel of
// attend_prompt (packed causal sequences) and of attend_pages' shared prefix (rows = the queries of
// the whole batch, keys from pages).
//
// Per tile, for a row r with logits s = q k^T (times scale log2(e) = c inside the exponent):
//   m' = max(m, max_j s_j),  p_j = 2^(c s_j - c m'),  l = l 2^(c m - c m') + sum p_j,
//   O = O 2^(c m - c m') + P V,  and O / l at the end.
// The rescaling of O and l is skipped while c (m' - m) <= 8: the weights then stay below 2^8, and
// the quotient O / l does not depend on which m was subtracted.
//
// A row tile holds tq tokens x gp heads that read one KV head (tq = 128 / gp rounded down), so a
// grouped-query model fills the 128 rows from few tokens.  A CTA runs two such streams, each with
// its own softmax warpgroup, so that the exponentials of one overlap the products of the other:
//   SPLIT = false: stream s takes row tile s, both read the same key tiles;
//   SPLIT = true : both take the same row tile, stream s the key tiles of parity s, merged at the
//                  end in shared memory (for grids that would not fill the GPU).
// Warps 0-3 / 4-7: softmax of stream 0 / 1, one thread per row (TMEM lane).  Warp 8: TMA loads of
// Q, K and V (128-byte swizzle) into a ring.  Warp 9: the MMAs: S = Q K^T from shared memory into
// TMEM, O += P V with P read from TMEM (it overwrites S) and V as MN-major operand.  Warps 10-11:
// clear the rows of V that no row of the CTA may see, see scrub().
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cstring>

#include "../../include/nexusquant_b200.h"
#include "nq_common.cuh"
#include "nq_internal.h"
#include "nq_umma.cuh"

namespace nq {
namespace {

constexpr int kTile = 128;         // rows of a row tile, keys of a key tile
constexpr int kTileThreads = 384;
constexpr uint32_t kTileWait = 1u << 22;  // tries of a bounded wait
constexpr float kLog2e = 1.4426950408889634f;

struct TileArgs {
  int32_t q_heads, heads, gp, tq, units;  // gp heads of one KV head per row tile, units = q_heads / gp
  float scale, c;                         // c = scale * log2(e)
  // packed sequences
  const int32_t *starts, *k_starts;
  int32_t n_seqs, q_tokens, k_tokens;
  const void *q, *k, *v;
  int64_t q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, o_stride_t, o_stride_h;
  void* out;
  float* lse;
  // shared prefix in pages
  const int32_t* table;
  int32_t batch, key_len, n_pages, page_shift;
  int32_t row_tiles, tiles_per_split, parts;  // parts: partial results per (sequence, head)
  float *ws_m, *ws_l, *ws_acc;                // [batch, q_heads, parts] x2, [batch, q_heads, parts, D]
};

__device__ __forceinline__ float ex2t(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Bounded wait of a whole warp with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, kTileWait));
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 TMEM columns of the warp's lanes: issue (no wait), and the wait that the values depend on.
__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_tie32(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                       uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

template <typename T>
struct Half16;  // the 16-bit type's pair conversions, MMA type and exponent bits
template <>
struct Half16<__half> {
  static constexpr int kType = 0;
  static constexpr uint32_t kExp = 0x7C007C00u, kOne = 0x04000400u;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float wide(__half x) { return __half2float(x); }
};
template <>
struct Half16<__nv_bfloat16> {
  static constexpr int kType = 1;
  static constexpr uint32_t kExp = 0x7F807F80u, kOne = 0x00800080u;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
};

template <int D, bool SPLIT>
struct TileLayout {
  static constexpr int kBlocks = (D + 63) / 64;          // column blocks of 64 elements (128 bytes)
  static constexpr int kBlock = kTile * 128;             // one column block of a tile
  static constexpr int kItem = kBlocks * kBlock;         // a K, V or Q tile
  static constexpr int kQ = (SPLIT ? 1 : 2) * kItem;
  static constexpr int kStages = (225 * 1024 - kQ) / kItem < 8 ? (225 * 1024 - kQ) / kItem : 8;
  static constexpr int kMerge = SPLIT ? kTile * D * 4 + kTile * 8 : 0;  // stream 1's result, over the ring
  static constexpr int kBytes = kQ + kStages * kItem + 1024;
  static_assert(kMerge <= kStages * kItem, "the merge buffer lies in the ring");
};

// Where a CTA works: rows q0 .. q0 + tokens of q (gp heads each), keys k0 .. k0 + klen, and the last
// key that its first token sees (each further token sees one more).
struct TileJob {
  int q0, tokens, k0, klen, lim0;
};

// Device error word of the bounded waits below (bit 8 of nq_device_error), one per including file.
__device__ unsigned int g_tiles_wait_error;

template <typename T, int D, bool PAGED, bool SPLIT>
__global__ void __launch_bounds__(kTileThreads, 1)
    attend_tiles(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const TileArgs a) {
  using Lo = TileLayout<D, SPLIT>;
  using H = Half16<T>;
  constexpr int NST = Lo::kStages;
  extern __shared__ uint8_t tiles_smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tiles_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sm + Lo::kQ;
  __shared__ uint64_t full[NST], empty[NST], qfull, sfull[2], pready[2], odone[2], vraw[4], scrubbed[4], drain;
  __shared__ uint32_t tmem_base, bad_keys[8];
  __shared__ int err;
  __shared__ TileJob job_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x % a.units;
  const int kh = unit * a.gp / (a.q_heads / a.heads);
  const int ctok = SPLIT ? a.tq : 2 * a.tq;  // tokens per CTA
  int split = 0;

  // ---- which rows and keys
  if (PAGED) {
    const int rest = blockIdx.x / a.units;
    split = rest / a.row_tiles;
    if (tid == 0) {
      const int q0 = (rest % a.row_tiles) * ctok;
      job_s = TileJob{q0, min(ctok, a.batch - q0), 0, a.key_len, a.key_len - 1};
    }
  } else if (warp == 0) {
    // tiles of the sequences before this one, 32 sequences at a time; a sequence's last tile (the
    // longest rows) comes first
    int want = blockIdx.x / a.units;
    TileJob j{0, 0, 0, 0, -1};
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
      const int s = s0 + lane;
      int q0 = 0, nq = 0, tiles = 0;
      if (s < a.n_seqs) {
        q0 = min(max(a.starts[s], 0), a.q_tokens);
        nq = max(min(a.starts[s + 1], a.q_tokens) - q0, 0);
        tiles = (nq + ctok - 1) / ctok;
      }
      int upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const bool mine = want >= upto - tiles && want < upto;
      const uint32_t who = __ballot_sync(0xffffffffu, mine);
      if (who) {
        if (mine) {
          const int k0 = min(max(a.k_starts[s], 0), a.k_tokens);
          const int nk = max(min(a.k_starts[s + 1], a.k_tokens) - k0, 0);
          const int t = (tiles - 1 - (want - (upto - tiles))) * ctok;
          job_s = TileJob{q0 + t, min(ctok, nq - t), k0, nk, nk - nq + t};
        }
        break;
      }
      want -= __shfl_sync(0xffffffffu, upto, 31);
      if (s0 + 32 >= a.n_seqs && lane == 0) job_s = j;
    }
  }
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&qfull, 1);
    mbar_init(&drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], 4);
      mbar_init(&odone[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&vraw[i], 1);
      mbar_init(&scrubbed[i], 2);
    }
    fence_mbar_init();
    err = 0;
  }
  if (tid < 8) bad_keys[tid] = 0u;
  __syncthreads();
  const TileJob job = job_s;
  if (job.tokens == 0) return;  // the grid is sized by a bound: no rows here
  if (warp == 9) tmem_alloc(&tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);  // S (and P): columns 0, 128; O: columns 256, 384

  // ---- key tiles of each stream: tile0 + u (SPLIT: tile0 + 2u + s), u < steps[s]
  int tile0 = 0, steps[2], lim_last;
  {
    lim_last = PAGED ? job.klen - 1 : job.lim0 + job.tokens - 1;
    int n = lim_last < 0 ? 0 : lim_last / kTile + 1;
    if (PAGED) {
      tile0 = split * a.tiles_per_split;
      n = max(min(n, tile0 + a.tiles_per_split) - tile0, 0);
    }
    if (SPLIT) {
      steps[0] = (n + 1) / 2;
      steps[1] = n / 2;
    } else {
      const int lim_a = PAGED ? lim_last : job.lim0 + min(job.tokens, a.tq) - 1;  // stream 0's last row
      steps[0] = PAGED ? n : (lim_a < 0 ? 0 : lim_a / kTile + 1);
      steps[1] = job.tokens > a.tq ? n : 0;
    }
  }
  steps[0] = __shfl_sync(0xffffffffu, steps[0], 0);  // the same in all threads: keep loops on them uniform
  steps[1] = __shfl_sync(0xffffffffu, steps[1], 0);
  const int all = max(steps[0], steps[1]);
  const int lim_first = PAGED ? job.klen - 1 : job.lim0;
  auto tile_of = [&](int u, int s) { return SPLIT ? tile0 + 2 * u + s : tile0 + u; };
  // a tile with a key that some row of the CTA may not see
  auto hidden_keys = [&](int tile) { return tile * kTile + kTile - 1 > lim_first; };

  // The ring holds the tiles in the order in which the MMA warp takes them.  Each role below walks
  // it with the same loop: visit(kind, u, s, first, last) with kind 0 = K, 1 = V; first / last say
  // whether this use takes the item from the ring, and whether it is the last use of it.
  auto walk = [&](auto&& visit) {
    if (all == 0) return;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (steps[s] > 0 && !visit(0, 0, s, SPLIT || s == 0 || steps[0] == 0, SPLIT || s == 1 || steps[1] == 0)) return;
    for (int u = 0; u < all; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int kind = 1; kind >= 0; --kind) {
          const int w = kind ? u : u + 1;
          if (w >= steps[s]) continue;
          if (!visit(kind, w, s, SPLIT || s == 0 || w >= steps[0], SPLIT || s == 1 || w >= steps[1])) return;
        }
  };

  // registers: 168 x 384 at launch, shared out again as 56 x 128 + 224 x 256 (the same sum)
  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
   if (warp == 8) {
    // -------------------------------------------------------------- loads
    if (all > 0) {
      if (lane == 0) {
        const uint32_t bytes = (uint32_t)(a.gp * a.tq * 128 * Lo::kBlocks);
        const int n_q = SPLIT || job.tokens <= a.tq ? 1 : 2;
        mbar_arrive_expect_tx(&qfull, n_q * bytes);
        for (int i = 0; i < n_q; ++i)
          for (int blk = 0; blk < Lo::kBlocks; ++blk)
            tma_3d(sm + i * Lo::kItem + blk * Lo::kBlock, &qmap, blk * 64, unit * a.gp, job.q0 + i * a.tq, &qfull);
      }
      int it = 0, raw = 0;
      bool ok = true;
      walk([&](int kind, int u, int s, bool first, bool) {
        if (!first) return true;
        const int slot = it % NST, round = it / NST;
        ++it;
        if (round > 0 && !warp_wait(&empty[slot], (round - 1) & 1)) { ok = false; --it; return false; }
        uint8_t* dst = ring + slot * Lo::kItem;
        const CUtensorMap* map = kind ? &vmap : &kmap;
        const int tile = tile_of(u, s);
        // values to be scrubbed land on a barrier of their own, and their slot counts as filled
        const bool hidden = kind == 1 && hidden_keys(tile);
        uint64_t* bar = hidden ? &vraw[raw++ & 3] : &full[slot];
        if (hidden && lane == 0) mbar_arrive(&full[slot]);
        if (PAGED) {
          // one lane per page of the tile; pages past the last token are not read
          const int per = kTile >> a.page_shift, left = a.key_len - tile * kTile;
          const int n = min(per, (left + (1 << a.page_shift) - 1) >> a.page_shift);
          if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(n * Lo::kBlocks) * (128u << a.page_shift));
          __syncwarp();
          if (lane < n) {
            const int page = min(max(a.table[tile * per + lane], 0), a.n_pages - 1);
            for (int blk = 0; blk < Lo::kBlocks; ++blk)
              tma_4d(dst + blk * Lo::kBlock + ((lane * 128) << a.page_shift), map, blk * 64, 0, kh, page, bar);
          }
        } else if (lane == 0) {
          mbar_arrive_expect_tx(bar, (uint32_t)Lo::kItem);
          for (int blk = 0; blk < Lo::kBlocks; ++blk)
            tma_3d(dst + blk * Lo::kBlock, map, blk * 64, kh, job.k0 + tile * kTile, bar);
        }
        return true;
      });
      if (!ok) {
        err = 1;
        // copies in flight land before the shared memory is given up
        mbar_wait(&qfull, 0, kTileWait);
        for (int i = 0; i < raw; ++i) mbar_wait(&vraw[i & 3], 0, kTileWait);
        for (int i = max(it - NST, 0); i < it; ++i) mbar_wait(&full[i % NST], (i / NST) & 1, kTileWait);
      }
    }
   } else if (warp == 9) {
    // -------------------------------------------------------------- products
    // The whole warp runs this loop, converged, with one elected lane around the instructions: their
    // descriptors then stay in uniform registers.  Issued by one lane of a divergent warp the same
    // 4 x 8 products took 3400 cycles a step instead of 2190 (2050 is the tensor cores' own time).
    if (all > 0) {
      constexpr uint32_t kIdS = f16_idesc(H::kType, kTile, kTile);
      constexpr uint32_t kIdO = f16_idesc(H::kType, kTile, D) | (1u << 16);  // B (values) MN-major
      // descriptors without the address: K-major, and MN-major with the column blocks kBlock apart
      constexpr uint64_t kDescK = (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
      constexpr uint64_t kDescV = ((uint64_t)(Lo::kBlock >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
      const uint32_t q16 = __shfl_sync(0xffffffffu, smem_u32(sm) >> 4, 0), ring16 = q16 + Lo::kQ / 16;
      int slot = 0, raw = 0;
      uint32_t round = 0;
      int slot_of[2] = {0, 0};  // where the K / V item in use lies
      bool ok = warp_wait(&qfull, 0);
      if (ok)
        walk([&](int kind, int u, int s, bool first, bool last) {
          if (first) {
            slot_of[kind] = slot;
            if (!warp_wait(&full[slot], round)) return ok = false;
            if (++slot == NST) { slot = 0; round ^= 1u; }
            if (kind == 1 && hidden_keys(tile_of(u, s)) && !warp_wait(&scrubbed[raw++ & 3], 0)) return ok = false;
          }
          if (kind == 1 && !warp_wait(&pready[s], u & 1)) return ok = false;
          tc_fence_after();
          const uint32_t item16 = ring16 + slot_of[kind] * (Lo::kItem / 16);
          if (elect_one()) {
            if (kind == 0) {
              const uint32_t qs16 = q16 + (SPLIT ? 0 : s * (Lo::kItem / 16));
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k >> 2) * (Lo::kBlock / 16) + (k & 3) * 2;
                umma_f16(tb + s * 128, kDescK | (qs16 + off), kDescK | (item16 + off), kIdS, k > 0 ? 1u : 0u);
              }
              umma_commit(&sfull[s]);
            } else {
#pragma unroll
              for (int k = 0; k < kTile / 16; ++k)
                umma_f16_ts(tb + 256 + s * 128, tb + s * 128 + k * 8, kDescV | (item16 + k * 128), kIdO, u > 0 || k > 0 ? 1u : 0u);
              if (u == steps[s] - 1) umma_commit(&odone[s]);
            }
            if (last) umma_commit(&empty[slot_of[kind]]);
          }
          __syncwarp();
          return true;
        });
      if (!ok) {
        err = 1;
        // products in flight end before the tensor memory is given up
        if (elect_one()) umma_commit(&drain);
        warp_wait(&drain, 0);
      }
    }
   } else {
    // -------------------------------------------------------------- scrub
    // The product of a zero weight and a value that is not finite would be NaN.  So in tiles with
    // keys that not every row sees, values past the sequence's end are set to zero, and so are rows
    // with a value that is not finite; the latter are remembered, and the rows that do see them get
    // their share at the end.  Tiles that every row sees whole are left alone.  (At most 256 tokens
    // per CTA: three such tiles, one barrier each.)
    int it = 0, raw = 0;
    bool ok = true;
    walk([&](int kind, int u, int s, bool first, bool) {
      if (!first) return true;
      const int slot = it++ % NST, tile = tile_of(u, s);
      if (kind == 0 || !hidden_keys(tile)) return true;
      if (!warp_wait(&vraw[raw & 3], 0)) return ok = false;
      uint8_t* v = ring + slot * Lo::kItem;
      const int key0 = tile * kTile;
      for (int r0 = (warp - 10) * 64; r0 < (warp - 10) * 64 + 64; r0 += 4) {
        const int r = r0 + (lane >> 3), key = key0 + r;
        uint4* p = reinterpret_cast<uint4*>(v + r * 128) + (lane & 7);
        uint32_t odd = 0;
#pragma unroll
        for (int blk = 0; blk < Lo::kBlocks; ++blk) {
          const uint4 x = p[blk * (Lo::kBlock / 16)];
          odd |= ((x.x & H::kExp) + H::kOne) | ((x.y & H::kExp) + H::kOne) | ((x.z & H::kExp) + H::kOne) |
                 ((x.w & H::kExp) + H::kOne);
        }
        const uint32_t who = __ballot_sync(0xffffffffu, (odd & 0x80008000u) != 0) >> (lane & 24);
        const bool past = key >= job.klen;
        if (past || ((who & 0xFFu) && key > lim_first)) {
#pragma unroll
          for (int blk = 0; blk < Lo::kBlocks; ++blk) p[blk * (Lo::kBlock / 16)] = make_uint4(0u, 0u, 0u, 0u);
          const int i = key - max(lim_first + 1, 0);
          if (!past && (lane & 7) == 0 && i < 256) atomicOr(&bad_keys[i >> 5], 1u << (i & 31));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&scrubbed[raw & 3]);
      ++raw;
      return true;
    });
    if (!ok) err = 1;
   }
  } else {
    // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int s = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tb + s * 128 + lanes, tO = tb + 256 + s * 128 + lanes;
    const int tok = row / a.gp;                             // token of the row within its tile
    const int jt = (SPLIT ? 0 : s * a.tq) + tok;            // and within the CTA
    const bool live = tok < a.tq && jt < job.tokens;
    const int lim = PAGED ? lim_last : min(job.lim0 + jt, lim_last);  // the last key that the row sees
    const int lim_min = PAGED ? lim_last : job.lim0 + (SPLIT ? 0 : s * a.tq);
    const int n = steps[s];
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int u = 0; u < n; ++u) {
      if (!warp_wait(&sfull[s], u & 1)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[128];
#pragma unroll
      for (int i = 0; i < 4; ++i) tm_ld32(tS + 32 * i, x + 32 * i);
      tm_wait_ld();
#pragma unroll
      for (int i = 0; i < 4; ++i) tm_tie32(x + 32 * i);
      const int key0 = tile_of(u, s) * kTile;
      if (key0 + kTile - 1 > lim_min) {
        const int seen = lim - key0;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > seen) x[i] = 0xFF800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(x[i]), __uint_as_float(x[4 + i]));
#pragma unroll
      for (int j = 8; j < 128; j += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], __uint_as_float(x[j + i]), __uint_as_float(x[j + 4 + i]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const float mn = fmaxf(m, top);
      const bool grow = mn > m && !((mn - m) * a.c <= 8.0f);
      if (u == 0) {
        m = mn;
      } else if (__any_sync(0xffffffffu, grow)) {
        // S of this step is complete, so the product before it is too: O is at rest
        const float f = !grow ? 1.0f : (m == -INFINITY ? 0.0f : ex2t((m - mn) * a.c));
        if (grow) m = mn;
        l *= f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tm_ld32(tO + 32 * i, o);
          tm_wait_ld();
          tm_tie32(o);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
          tm_st32(tO + 32 * i, o);
        }
        tm_wait_st();
      }
      const float mc = m == -INFINITY ? 0.0f : m * a.c;
      const u64 c2 = pk(a.c, a.c), mc2 = pk(-mc, -mc);
      u64 sum[2] = {0ull, 0ull};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float y0, y1;
          upk(fma2(pk(__uint_as_float(x[64 * i + 2 * j]), __uint_as_float(x[64 * i + 2 * j + 1])), c2, mc2), y0, y1);
          y0 = ex2t(y0);
          y1 = ex2t(y1);
          sum[j & 1] = add2(sum[j & 1], pk(y0, y1));
          w[j] = H::pack(y0, y1);
        }
        tm_st32(tS + 32 * i, w);
      }
      float s0, s1;
      upk(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tm_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pready[s]);
    }
    if (ok && n > 0) ok = warp_wait(&odone[s], 0);
    if (SPLIT && ok && steps[s ^ 1] > 0) ok = warp_wait(&odone[s ^ 1], 0);  // the ring is free
    if (!ok) err = 1;
    tc_fence_after();
    __syncwarp();

    // ---- O of the row, 32 columns at a time
    const int head = unit * a.gp + row % a.gp;
    const float mc = m == -INFINITY ? 0.0f : m * a.c;
    bool any_bad = false;
    if (!PAGED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) any_bad |= bad_keys[i] != 0u;
    }
    auto o_chunk = [&](int i, float* o) {
      if (n > 0) {
        uint32_t r[32];
        tm_ld32(tO + 32 * i, r);
        tm_wait_ld();
        tm_tie32(r);
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(r[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = 0.0f;
      }
      if (!PAGED && any_bad && live) {
        // values that were taken out of the product, for the rows that see them
        for (int b = 0; b < 256; ++b) {
          if (!(bad_keys[b >> 5] >> (b & 31) & 1u)) continue;
          const int key = max(lim_first + 1, 0) + b;
          if (key > lim || (SPLIT && ((key / kTile - tile0) & 1) != s)) continue;
          const T* q = static_cast<const T*>(a.q) + (int64_t)(job.q0 + jt) * a.q_stride_t + head * a.q_stride_h;
          const T* k = static_cast<const T*>(a.k) + (int64_t)(job.k0 + key) * a.k_stride_t + kh * a.k_stride_h;
          const T* v = static_cast<const T*>(a.v) + (int64_t)(job.k0 + key) * a.v_stride_t + kh * a.v_stride_h;
          float dot = 0.0f;
          for (int e = 0; e < D; ++e) dot = fmaf(H::wide(q[e]), H::wide(k[e]), dot);
          const float p = ex2t(fmaf(dot, a.c, -mc));
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = fmaf(p, H::wide(v[32 * i + j]), o[j]);
        }
      }
    };
    float* mg = reinterpret_cast<float*>(ring);  // [D / 4][128 rows] float4, then m, l
    float f_own = 1.0f, f_other = 0.0f;
    if (SPLIT) {
      float* ml = mg + kTile * D;
      if (s == 1) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          float o[32];
          o_chunk(i, o);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<float4*>(mg)[(8 * i + j) * kTile + row] =
                make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
        ml[2 * row] = m;
        ml[2 * row + 1] = l;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (s == 0) {
        const float mo = ml[2 * row], lo = ml[2 * row + 1], mm = fmaxf(m, mo);
        f_own = m == -INFINITY ? 0.0f : (m == mm ? 1.0f : ex2t((m - mm) * a.c));
        f_other = mo == -INFINITY ? 0.0f : (mo == mm ? 1.0f : ex2t((mo - mm) * a.c));
        l = l * f_own + lo * f_other;
        m = mm;
      }
    }
    if (!SPLIT || s == 0) {
      const int64_t t = job.q0 + jt;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // a row without keys gives zeros
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float o[32];
        o_chunk(i, o);
        if (SPLIT) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 y = reinterpret_cast<const float4*>(mg)[(8 * i + j) * kTile + row];
            o[4 * j] = o[4 * j] * f_own + y.x * f_other;
            o[4 * j + 1] = o[4 * j + 1] * f_own + y.y * f_other;
            o[4 * j + 2] = o[4 * j + 2] * f_own + y.z * f_other;
            o[4 * j + 3] = o[4 * j + 3] * f_own + y.w * f_other;
          }
        }
        if (!live) continue;
        if (PAGED) {
          float4* dst = reinterpret_cast<float4*>(a.ws_acc + ((t * a.q_heads + head) * a.parts + split) * D + 32 * i);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + t * a.o_stride_t + head * a.o_stride_h + 32 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = H::pack(o[8 * j + 2 * e] * inv, o[8 * j + 2 * e + 1] * inv);
            dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (live && PAGED) {
        a.ws_m[(t * a.q_heads + head) * a.parts + split] = m == -INFINITY ? m : m * a.c;
        a.ws_l[(t * a.q_heads + head) * a.parts + split] = l;
      } else if (live && a.lse) {
        a.lse[t * a.q_heads + head] = l > 0.0f || l != l ? m * a.scale + logf(l) : -INFINITY;
      }
    }
  }
  __syncwarp();
  if (err && lane == 0) atomicOr(&g_tiles_wait_error, 1u);
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tb, 512);
}

// --------------------------------------------------------------------------------- host side
inline PFN_cuTensorMapEncodeTiled_v12000 tiles_encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// Map over `rank` dimensions of a 16-bit tensor (innermost first, strides of the others in elements)
// with a box of 64 x box[1] x ..., 128-byte swizzle, zeros outside.
inline bool tiles_map(CUtensorMap* m, const void* base, int type, int rank, const cuuint64_t* dims, const int64_t* strides,
                      const cuuint32_t* box) {
  const auto fn = tiles_encode_fn();
  if (!fn) return false;
  cuuint64_t bytes[4];
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = (cuuint64_t)strides[i] * 2;
  return fn(m, type == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
            const_cast<void*>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool PAGED, bool SPLIT>
cudaError_t run_tiles(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileArgs& a, int64_t ctas,
                      cudaStream_t s) {
  auto kern = attend_tiles<T, D, PAGED, SPLIT>;
  constexpr int smem = TileLayout<D, SPLIT>::kBytes;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (ctas <= 0 || ctas > 0x7fffffff) return cudaErrorInvalidValue;
  kern<<<(unsigned)ctas, kTileThreads, smem, s>>>(q, k, v, a);
  return cudaGetLastError();
}

// Read and clear the error word.
inline cudaError_t tiles_error(unsigned int* bits, cudaStream_t s) {
  unsigned int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_tiles_wait_error, sizeof(v), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && v) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_tiles_wait_error, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  *bits = v;
  return e;
}

inline int device_sms() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

}  // namespace
}  // namespace nq
