// TMA pieces that the tensor-core kernels over a paged cache share: tensor maps
// of the queries and caches, and the load of a 128-key tile page by page.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "afa_common.cuh"
#include "afa_paged.cuh"
#include "afa_tmap.h"

namespace afa {

__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// True in one lane of the (whole) warp. The compiler knows that a branch on it
// is one thread's: the tcgen05 instructions behind it take their operands from
// uniform registers with fewer instructions than behind `lane == 0` (39 against
// 49 cycles for each of a run of small MMAs on an idle SM), which counts where
// the octic warps compete for the same issue slots.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
  return e != 0;
}

// A value that every lane of the warp holds, told to the compiler.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Place in a ring of N barriers and slots.
template <int N>
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step(int by = 1) {  // by < N
    slot += by;
    if (slot >= N) {
      slot -= N;
      phase ^= 1u;
    }
  }
};

// The pages of a key tile, one per lane of the loading warp (one in all when a
// page holds a whole tile).
struct KvPages {
  int per_tile, box_rows, ps;

  __device__ __forceinline__ explicit KvPages(const PagedArgs& a) {
    ps = 1 << a.page_shift;
    per_tile = ps < kPagedTile ? kPagedTile >> a.page_shift : 1;
    box_rows = ps < kPagedTile ? ps : kPagedTile;
  }

  // This lane's page of tile i of a piece; outside the cache, where TMA fills
  // zeros, behind the request's last token and for an entry that names no page.
  __device__ __forceinline__ int page(const PagedArgs& a, const PagedPiece& p, int i) const {
    const int lane = threadIdx.x & 31;
    const int key = (p.t0 + i) * kPagedTile + lane * box_rows;
    if (p.t0 + i >= p.t1 || lane >= per_tile || key >= p.r.len) return a.num_pages;
    const int e = a.table[p.b * a.table_ld + (key >> a.page_shift)];
    return e >= 0 && e < a.num_pages ? e : a.num_pages;
  }

  // Loads tile i (64-column halves, 16 KB apart) into dst; all lanes call it.
  template <int KSUB>
  __device__ __forceinline__ void load(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, const PagedPiece& p, int i,
                                       int page) const {
    const int lane = threadIdx.x & 31;
    const int key = (p.t0 + i) * kPagedTile + lane * box_rows;
    if (lane < per_tile)
      for (int h = 0; h < KSUB; ++h)
        tma_load_4d(dst + h * 128 * 128 + lane * box_rows * 128, map, bar, 64 * h, key & (ps - 1), p.h, page);
  }
};

// Clears the rows of a V tile between a request's last token (`lim` keys of the
// tile are its) and the end of that page: they may hold anything, and 0 * NaN is
// NaN. The warp calls it after the tile has arrived, before the product.
template <int KSUB>
__device__ __forceinline__ void clear_v_tail(uint8_t* tile, int lim, int page_shift, int lane) {
  if (lim >= kPagedTile) return;
  const int ps = 1 << page_shift;
  const int end = min(kPagedTile, (lim + ps - 1) & ~(ps - 1));
  for (int x = lim * 8 + lane; x < end * 8; x += 32)
#pragma unroll
    for (int h = 0; h < KSUB; ++h)
      st_shared_v4(smem_u32(tile + h * 128 * 128 + x * 16), make_uint4(0u, 0u, 0u, 0u));
  fence_proxy_async_shared();
  __syncwarp();
}

// A bf16 tensor map of four dimensions, 128-byte swizzle; strides in elements,
// from the second dimension on.
inline bool map_4d(CUtensorMap* m, const void* base, const long long (&dims)[4], const long long (&strides)[3],
                   const int (&box)[4]) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], e[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
  }
  for (int i = 0; i < 3; ++i) s[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), d, s, b, e,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries: a box is `tokens` tokens of a group's G heads; caches: 64 channels of
// up to 128 rows of a page.
inline bool paged_tmaps(const PagedArgs& a, int tokens, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v) {
  const int ps = 1 << a.page_shift, rows = ps < kPagedTile ? ps : kPagedTile;
  return map_4d(q, a.q, {a.D, a.G, a.Hkv, a.T}, {a.q_sh, a.q_sh * a.G, a.q_st}, {64, a.G, 1, tokens}) &&
         map_4d(k, a.k, {a.D, ps, a.Hkv, a.num_pages}, {a.k_sr, a.k_sh, a.k_sp}, {64, rows, 1, 1}) &&
         map_4d(v, a.v, {a.D, ps, a.Hkv, a.num_pages}, {a.v_sr, a.v_sh, a.v_sp}, {64, rows, 1, 1});
}

}  // namespace afa
