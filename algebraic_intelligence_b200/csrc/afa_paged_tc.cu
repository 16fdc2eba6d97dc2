// AFA over a paged cache on the 5th-generation tensor cores (tcgen05 + TMEM),
// bf16, head_dim 64 or 128. Math and work split: afa_paged.cu, afa_paged.cuh.
//
// One persistent CTA per SM walks its share of the work units. Two "streams" of
// eight octic warps each map scores, as in the prefill kernels: one stream's
// map runs while the tensor core computes the other's P.V and next scores. A
// unit is two 128-row query tiles at most, and what the streams are depends on
// its rows:
//   pair   more rows than a tile: stream i maps query tile i; both use the same
//          K/V tile, which is read once for up to 256 rows;
//   split  at most one tile of rows (single tokens, most trees): stream i maps
//          the key tiles i, i + 2, ... of the piece for the same query tile.
//          Octic sums only add, so the two O accumulators meet in the epilogue.
// Warps whose 32 rows are all beyond the unit's last row skip the map.
//
//   warps 16,18 TMA, K (and Q) and V: lane l loads page l of a tile (64-column
//               halves, 128-byte swizzle). Tiles are loaded in the order the tensor core
//               consumes them: LA K tiles first (2 split, 1 pair), then V_i,
//               K_{i + LA}, so ring slots free up in order. Pages behind a
//               request's last token and entries that name no page are given a
//               coordinate outside the cache, where TMA fills zeros.
//   warp 17     allocates TMEM and issues every tcgen05.mma. In a request's last
//               tile it first clears the V rows between its last token and the
//               end of that page: they may hold anything, and 0 * NaN is NaN.
//   warps 0-15  octic map and epilogue. Visibility is a 32-bit word per row and
//               32-key chunk (paged_seen); tiles wholly before the new tokens
//               take the unmasked map.
// Query tile: a tile is floor(128 / G) tokens of G heads, loaded by one TMA box
// (64 columns, G heads, tokens), so a group's heads share every K/V tile.
// TMEM columns: S0/P0 [0,128), S1/P1 [128,256), O0 [256,256+D), O1 [256+D, ...).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "afa_common.cuh"
#include "afa_internal.h"
#include "afa_paged.cuh"
#include "afa_paged_tma.cuh"
#include "afa_tc_shared.cuh"

namespace afa {
namespace {

template <int HD>
struct PgCfg {
  static constexpr int kOcticWarps = 16;
  static constexpr int kTmaWarp = 16;
  static constexpr int kMmaWarp = 17;
  static constexpr int kTmaVWarp = 18;
  static constexpr int kThreads = 19 * 32;
  static constexpr int KSUB = HD / 64;
  static constexpr int SUB_BYTES = 128 * 128;  // 128 rows x 128 B
  static constexpr int TILE_BYTES = KSUB * SUB_BYTES;
  static constexpr int NSLOT = (HD == 128) ? 5 : 8;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = 2 * TILE_BYTES;
  static constexpr int BAR_OFF = KV_OFF + NSLOT * TILE_BYTES;
  static constexpr int NBAR = 4 + 2 * NSLOT + 2 + 2 + 2 + 1;
  static constexpr int TMEM_OFF = BAR_OFF + NBAR * 8;
  static constexpr int RED_OFF = TMEM_OFF + 8;               // fp32 row sums [stream][row]
  static constexpr int SHARE_OFF = RED_OFF + 2 * 128 * 4;    // scratch of paged_share
  static constexpr int SMEM_BYTES = SHARE_OFF + (kThreads / 32 + 4) * 8 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
  static constexpr uint32_t TMEM_COLS = 512;
  __device__ static constexpr uint32_t s_col(int i) { return static_cast<uint32_t>(i) * 128u; }
  __device__ static constexpr uint32_t o_col(int i) { return 256u + static_cast<uint32_t>(i) * HD; }
  // P of keys [16 kk, 16 kk + 16): the chunk [32c, 32c + 32) is packed into columns [32c, 32c + 16).
  __device__ static constexpr uint32_t p_col(int kk) {
    return static_cast<uint32_t>((kk >> 1) * 32 + (kk & 1) * 8);
  }
};

// Octic map of one 32-column chunk of a score row into 16 packed bf16 pairs;
// returns the fp32 sum of the weights. MASK: bit e of `seen` tells whether the
// row sees key e.
// The weights enter the second product as one bf16 (half a step, 2^-8 of each;
// their sum does not), as in the prefill kernels: here the chain of product, map
// and product bounds a tile, and a second part, which the transposed kernel has
// room for, would be half as much tensor work again and twice the stores to
// TMEM. Outputs of rows of few keys are up to 3.4e-3 of the largest off, 2.3e-3
// over thousands of keys, where their own rounding to bf16 is up to 1.7e-3.
template <bool MASK, bool EXACT>
__device__ __forceinline__ float map_seen(const uint32_t (&sv)[32], uint32_t (&pk)[16], float scale, unsigned seen) {
  float2 acc = make_float2(0.f, 0.f);
  const float2 sc = make_float2(scale, scale);
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 s = __fmul2_rn(make_float2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), sc);
    float2 p = EXACT ? octic_exact2(s) : octic_fast2(s);
    if (MASK) {
      p.x = (seen & (1u << e)) ? p.x : 0.f;
      p.y = (seen & (2u << e)) ? p.y : 0.f;
    }
    acc = __fadd2_rn(acc, p);
    pk[e >> 1] = pack_bf16x2(p.x, p.y);
  }
  return acc.x + acc.y;
}

// The chunk at s_tm, mapped with the single-MUFU form, and again with the exact
// one when some row that sees a key of it has all its weights so far and the
// chunk's deep in the negative tail (see kTailChunkSum, kTailRowSum).
template <bool MASK>
__device__ __forceinline__ float map_seen_tmem(uint32_t s_tm, uint32_t (&pk)[16], float scale, unsigned seen,
                                               bool live, bool check) {
  uint32_t sv[32];
  tmem_ld32(s_tm, sv);
  tmem_ld_wait();
  float part = map_seen<MASK, false>(sv, pk, scale, seen);
  if (check && __any_sync(0xffffffffu, live && (!MASK || seen != 0u) && part < kTailChunkSum)) {
    tmem_ld32(s_tm, sv);
    tmem_ld_wait();
    part = map_seen<MASK, true>(sv, pk, scale, seen);
  }
  return part;
}

// What a piece is to the streams.
struct PgPiece {
  bool split;
  int n;        // key tiles
  int rows[2];  // live rows of each query tile
  int n0;       // pair: key tiles of query tile 0 within the piece (<= n)
};

__device__ __forceinline__ PgPiece pg_piece(const PagedArgs& a, const PagedPiece& p, int tile_rows) {
  PgPiece g;
  const long long row0 = static_cast<long long>(p.u) * a.unit_rows;
  const long long left = static_cast<long long>(p.r.n) * a.G - row0;
  const int rows = left < a.unit_rows ? static_cast<int>(left) : a.unit_rows;
  g.split = rows <= tile_rows;
  g.rows[0] = rows < tile_rows ? rows : tile_rows;
  g.rows[1] = rows - g.rows[0];
  g.n = p.tiles > 0 ? p.t1 - p.t0 : 0;
  g.n0 = g.n;
  if (!g.split) {
    const int vis = (paged_visible(a, p.r, row0 + tile_rows) + kPagedTile - 1) / kPagedTile;
    g.n0 = max(0, min(g.n, vis - p.t0));
  }
  return g;
}

// The two query buffers: a pair takes both, a split piece the one used less, so
// that a split piece's queries load while the piece before still runs. Loader
// and MMA warp keep the same count.
struct QBuffers {
  int uses[2] = {0, 0};
  int first = 0, last = 0;  // of this piece
  __device__ __forceinline__ void next(bool split) {
    first = split && uses[1] < uses[0] ? 1 : 0;
    last = split ? first : 1;
  }
  __device__ __forceinline__ uint32_t phase(int i) const { return (i ? uses[1] : uses[0]) & 1; }
  __device__ __forceinline__ void take(int i) {
    if (i)
      ++uses[1];
    else
      ++uses[0];
  }
};

template <int HD>
__global__ void __launch_bounds__(608, 1)
    afa_paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedArgs a) {
  using C = PgCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 2;
  uint64_t* kv_full = bars + 4;
  uint64_t* kv_empty = kv_full + C::NSLOT;
  uint64_t* s_full = kv_empty + C::NSLOT;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TMEM_OFF);
  float* red = reinterpret_cast<float*>(smem + C::RED_OFF);
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int tile_tok = 128 / a.G;  // tokens per query tile
  const int tile_rows = tile_tok * a.G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int s = 0; s < C::NSLOT; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_empty + s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 8);  // one elected arrive per octic warp of the stream
      mbar_init(o_full + i, 1);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    paged_meta_clear(a.meta);
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // see paged_combine_kernel
  PagedWalk<true> walk;
  walk.init(a, paged_share<C::kThreads, true>(a, reinterpret_cast<long long*>(smem + C::SHARE_OFF)));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  PagedPiece p;

  if (warp == C::kTmaWarp || warp == C::kTmaVWarp) {
    // ------------------------------------------------------------------ TMA
    const bool is_v = warp == C::kTmaVWarp;
    KvPages pages(a);
    int u = 0;
    QBuffers qb;
    bool ok = true;
    while (ok && walk.next(a, p)) {
      if (!is_v && lane == 0) paged_meta_piece(a.meta, p);
      const PgPiece g = pg_piece(a, p, tile_rows);
      if (g.n == 0) continue;
      qb.next(g.split);
      for (int i = qb.first; ok && !is_v && i <= qb.last; ++i) {
        // The last S = Q K^T of the piece that held this buffer must be done.
        ok = __all_sync(0xffffffffu, mbar_wait(q_empty + i, qb.phase(i) ^ 1, a.status, kDevTimeoutProducer));
        if (ok && lane == 0) {
          mbar_arrive_expect_tx(q_full + i, C::KSUB * tile_rows * 128);
          for (int h = 0; h < C::KSUB; ++h)
            tma_load_4d(smem + C::Q_OFF + (i * C::KSUB + h) * C::SUB_BYTES, &tm_q, q_full + i, 64 * h, 0, p.h,
                        p.r.tok0 + (p.u * 2 + i - qb.first) * tile_tok);
        }
        if (ok) qb.take(i);
      }
      if (!ok) break;
      auto load = [&](int i, bool v, int page) {  // tile i of the piece
        const int slot = u++ % C::NSLOT;
        if (v != is_v) return;  // the other warp's
        if (!(ok = ok && __all_sync(0xffffffffu, mbar_wait(kv_empty + slot, (((u - 1) / C::NSLOT) & 1) ^ 1, a.status,
                                                           kDevTimeoutProducer))))
          return;
        if (lane == 0) mbar_arrive_expect_tx(kv_full + slot, C::TILE_BYTES);
        __syncwarp();
        pages.template load<C::KSUB>(smem + C::KV_OFF + slot * C::TILE_BYTES, v ? &tm_v : &tm_k, kv_full + slot,
                                     p, i, page);
      };
      // Table entries are read three tiles ahead of their loads' use, so no
      // load waits for them.
      int page[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) page[i] = pages.page(a, p, i);
      load(0, false, page[0]);
      if (g.split && g.n > 1) load(1, false, page[1]);
      for (int i = 0; ok && i < g.n; ++i) {
        load(i, true, page[0]);
        if (g.split) {
          if (ok && i + 2 < g.n) load(i + 2, false, page[2]);
        } else {
          if (ok && i + 1 < g.n) load(i + 1, false, page[1]);
        }
        page[0] = page[1];
        page[1] = page[2];
        page[2] = page[3];
        page[3] = pages.page(a, p, i + 4);
      }
    }
    // Do not leave the CTA while loads into its shared memory are in flight.
    for (int i = 0; i < 2; ++i)
      if (qb.uses[i] > 0) (void)mbar_wait(q_full + i, (qb.uses[i] - 1) & 1, nullptr, 0);
    for (int x = u - C::NSLOT < 0 ? 0 : u - C::NSLOT; x < u; ++x)
      (void)mbar_wait(kv_full + (x % C::NSLOT), (x / C::NSLOT) & 1, nullptr, 0);
  } else if (warp == C::kMmaWarp) {
    // ------------------------------------------------------------------ MMA
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(128, HD, true);
    const uint64_t q_desc = sw128_desc(smem_u32(smem + C::Q_OFF), 16, 1024);
    const uint64_t k_desc = sw128_desc(smem_u32(smem + C::KV_OFF), 16, 1024);
    const uint64_t v_desc = sw128_desc(smem_u32(smem + C::KV_OFF), C::SUB_BYTES, 1024);
    auto issue_s = [&](int st, int q, int slot) {
      const uint64_t kb = desc_add(k_desc, slot * C::TILE_BYTES), qd = desc_add(q_desc, q * C::TILE_BYTES);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint32_t off = (kk >> 2) * C::SUB_BYTES + (kk & 3) * 32;
        umma_ss(tmem + C::s_col(st), desc_add(qd, off), desc_add(kb, off), idesc_s, kk > 0 ? 1u : 0u);
      }
    };
    auto issue_o = [&](int st, int slot, bool acc) {
      const uint64_t vb = desc_add(v_desc, slot * C::TILE_BYTES);
#pragma unroll
      for (int kk = 0; kk < kPagedTile / 16; ++kk)
        umma_ts(tmem + C::o_col(st), tmem + C::s_col(st) + C::p_col(kk), desc_add(vb, kk * 2048), idesc_o,
                     (acc || kk > 0) ? 1u : 0u);
    };
    int pc0 = 0, pc1 = 0;
    QBuffers qb;
    RingPos<C::NSLOT> kv;
    bool ok = true;
    auto wait_kv = [&](const RingPos<C::NSLOT>& x) {
      return __all_sync(0xffffffffu, mbar_wait(kv_full + x.slot, x.phase, a.status, kDevTimeoutMma));
    };
    auto wait_p = [&](int st) {
      const int phase = st ? pc1++ : pc0++;
      return __all_sync(0xffffffffu, mbar_wait(p_full + st, phase & 1, a.status, kDevTimeoutMma));
    };
    while (ok && walk.next(a, p)) {
      const PgPiece g = pg_piece(a, p, tile_rows);
      const int n = uniform(g.n), n0 = uniform(g.n0), t0 = uniform(p.t0), len = uniform(p.r.len);
      if (n == 0) continue;
      auto clear_tail = [&](int i, int slot) {
        clear_v_tail<C::KSUB>(smem + C::KV_OFF + slot * C::TILE_BYTES, len - (t0 + i) * kPagedTile, a.page_shift,
                              lane);
      };
      const bool split = uniform(g.split);
      qb.next(split);
      for (int i = qb.first; ok && i <= qb.last; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait(q_full + i, qb.phase(i), a.status, kDevTimeoutMma));
        qb.take(i);
      }
      if (!ok) break;
      const int q0 = uniform(qb.first);
      if (split) {
        for (int i = 0; ok && i < min(2, n); ++i) {
          if (!(ok = wait_kv(kv))) break;
          tc_fence_after();
          if (elect_one()) {
            issue_s(i, q0, kv.slot);
            umma_commit(s_full + i);
            umma_commit(kv_empty + kv.slot);
            if (i + 1 == n) umma_commit(q_empty + q0);
          }
          kv.step();
        }
        for (int i = 0; ok && i < n; ++i) {
          const int st = i & 1, sv = kv.slot;
          const bool more = i + 2 < n;
          if (!(ok = wait_kv(kv))) break;
          clear_tail(i, sv);
          kv.step();
          if (more && !(ok = wait_kv(kv))) break;
          if (!(ok = wait_p(st))) break;
          tc_fence_after();
          if (elect_one()) {
            issue_o(st, sv, i >= 2);
            umma_commit(kv_empty + sv);
            if (more) {
              issue_s(st, q0, kv.slot);
              umma_commit(s_full + st);
              umma_commit(kv_empty + kv.slot);
              if (i + 3 == n) umma_commit(q_empty + q0);
            } else {
              umma_commit(o_full + st);
            }
          }
          if (more) kv.step();
        }
      } else {
        if (!(ok = wait_kv(kv))) break;
        tc_fence_after();
        if (elect_one()) {
          if (n0 > 0) {
            issue_s(0, 0, kv.slot);
            umma_commit(s_full + 0);
          }
          issue_s(1, 1, kv.slot);
          umma_commit(s_full + 1);
          umma_commit(kv_empty + kv.slot);
          if (n == 1) {
            umma_commit(q_empty + 0);
            umma_commit(q_empty + 1);
          }
        }
        kv.step();
        for (int i = 0; ok && i < n; ++i) {
          const int sv = kv.slot;
          const bool more = i + 1 < n;
          if (!(ok = wait_kv(kv))) break;
          clear_tail(i, sv);
          kv.step();
          const int sk = kv.slot;
          if (more && !(ok = wait_kv(kv))) break;
          if (i < n0) {
            if (!(ok = wait_p(0))) break;
            tc_fence_after();
            if (elect_one()) {
              issue_o(0, sv, i > 0);
              if (i + 1 < n0) {
                issue_s(0, 0, sk);
                umma_commit(s_full + 0);
              } else {
                umma_commit(o_full + 0);
              }
            }
          }
          if (!(ok = wait_p(1))) break;
          tc_fence_after();
          if (elect_one()) {
            issue_o(1, sv, i > 0);
            umma_commit(kv_empty + sv);
            if (more) {
              issue_s(1, 1, sk);
              umma_commit(s_full + 1);
              umma_commit(kv_empty + sk);
              if (i + 2 == n) {
                umma_commit(q_empty + 0);
                umma_commit(q_empty + 1);
              }
            } else {
              umma_commit(o_full + 1);
            }
          }
          if (more) kv.step();
        }
      }
    }
    // Every MMA issued must finish before TMEM is released.
    if (elect_one()) umma_commit(drain);
    (void)mbar_wait(drain, 0, nullptr, 0);
    __syncwarp();
  } else {
    // --------------------------------------------------- octic map + epilogue
    const int sub = warp & 3;        // TMEM lane quarter
    const int st = warp >> 3;        // stream
    const int half = (warp >> 2) & 1;  // its half of the key columns
    const int row = sub * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(sub * 32) << 16;
    const float scale = a.scale;
    const int ps = 1 << a.page_shift;
    const int per_tile = ps < kPagedTile ? kPagedTile >> a.page_shift : 1;
    int sc = 0, oc[2] = {0, 0};
    bool ok = true;
    auto sync_map = [] { asm volatile("bar.sync 1, %0;" ::"r"(C::kOcticWarps * 32) : "memory"); };
    // Every octic warp walks every piece and meets at the same barriers, also
    // after a wait ran out (ok false).
    while (walk.next(a, p)) {
      const PgPiece g = pg_piece(a, p, tile_rows);
      const int qt = g.split ? 0 : st;
      const int live_rows = g.rows[qt];
      const bool live = row < live_rows;
      const bool busy = sub * 32 < live_rows;  // some row of this warp is live
      const long long row0 = static_cast<long long>(p.u) * a.unit_rows + qt * tile_rows;
      const int node = static_cast<int>((row0 + (live ? row : 0)) / a.G);
      const int prefix = p.r.len - p.r.n;
      const int first = g.split ? st : 0, step = g.split ? 2 : 1;
      const int nmap = g.split || st ? g.n : g.n0;
      float dsum = 0.f;
      bool tail_check = true;  // warp-uniform: some row's weights so far < kTailRowSum
      // This lane's table entry of tile i, read a tile ahead of its use.
      auto entry = [&](int i) {
        const int key = (p.t0 + i) * kPagedTile + lane * ps;
        return busy && i < nmap && lane < per_tile && key < p.r.len
                   ? a.table[p.b * a.table_ld + (key >> a.page_shift)]
                   : 0;
      };
      int next_entry = entry(first);
      for (int i = first; i < nmap && ok; i += step) {
        const int key0 = (p.t0 + i) * kPagedTile;
        // Pages of the tile that the table does not name in the cache.
        const unsigned bad = __ballot_sync(0xffffffffu, next_entry < 0 || next_entry >= a.num_pages);
        next_entry = entry(i + step);
        ok = __all_sync(0xffffffffu, mbar_wait(s_full + st, sc & 1, a.status, kDevTimeoutSoftmax));
        ++sc;
        if (!ok) break;
        tc_fence_after();
        if (busy) {
          const bool need_mask = bad != 0 || key0 + kPagedTile > prefix;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            const int col = 64 * half + 32 * c;
            const uint32_t s_tm = tmem + C::s_col(st) + lane_off + col;
            uint32_t pk[16];
            float part = 0.f;
            if (!need_mask) {
              part = map_seen_tmem<false>(s_tm, pk, scale, 0u, live, tail_check);
            } else {
              unsigned seen = live ? paged_seen(a, p.r, node, key0 + col) : 0u;
              if (bad) {
                if (ps == 16) {
                  seen &= (bad >> (col >> 4)) & 1u ? 0xffff0000u : 0xffffffffu;
                  seen &= (bad >> ((col >> 4) + 1)) & 1u ? 0x0000ffffu : 0xffffffffu;
                } else if ((bad >> (col >> a.page_shift)) & 1u) {
                  seen = 0u;
                }
              }
              if (__any_sync(0xffffffffu, seen != 0u)) {
                part = map_seen_tmem<true>(s_tm, pk, scale, seen, live, tail_check);
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) pk[e] = 0u;
              }
            }
            // P of these 32 keys -> the first 16 of the 32 columns just read.
            tmem_st16(s_tm, pk);
            dsum += part;
          }
          tail_check = __any_sync(0xffffffffu, live && dsum < kTailRowSum);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + st);
      }
      // Row sums: the two column halves, then (split) the two streams.
      if (half == 1) red[st * 128 + row] = dsum;
      sync_map();
      if (half == 0) red[st * 128 + row] += dsum;
      sync_map();
      const float total = g.split ? red[row] + red[128 + row] : red[st * 128 + row];
      const bool has[2] = {g.split ? g.n > 0 : g.n0 > 0, g.split ? g.n > 1 : g.n > 0};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!has[i]) continue;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(o_full + i, oc[i] & 1, a.status, kDevTimeoutEpilogue));
        ++oc[i];
      }
      tc_fence_after();
      const bool whole = p.whole();
      const float denom = total + a.sink;
      const float inv = denom > 0.f ? 1.0f / denom : 0.f;
      const long long tok = p.r.tok0 + node;
      const long long orow = tok * a.Hkv * a.G + static_cast<long long>(p.h) * a.G + (row0 + (live ? row : 0)) % a.G;
      const int frow = qt * tile_rows + row;
      float* frag = static_cast<float*>(a.frag) +
                    (2LL * blockIdx.x + paged_frag_slot(p)) * a.frag_rows * (HD + 1);
      // 32-column chunks: in a pair, a warp's half of its own tile's; in a
      // split, one of the tile's chunks for each (stream, half).
      constexpr int CH = HD / 32;
      const int c0 = g.split ? st * 2 + half : half * (CH / 2);
      const int c1 = g.split ? min(c0 + 1, CH) : c0 + CH / 2;
      const bool o_here = ok && (g.split ? has[0] : has[st]);
      if (busy) {
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          const int col0 = 32 * c;
          uint32_t ov[32];
          if (o_here) {
            tmem_ld32(tmem + C::o_col(g.split ? 0 : st) + lane_off + col0, ov);
            tmem_ld_wait();
            if (g.split && has[1]) {
              uint32_t ow[32];
              tmem_ld32(tmem + C::o_col(1) + lane_off + col0, ow);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                ov[e] = __float_as_uint(__uint_as_float(ov[e]) + __uint_as_float(ow[e]));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = 0u;
          }
          if (whole) {
            // Four lanes trade 16-byte chunks, so that a store instruction
            // writes 64 contiguous bytes of each of 8 rows.
            constexpr int NCH = 4;
            const int gi = lane % NCH;
            uint32_t pk[32];
#pragma unroll
            for (int w = 0; w < 16; ++w)
              pk[w] = pack_bf16x2(__uint_as_float(ov[2 * w]) * inv, __uint_as_float(ov[2 * w + 1]) * inv);
            transpose_chunks<NCH>(pk, gi);
#pragma unroll
            for (int kr = 0; kr < NCH; ++kr) {
              const int src = (lane & ~(NCH - 1)) + kr;
              const long long r = __shfl_sync(0xffffffffu, orow, src);
              if (sub * 32 + src < live_rows) {
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + r * HD + col0 + 8 * gi;
                if (a.out_wide) {
                  *reinterpret_cast<uint4*>(dst) =
                      make_uint4(pk[4 * kr], pk[4 * kr + 1], pk[4 * kr + 2], pk[4 * kr + 3]);
                } else {  // `out` may be any part of a larger buffer
                  uint16_t* h = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    h[2 * e] = static_cast<uint16_t>(pk[4 * kr + e]);
                    h[2 * e + 1] = static_cast<uint16_t>(pk[4 * kr + e] >> 16);
                  }
                }
              }
            }
          } else {
            // Eight lanes: 128 contiguous bytes of each of 4 rows.
            constexpr int NCH = 8;
            const int gi = lane % NCH;
            transpose_chunks<NCH>(ov, gi);
#pragma unroll
            for (int kr = 0; kr < NCH; ++kr) {
              const int src = (lane & ~(NCH - 1)) + kr;
              if (sub * 32 + src < live_rows)
                *reinterpret_cast<uint4*>(frag + static_cast<long long>(frow - lane + src) * HD + col0 + 4 * gi) =
                    make_uint4(ov[4 * kr], ov[4 * kr + 1], ov[4 * kr + 2], ov[4 * kr + 3]);
            }
          }
        }
        if (half == 0 && live && (!g.split || st == 0)) {
          if (!whole)
            frag[static_cast<long long>(a.frag_rows) * HD + frow] = total;
          else if (a.dtot)
            static_cast<float*>(a.dtot)[orow] = denom;
        }
      }
      // O and the row sums are read: the next piece's first P may be announced.
      tc_fence_before();
      sync_map();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int HD>
cudaError_t launch_hd(const PagedArgs& a, int ctas, cudaStream_t stream, const char** detail) {
  using C = PgCfg<HD>;
  static PerDeviceOnce setup;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = setup.run(dev, [&] {
      return cudaFuncSetAttribute(afa_paged_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    });
  if (e != cudaSuccess) {
    *detail = "kernel set-up failed (max dynamic shared memory attribute)";
    return e;
  }
  CUtensorMap tq, tk, tv;
  if (!paged_tmaps(a, 128 / a.G, &tq, &tk, &tv)) {
    *detail = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  afa_paged_tc_kernel<HD><<<ctas, C::kThreads, C::SMEM_BYTES, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

}  // namespace

// TMA reads rows that start on 16 bytes at strides of 16 bytes; a stride of 0
// (a broadcast view) or of 2^31 elements or more is left to the CUDA cores.
bool paged_tc_supported(const PagedArgs& a, int dtype) {
  if (dtype != kBF16 || (a.D != 64 && a.D != 128) || a.G > 128) return false;
  for (const void* p : {a.q, a.k, a.v})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (long long s : {a.q_st, a.q_sh, a.k_sp, a.k_sh, a.k_sr, a.v_sp, a.v_sh, a.v_sr})
    if (s <= 0 || s % 8 != 0 || s >= (1LL << 31)) return false;
  return true;
}

int paged_tc_unit_rows(int G) { return 2 * (128 / G) * G; }

cudaError_t launch_paged_tc(const PagedArgs& a, int ctas, cudaStream_t stream, const char** detail) {
  return a.D == 128 ? launch_hd<128>(a, ctas, stream, detail) : launch_hd<64>(a, ctas, stream, detail);
}

}  // namespace afa
