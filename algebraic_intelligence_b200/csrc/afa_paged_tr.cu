// AFA over a paged cache for few query rows per key head (single tokens, small
// trees), bf16, head_dim 64 or 128, on the tensor cores with the scores
// transposed. Math and work split: afa_paged.cu, afa_paged.cuh.
//
//   S^T = K Q^T     M = 128 keys, N = NT query rows
//   O^T += V^T P^T  M = head_dim,  N = NT, over the tile's 128 keys
//
// The query rows are the narrow side of both products, so the tensor core and
// the octic map work on NT (16 or 32) rows and not on the 128 that a row
// tile of the other kernel has: a thread owns one key and maps NT scores, and
// every warp has the same share whatever the number of rows. What is left is
// the cache's bytes. That leaves room for exactness: a weight enters the second
// product as two bf16 numbers, p = hi + lo within 2^-17 (NT more columns of
// P^T; the two halves of O^T meet in the epilogue), so that rows of few keys,
// where the roundings of single weights do not average out, are as exact as
// long ones.
//
//   warps 16,18 TMA: K (and Q) and V tiles through one ring, in the order they
//               are used; Q double buffered, so the next unit's loads never wait.
//               With pages of 16 tokens a tile of K and V is 32 copies of 65
//               cycles each to issue, more than one warp has time for.
//   warp 17     every tcgen05.mma, and the clearing of V rows behind a request's
//               last token (see afa_paged_tc.cu).
//   warps 0-15  two groups of eight warps take tiles in turn: scores from TMEM,
//               P^T to shared memory as bf16 ([key][row: hi, then lo], 128-byte
//               swizzle: the layout V has), row sums in registers. One group maps
//               while the tensor core works on the other's tile; within a group
//               four warps cover the keys of each half of the rows. (With four
//               warps a group, 64 rows took 2.3 us a tile: one warp's chain.)
//               A piece's output is written after the next piece's scores were
//               mapped (O^T and the row sums are double buffered), so that no
//               warp waits for the last P.V: in batches of short requests that
//               wait and the barriers around it were most of the time.
// TMEM columns: S^T of group g at [NT g, NT g + NT), O^T of every other piece at
// [128, 128 + 2 NT) and [128 + 2 NT, 128 + 4 NT).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "afa_common.cuh"
#include "afa_internal.h"
#include "afa_paged.cuh"
#include "afa_paged_tma.cuh"

namespace afa {
namespace {

template <int HD, int NT>
struct TrCfg {
  static constexpr int kMapWarps = 16;
  static constexpr int kTmaWarp = 16;
  static constexpr int kMmaWarp = 17;
  static constexpr int kTmaVWarp = 18;
  static constexpr int kThreads = 19 * 32;
  static constexpr int NH = NT / 2;  // rows of a warp
  static constexpr int KSUB = HD / 64;
  static constexpr int SUB_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = KSUB * SUB_BYTES;
  static constexpr int QSUB_BYTES = NT * 128;
  static constexpr int Q_BYTES = KSUB * QSUB_BYTES;
  static constexpr int P_BYTES = SUB_BYTES;  // 128 keys x 64 columns: hi and lo of up to 32 rows
  static constexpr int Q_OFF = 0;
  static constexpr int P_OFF = 2 * Q_BYTES;
  static constexpr int KV_OFF = P_OFF + 2 * P_BYTES;
  static constexpr int NSLOT = HD == 128 ? 5 : 8;
  static constexpr int BAR_OFF = KV_OFF + NSLOT * TILE_BYTES;
  static constexpr int NBAR = 4 + 2 * NSLOT + 2 + 2 + 2 + 2 + 2 + 1;
  static constexpr int TMEM_OFF = BAR_OFF + NBAR * 8;
  static constexpr int RED_OFF = TMEM_OFF + 16;  // fp32 row sums [piece parity][group, lane quarter][row]
  static constexpr int SHARE_OFF = RED_OFF;      // paged_share's scratch: before any sum is written
  static_assert((kThreads / 32 + 4) * 8 <= 2 * 8 * NT * 4, "scratch fits in the sums");
  static constexpr int SMEM_BYTES = RED_OFF + 2 * 8 * NT * 4 + 1024;
  static_assert(Q_BYTES % 1024 == 0 && SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
  // The ring holds tiles in the order the tensor core uses them: K0 K1 V0 K2 V1
  // K3 V2 ...: tile t's K is at position 2 t - 1 (0 for t = 0), its V at 2 t + 2.
  struct KPos : RingPos<NSLOT> {
    __device__ __forceinline__ void next(int t) { this->step(t == 0 ? 1 : 2); }  // from tile t to t + 1
  };
  struct VPos : RingPos<NSLOT> {
    __device__ __forceinline__ VPos() { this->slot = 2; }
    __device__ __forceinline__ void next() { this->step(2); }
  };
  static constexpr uint32_t TMEM_COLS = 256;
  __device__ static constexpr uint32_t o_col(int parity) { return 128u + static_cast<uint32_t>(parity) * 2 * NT; }
};

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// N columns (1 or 2) of this thread's lane.
template <int N>
__device__ __forceinline__ void tmem_ld_few(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 1)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r[0]) : "r"(taddr));
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(taddr));
}

// Clears the rows of a query tile behind the unit's: TMA has put the next
// tokens' queries there, or nothing (unit_rows may be less than NT). Their
// outputs go nowhere, but their scores would have a say in which form a chunk of
// weights is computed in (see kTrTail), so that a row's last bits depended on
// other requests and on what the shared memory held before. The warp that issues
// the products calls it after the tile has arrived.
template <int KSUB, int NT>
__device__ __forceinline__ void clear_q_rows(uint8_t* tile, int rows, int lane) {
  if (rows >= NT) return;
  for (int x = rows * 8 + lane; x < NT * 8; x += 32)
#pragma unroll
    for (int h = 0; h < KSUB; ++h)
      st_shared_v4(smem_u32(tile + h * NT * 128 + x * 16), make_uint4(0u, 0u, 0u, 0u));
  fence_proxy_async_shared();
  __syncwarp();
}

// Sums of 8 values over the warp's lanes: lane l returns value l / 4's.
__device__ __forceinline__ float reduce8(const float* v, int lane) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
  for (int m = 4; m >= 1; m >>= 1) {
    const bool hi = (lane & (4 * m)) != 0;
#pragma unroll
    for (int i = 0; i < m; ++i) {
      const float send = hi ? x[i] : x[i + m];
      const float keep = hi ? x[i + m] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, 4 * m);
    }
  }
  x[0] += __shfl_xor_sync(0xffffffffu, x[0], 2);
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 1);
}

// Below this score a chunk of weights is computed in the form that is exact in
// the negative tail; above it octic_fast2 is within 2.5e-6 s^2 <= 4e-5 of a
// weight, and one special-function operation cheaper.
constexpr float kTrTail = -4.0f;
constexpr uint64_t kDrainNs = 1000000;  // 1 ms

// Weights of 8 rows for one key, as bf16 pairs hi and lo with p = hi + lo, and
// their sums. Bit e of `seen`: row e sees the key.
template <bool MASK>
__device__ __forceinline__ void map8(const uint32_t* sv, float scale, unsigned seen, float* sum, uint32_t (&hi)[4],
                                     uint32_t (&lo)[4]) {
  const float2 sc = make_float2(scale, scale);
  float2 s[4], w[4];
  float least = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s[e] = __fmul2_rn(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc);
    // Of the scores that count: keys behind the request's last token may be anything.
    const float x = !MASK || (seen & (1u << (2 * e))) ? s[e].x : 0.f;
    const float y = !MASK || (seen & (2u << (2 * e))) ? s[e].y : 0.f;
    least = fminf(least, fminf(x, y));
  }
  if (__any_sync(0xffffffffu, least < kTrTail)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = octic_exact2(s[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = octic_fast2(s[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (MASK) {
      w[e].x = seen & (1u << (2 * e)) ? w[e].x : 0.f;
      w[e].y = seen & (2u << (2 * e)) ? w[e].y : 0.f;
    }
    sum[2 * e] += w[e].x;
    sum[2 * e + 1] += w[e].y;
    const uint32_t h = pack_bf16x2(w[e].x, w[e].y);
    hi[e] = h;
    lo[e] = pack_bf16x2(w[e].x - __uint_as_float(h << 16), w[e].y - __uint_as_float(h & 0xFFFF0000u));
  }
}

template <int HD, int NT>
__global__ void __launch_bounds__(608, 1)
    afa_paged_tr_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedArgs a) {
  using C = TrCfg<HD, NT>;
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
  uint64_t* o_empty = o_full + 2;   // a piece's outputs are written: its O^T and row sums may be overwritten
  uint64_t* r_full = o_empty + 2;   // every warp's row sums are written
  uint64_t* drain = r_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TMEM_OFF);
  float* red = reinterpret_cast<float*>(smem + C::RED_OFF);
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 8);  // one elected arrive per warp of the group
      mbar_init(o_full + i, 1);
      mbar_init(o_empty + i, C::kMapWarps);
      mbar_init(r_full + i, C::kMapWarps);
    }
    for (int s = 0; s < C::NSLOT; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_empty + s, 1);
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
  PagedWalk<false> walk;
  walk.init(a, paged_share<C::kThreads, false>(a, reinterpret_cast<long long*>(smem + C::SHARE_OFF)));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  PagedPiece p;

  if (warp == C::kTmaWarp || warp == C::kTmaVWarp) {
    // ------------------------------------------------------------------ TMA
    const bool is_v = warp == C::kTmaVWarp;
    KvPages pages(a);
    RingPos<C::NSLOT> pos;  // as KPos and VPos
    if (is_v) pos.slot = 2;
    int tile = 0, qn = 0;  // tile counts through all pieces of the CTA
    bool ok = true;
    while (ok && walk.next(a, p)) {
      if (!is_v && lane == 0) paged_meta_piece(a.meta, p);
      const int n = p.tiles > 0 ? p.t1 - p.t0 : 0;
      if (n == 0) continue;
      int page[4];  // table entries are read ahead of their use
#pragma unroll
      for (int i = 0; i < 4; ++i) page[i] = pages.page(a, p, i);
      if (!is_v) {
        const int qb = qn & 1;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(q_empty + qb, ((qn >> 1) & 1) ^ 1, a.status,
                                                     kDevTimeoutProducer))))
          break;
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full + qb, C::KSUB * a.unit_rows * 128);
          for (int h = 0; h < C::KSUB; ++h)
            tma_load_4d(smem + C::Q_OFF + qb * C::Q_BYTES + h * C::QSUB_BYTES, &tm_q, q_full + qb, 64 * h, 0, p.h,
                        p.r.tok0 + p.u * (a.unit_rows / a.G));
        }
        ++qn;
      }
      for (int i = 0; i < n; ++i, ++tile) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(kv_empty + pos.slot, pos.phase ^ 1, a.status,
                                                     kDevTimeoutProducer))))
          break;
        if (lane == 0) mbar_arrive_expect_tx(kv_full + pos.slot, C::TILE_BYTES);
        __syncwarp();
        pages.template load<C::KSUB>(smem + C::KV_OFF + pos.slot * C::TILE_BYTES, is_v ? &tm_v : &tm_k,
                                     kv_full + pos.slot, p, i, page[0]);
        pos.step(!is_v && tile == 0 ? 1 : 2);
        page[0] = page[1];
        page[1] = page[2];
        page[2] = page[3];
        page[3] = pages.page(a, p, i + 4);
      }
    }
    // Do not leave the CTA while loads into its shared memory are in flight:
    // those of the ring's last round, whose slots nothing took after them. (The
    // short budget is for a launch that failed, where that may not hold.)
    for (int x = qn - 2 < 0 ? 0 : qn - 2; x < qn; ++x)
      (void)mbar_wait(q_full + (x & 1), (x >> 1) & 1, nullptr, 0, kDrainNs);
    for (int x = tile - 1; x >= 0; --x) {
      const int at = is_v ? 2 * x + 2 : x > 0 ? 2 * x - 1 : 0;
      if (at <= 2 * tile - C::NSLOT) break;
      (void)mbar_wait(kv_full + at % C::NSLOT, (at / C::NSLOT) & 1, nullptr, 0, kDrainNs);
    }
  } else if (warp == C::kMmaWarp) {
    // ------------------------------------------------------------------ MMA
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, NT, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(HD, 2 * NT, true) | (1u << 15);  // A = V^T: its M (head_dim) is contiguous
    const uint64_t q_desc = sw128_desc(smem_u32(smem + C::Q_OFF), 16, 1024);
    const uint64_t k_desc = sw128_desc(smem_u32(smem + C::KV_OFF), 16, 1024);
    const uint64_t v_desc = sw128_desc(smem_u32(smem + C::KV_OFF), C::SUB_BYTES, 1024);
    const uint64_t p_desc = sw128_desc(smem_u32(smem + C::P_OFF), C::SUB_BYTES, 1024);
    auto issue_s = [&](int g, int qb, int slot) {
      const uint64_t kb = desc_add(k_desc, slot * C::TILE_BYTES), qd = desc_add(q_desc, qb * C::Q_BYTES);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        umma_ss(tmem + g * NT, desc_add(kb, (kk >> 2) * C::SUB_BYTES + (kk & 3) * 32),
                     desc_add(qd, (kk >> 2) * C::QSUB_BYTES + (kk & 3) * 32), idesc_s, kk > 0 ? 1u : 0u);
    };
    auto issue_o = [&](int g, int par, int slot, bool acc) {
      const uint64_t vb = desc_add(v_desc, slot * C::TILE_BYTES), pd = desc_add(p_desc, g * C::P_BYTES);
#pragma unroll
      for (int kk = 0; kk < kPagedTile / 16; ++kk)
        umma_ss(tmem + C::o_col(par), desc_add(vb, kk * 2048), desc_add(pd, kk * 2048), idesc_o,
                (acc || kk > 0) ? 1u : 0u);
    };
    // The tiles of all pieces are one stream: the scores run two tiles ahead of
    // the outputs, also from one piece into the next, with a walk of their own.
    PagedWalk<false> swalk = walk;
    typename C::KPos kpos;
    typename C::VPos vpos;
    bool ok = true, s_more = true;
    int s_tile = 0, s_left = 0, s_qn = -1;
    // Waits for the next tile's K (and its piece's Q): false when there is none.
    auto wait_scores = [&]() {
      while (s_left == 0) {
        PagedPiece sp;
        if (!s_more || !(s_more = swalk.next(a, sp))) return false;
        s_left = uniform(sp.tiles > 0 ? sp.t1 - sp.t0 : 0);
        if (s_left == 0) continue;
        ++s_qn;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(q_full + (s_qn & 1), (s_qn >> 1) & 1, a.status,
                                                     kDevTimeoutMma))))
          return false;
        clear_q_rows<C::KSUB, NT>(smem + C::Q_OFF + (s_qn & 1) * C::Q_BYTES,
                                  uniform(min(sp.r.n * a.G - sp.u * a.unit_rows, a.unit_rows)), lane);
      }
      return ok = __all_sync(0xffffffffu, mbar_wait(kv_full + kpos.slot, kpos.phase, a.status, kDevTimeoutMma));
    };
    auto issue_scores = [&]() {  // one lane
      issue_s(s_tile & 1, s_qn & 1, kpos.slot);
      umma_commit(s_full + (s_tile & 1));
      umma_commit(kv_empty + kpos.slot);
      if (s_left == 1) umma_commit(q_empty + (s_qn & 1));
    };
    auto scores_issued = [&]() {
      kpos.next(s_tile);
      ++s_tile;
      --s_left;
    };
    int piece = -1, tile = 0;
    for (int i = 0; i < 2 && wait_scores(); ++i) {
      tc_fence_after();
      if (elect_one()) issue_scores();
      scores_issued();
    }
    while (ok && walk.next(a, p)) {
      const int t0 = uniform(p.t0), n = uniform(p.tiles > 0 ? p.t1 : p.t0) - t0, len = uniform(p.r.len);
      ++piece;
      const int par = piece & 1;
      for (int i = 0; ok && i < n; ++i, ++tile) {
        const int g = tile & 1, slot = vpos.slot;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(kv_full + slot, vpos.phase, a.status, kDevTimeoutMma)))) break;
        clear_v_tail<C::KSUB>(smem + C::KV_OFF + slot * C::TILE_BYTES, len - (t0 + i) * kPagedTile, a.page_shift, lane);
        const bool scores = wait_scores();
        if (!ok) break;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(p_full + g, (tile >> 1) & 1, a.status, kDevTimeoutMma)))) break;
        if (i == 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(o_empty + par, ((piece >> 1) & 1) ^ 1, a.status,
                                                                kDevTimeoutMma))))
          break;
        tc_fence_after();
        if (elect_one()) {
          issue_o(g, par, slot, i > 0);
          umma_commit(kv_empty + slot);
          if (i + 1 == n) umma_commit(o_full + par);
          if (scores) issue_scores();
        }
        if (scores) scores_issued();
        vpos.next();
      }
    }
    // Every MMA issued must finish before TMEM is released.
    if (elect_one()) umma_commit(drain);
    (void)mbar_wait(drain, 0, nullptr, 0);
    __syncwarp();
  } else {
    // --------------------------------------------------- octic map + epilogue
    const int g = warp >> 3;           // group: every other tile of the CTA
    const int half = (warp >> 2) & 1;  // its half of the rows
    const int sub = warp & 3;          // TMEM lane quarter
    constexpr int NH = C::NH;
    const uint32_t lane_off = static_cast<uint32_t>(sub * 32) << 16;
    const int krow = sub * 32 + lane;  // this thread's key of a tile
    const uint32_t p_row = smem_u32(smem + C::P_OFF + g * C::P_BYTES + krow * 128);
    // Columns [r, r + 8) of this thread's key: 16-byte chunk j of key row k lies
    // at (j ^ (k % 8)) * 16 of the row's 128 bytes.
    auto put = [&](int r, const uint32_t (&v)[4]) {
      st_shared_v4(p_row + (((r >> 3) ^ (krow & 7)) << 4), make_uint4(v[0], v[1], v[2], v[3]));
    };
    int scnt = 0, piece = -1, tiles = 0;  // tiles: of the pieces before
    int oc[2] = {0, 0};  // pieces with an O^T, by parity
    bool ok = true;
    // Outputs of a piece: O / (sum + sink), or the fragment.
    int d_rows = 0, d_tok = 0, d_h = 0, d_kind = 0;  // of the piece to write: kind bit 0 whole, 1 later fragment, 2 has O
    auto write_piece = [&](int par, int use) {
      const bool whole = d_kind & 1, has_o = d_kind & 4;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(r_full + par, use & 1, a.status, kDevTimeoutEpilogue));
      if (has_o) {
        const int phase = par ? oc[1]++ : oc[0]++;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(o_full + par, phase & 1, a.status, kDevTimeoutEpilogue));
      }
      tc_fence_after();
      const bool o_here = ok && has_o;
      // Head channel of this thread's TMEM lane: with 64 channels (M = 64) the
      // accumulator uses 16 lanes of every quarter.
      const bool chan = HD == 128 || lane < 16;
      const int d = HD == 128 ? krow : sub * 16 + (lane & 15);
      const float* r = red + par * 8 * NT;
      float* frag = static_cast<float*>(a.frag) + (2LL * blockIdx.x + ((d_kind >> 1) & 1)) * a.frag_rows * (HD + 1);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out);
      // The four sets of warps that cover the lanes share the rows, a few at a
      // time so that all have some of a single token's.
      constexpr int CH = NT / 16;
#pragma unroll 1
      for (int c = CH * (warp >> 2); c < d_rows; c += 4 * CH) {
        float total = 0.f;  // of row c + lane % CH; groups and quarters in a fixed order
#pragma unroll
        for (int w = 0; w < 8; ++w) total += r[w * NT + c + lane % CH];
        const float denom = total + a.sink;
        const float scale_o = whole ? (denom > 0.f ? __frcp_rn(denom) : 0.f) : 1.f;
        uint32_t ov[CH], ol[CH];
        __syncwarp();
        if (o_here) {
          tmem_ld_few<CH>(tmem + C::o_col(par) + lane_off + c, ov);
          tmem_ld_few<CH>(tmem + C::o_col(par) + NT + lane_off + c, ol);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < CH; ++e) ov[e] = ol[e] = 0u;
        }
        const int row = c + lane % CH, tok = row / a.G;
        const long long my_row = static_cast<long long>(d_tok + tok) * a.Hkv * a.G +
                                 static_cast<long long>(d_h) * a.G + (row - tok * a.G);
        if (sub == 0 && lane < CH && row < d_rows) {
          if (!whole)
            frag[static_cast<long long>(a.frag_rows) * HD + row] = total;
          else if (a.dtot)
            static_cast<float*>(a.dtot)[my_row] = denom;
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const float y = (__uint_as_float(ov[e]) + __uint_as_float(ol[e])) *
                          (CH > 1 ? __shfl_sync(0xffffffffu, scale_o, e) : scale_o);
          const long long orow = CH > 1 ? __shfl_sync(0xffffffffu, my_row, e) : my_row;
          if (chan && c + e < d_rows) {
            if (whole)
              out[orow * HD + d] = __float2bfloat16_rn(y);
            else
              frag[static_cast<long long>(c + e) * HD + d] = y;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty + par);
    };
    // Every warp walks every piece, also after a wait ran out (ok false).
    // Table entry of this thread's key of tile i, read a tile (or a piece) ahead
    // of its use; -1 where there is no key.
    auto entry = [&](int i) {
      const int key = (p.t0 + i) * kPagedTile + krow;
      return p.t0 + i < p.t1 && key < p.r.len ? a.table[p.b * a.table_ld + (key >> a.page_shift)] : -1;
    };
    bool have = walk.next(a, p);
    int next_entry = have ? entry(g) : -1;  // of this group's first tile of the piece
    while (have) {
      ++piece;
      const int n = p.tiles > 0 ? p.t1 - p.t0 : 0;
      const int row0 = p.u * a.unit_rows, rows = min(p.r.n * a.G - row0, a.unit_rows);
      const int tok_u = p.u * (a.unit_rows / a.G);  // first new token of the unit
      const int prefix = p.r.len - p.r.n;
      const bool mine = half * NH < rows;  // some row of this half exists
      float sum[NH];
#pragma unroll
      for (int i = 0; i < NH; ++i) sum[i] = 0.f;
      for (int i = (g ^ tiles) & 1; i < n && ok; i += 2) {
        const int key = (p.t0 + i) * kPagedTile + krow;
        const bool in = next_entry >= 0 && next_entry < a.num_pages;
        next_entry = entry(i + 2);
        // Rows that see this thread's key.
        unsigned seen = in ? ~0u : 0u;
        const int at = key - prefix;
        if (in && at >= 0) {
          if (a.anc) {
            seen = 0;
            const int w = at >> 5;
            if (w < a.words)
              for (int j = 0; j * a.G < rows; ++j) {
                const unsigned word = a.anc[static_cast<long long>(p.r.tok0 + tok_u + j) * a.anc_ld + w];
                if ((word >> (at & 31)) & 1u) seen |= ((1u << (a.G - 1)) * 2u - 1u) << (j * a.G);
              }
          } else {
            const long long first = static_cast<long long>(at) * a.G - row0;  // first row of token `at`
            seen = first <= 0 ? ~0u : first >= 32 ? 0u : ~0u << first;
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(s_full + g, scnt & 1, a.status, kDevTimeoutSoftmax));
        ++scnt;
        if (!ok) break;
        tc_fence_after();
        __syncwarp();
        if (mine) {
          const uint32_t s_tm = tmem + g * NT + lane_off + half * NH;
          uint32_t sv[NH];
          if constexpr (NH == 16)
            tmem_ld16(s_tm, sv);
          else
            tmem_ld8(s_tm, sv);
          tmem_ld_wait();
          const unsigned word = seen >> (half * NH);
          const bool all_seen = __all_sync(0xffffffffu, seen == ~0u);
#pragma unroll
          for (int c = 0; c < NH; c += 8) {
            uint32_t hi[4], lo[4];
            if (all_seen)
              map8<false>(sv + c, a.scale, 0u, sum + c, hi, lo);
            else
              map8<true>(sv + c, a.scale, word >> c, sum + c, hi, lo);
            put(half * NH + c, hi);
            put(NT + half * NH + c, lo);
          }
        }
        fence_proxy_async_shared();  // P is read by the tensor core
        tc_fence_before();           // and the scores may be overwritten
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + g);
      }
      // Row sums over the lanes, into this parity's buffer once the outputs of
      // the piece before the last are written.
      const int par = piece & 1, use = piece >> 1;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(o_empty + par, (use & 1) ^ 1, a.status, kDevTimeoutEpilogue));
#pragma unroll
      for (int c = 0; c < NH; c += 8) {
        const float s = reduce8(sum + c, lane);
        if ((lane & 3) == 0) red[par * 8 * NT + (g * 4 + sub) * NT + half * NH + c + (lane >> 2)] = s;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(r_full + par);
      const int tok = p.r.tok0 + tok_u, head = p.h;
      const int kind = (p.whole() ? 1 : 0) | paged_frag_slot(p) << 1 | (n > 0 ? 4 : 0);
      // The next piece's first table entry is under way while the outputs are
      // written.
      tiles += n;
      have = walk.next(a, p);
      next_entry = have ? entry((g ^ tiles) & 1) : -1;
      if (piece > 0) write_piece(par ^ 1, (piece - 1) >> 1);
      d_rows = rows;
      d_tok = tok;
      d_h = head;
      d_kind = kind;
    }
    if (piece >= 0) write_piece(piece & 1, piece >> 1);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int HD, int NT>
cudaError_t launch_nt(const PagedArgs& a, int ctas, cudaStream_t stream, const char** detail) {
  using C = TrCfg<HD, NT>;
  static PerDeviceOnce setup;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = setup.run(dev, [&] {
      return cudaFuncSetAttribute(afa_paged_tr_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  C::SMEM_BYTES);
    });
  if (e != cudaSuccess) {
    *detail = "kernel set-up failed (max dynamic shared memory attribute)";
    return e;
  }
  CUtensorMap tq, tk, tv;
  if (!paged_tmaps(a, a.unit_rows / a.G, &tq, &tk, &tv)) {
    *detail = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  afa_paged_tr_kernel<HD, NT><<<ctas, C::kThreads, C::SMEM_BYTES, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_hd(const PagedArgs& a, int nt, int ctas, cudaStream_t stream, const char** detail) {
  return nt == 16 ? launch_nt<HD, 16>(a, ctas, stream, detail) : launch_nt<HD, 32>(a, ctas, stream, detail);
}

}  // namespace

// Measured against the row-tile kernel over 64 x 8192 keys of 8 heads: 32 rows
// 264 us (row tiles 320), 64 rows, with a variant that had twice the columns,
// 348 (322); over 256 x 200 keys 64 rows 203 (117).
int paged_tr_rows(int B, int T, int G) {
  const long long rows = (static_cast<long long>(T) + B - 1) / B * G;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 0;
}

cudaError_t launch_paged_tr(const PagedArgs& a, int nt, int ctas, cudaStream_t stream, const char** detail) {
  return a.D == 128 ? launch_hd<128>(a, nt, ctas, stream, detail) : launch_hd<64>(a, nt, ctas, stream, detail);
}

}  // namespace afa
