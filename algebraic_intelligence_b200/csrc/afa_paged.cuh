// Work split of the attention over a paged cache.
//
// A work unit is up to unit_rows query rows (row r of a request: token r / G,
// query head r % G of the key head's group) of one request and key head against
// the keys those rows can see, in tiles of kPagedTile. The units, ordered by
// request, key head and rows, are laid end to end, one cost unit per key tile
// (two where a unit has two query tiles), and CTA c takes the c-th of equal
// shares of that line, the key tiles that begin in it: every CTA has about the
// same work whatever the lengths are, without knowing them on the host. A unit
// cut by the end of a share is computed in fragments. Octic
// weights need no running maximum, so fragments only add; they go to a
// workspace and paged_combine_kernel adds them in CTA order (no atomics: the
// same inputs give the same bits) and divides.
#pragma once

#include "afa_common.cuh"
#include "afa_paged.h"

namespace afa {

struct PagedReq {
  int tok0, n, len;  // first token, new tokens, keys (the new tokens' included)
};

__device__ __forceinline__ PagedReq paged_req(const PagedArgs& a, int b) {
  PagedReq r;
  const int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.lens[b];
  r.tok0 = min(max(c0, 0), a.T);
  r.n = min(max(c1, r.tok0), a.T) - r.tok0;
  const long long cap = static_cast<long long>(a.table_cols) << a.page_shift;
  r.len = len < 0 ? 0 : (len > cap ? static_cast<int>(cap) : len);
  return r;
}

__device__ __forceinline__ int paged_units(const PagedArgs& a, const PagedReq& r) {
  return (r.n * a.G + a.unit_rows - 1) / a.unit_rows;  // rows of a launch stay below 2^30
}

// Keys that some row of rows [.., row_end) of a request can see: all of them
// with a mask of drafted nodes, otherwise those up to the last row's token.
__device__ __forceinline__ int paged_visible(const PagedArgs& a, const PagedReq& r, int row_end) {
  if (a.anc) return r.len;
  const int last = (min(row_end, r.n * a.G) - 1) / a.G;
  const int vis = r.len - r.n + last + 1;
  return vis < 0 ? 0 : vis;
}

__device__ __forceinline__ int paged_tiles(const PagedArgs& a, const PagedReq& r, int u) {
  return (paged_visible(a, r, (u + 1) * a.unit_rows) + kPagedTile - 1) / kPagedTile;
}

// log2 of a key tile's cost. PAIRS: a unit with two query tiles takes 1.6 to 1.8
// times as long for a key tile as one with a single one, and counts twice (counted
// alike, the CTAs with pairs ended last: 16 trees of 17 to 34 nodes over 6000 keys
// took 104 us, 88 now, of 24 to 48 nodes 120, 113 now).
template <bool PAIRS>
__device__ __forceinline__ int paged_tile_shift(const PagedArgs& a, const PagedReq& r, int u) {
  return PAIRS && r.n * a.G - u * a.unit_rows > a.unit_rows / 2;
}

// Cost of a unit: its key tiles'; a unit that sees no key still writes its rows.
template <bool PAIRS>
__device__ __forceinline__ int paged_cost(const PagedArgs& a, const PagedReq& r, int u) {
  const int t = paged_tiles(a, r, u);
  return (t > 0 ? t : 1) << paged_tile_shift<PAIRS>(a, r, u);
}

// Cost of a request's units for one key head.
template <bool PAIRS>
__device__ __forceinline__ long long paged_req_cost(const PagedArgs& a, const PagedReq& r) {
  const int units = paged_units(a, r);
  if (units == 0) return 0;
  if (a.anc)  // all but the last are alike
    return static_cast<long long>(units - 1) * paged_cost<PAIRS>(a, r, 0) + paged_cost<PAIRS>(a, r, units - 1);
  long long c = 0;
  for (int u = 0; u < units; ++u) c += paged_cost<PAIRS>(a, r, u);
  return c;
}

struct PagedShare {
  int b;           // request the share starts in
  long long x;     // cost before it within that request
  long long left;  // the share's cost
  int ctas;        // CTAs that have a share
};

// This CTA's share. Called by all NT threads; `sm` is scratch of NT / 32 + 4
// 8-byte words. Every CTA adds up the requests' costs by itself: it costs less
// than a launch that would do it once.
template <int NT, bool PAIRS>
__device__ __forceinline__ PagedShare paged_share(const PagedArgs& a, long long* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int NW = NT / 32;
  // Cost of this thread's run of requests.
  const int per = (a.B + NT - 1) / NT;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, a.B), b1 = min(b0 + per, a.B);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += paged_req_cost<PAIRS>(a, paged_req(a, b)) * a.Hkv;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sm[warp] = inc;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const long long y = sm[w];
    before += w < warp ? y : 0;
    total += y;
  }
  const long long first = before + inc - mine;  // cost before this thread's requests
  PagedShare s;
  // PAIRS: no share is shorter than two, so that some key tile begins in each.
  const long long most = PAIRS ? max(total / a.min_share, min(total, 1LL)) : (total + a.min_share - 1) / a.min_share;
  s.ctas = most < gridDim.x ? static_cast<int>(most) : static_cast<int>(gridDim.x);
  const int c = blockIdx.x;
  if (c >= s.ctas) {
    s.b = 0;
    s.x = 0;
    s.left = 0;
    return s;
  }
  const long long lo = total * c / s.ctas, hi = total * (c + 1) / s.ctas;
  if (lo >= first && lo < first + mine) {
    long long x = lo - first;
    int b = b0;
    while (b < b1 - 1) {
      const long long cost = paged_req_cost<PAIRS>(a, paged_req(a, b)) * a.Hkv;
      if (x < cost) break;
      x -= cost;
      ++b;
    }
    sm[NW] = b;
    sm[NW + 1] = x;
  }
  __syncthreads();
  s.b = static_cast<int>(sm[NW]);
  s.x = sm[NW + 1];
  s.left = hi - lo;
  return s;
}

// A piece of a unit: key tiles [t0, t1) of `cost`; whole when it covers all.
struct PagedPiece {
  int b, h, u;
  int t0, t1, cost, tiles;
  PagedReq r;
  __device__ bool whole() const { return t0 == 0 && t1 == cost; }
};

template <bool PAIRS>
struct PagedWalk {
  int b, h, u, x, units;  // x: cost of unit u before the share
  long long left;
  PagedReq r;

  __device__ __forceinline__ void init(const PagedArgs& a, const PagedShare& s) {
    left = s.left;
    b = s.b;
    h = 0;
    u = 0;
    x = 0;
    units = 0;
    if (left <= 0) return;
    r = paged_req(a, b);
    units = paged_units(a, r);
    const long long cost = paged_req_cost<PAIRS>(a, r);
    h = static_cast<int>(s.x / cost);
    long long y = s.x - h * cost;
    if (a.anc) {
      const int c = paged_cost<PAIRS>(a, r, 0);
      u = static_cast<int>(min(y / c, static_cast<long long>(units - 1)));
      y -= static_cast<long long>(u) * c;
    } else {
      while (true) {
        const int c = paged_cost<PAIRS>(a, r, u);
        if (y < c) break;
        y -= c;
        ++u;
      }
    }
    x = static_cast<int>(y);
  }

  __device__ __forceinline__ bool next(const PagedArgs& a, PagedPiece& p) {
    while (left > 0) {
      if (u == units) {
        u = 0;
        if (++h == a.Hkv) {
          h = 0;
          do {
            if (++b >= a.B) return false;
            r = paged_req(a, b);
            units = paged_units(a, r);
          } while (units == 0);
        }
      }
      p.b = b;
      p.h = h;
      p.u = u;
      p.r = r;
      p.tiles = paged_tiles(a, r, u);
      p.cost = p.tiles > 0 ? p.tiles : 1;
      const int sh = paged_tile_shift<PAIRS>(a, r, u), total = p.cost << sh;
      const int end = left < total - x ? x + static_cast<int>(left) : total;
      p.t0 = (x + sh) >> sh;  // the tiles that begin in [x, end)
      p.t1 = (end + sh) >> sh;
      left -= end - x;
      x = 0;
      ++u;
      if (!PAIRS || p.t1 > p.t0) return true;
    }
    return false;
  }
};

// Fragments. CTA c has at most one piece that starts inside its unit (the
// first, fragment 0) and at most one that starts its unit and does not end it
// (the last, fragment 1). meta[4c]: 1 when fragment 0 ends its unit, 0 when it
// does not or there is none; meta[4c+1 ..]: request, key head and unit of
// fragment 1, request -1 when there is none.
__device__ __forceinline__ int paged_frag_slot(const PagedPiece& p) { return p.t0 > 0 ? 0 : 1; }

__device__ __forceinline__ void paged_meta_clear(int* meta) {
  int* m = meta + 4 * blockIdx.x;
  m[0] = 0;
  m[1] = -1;
}
__device__ __forceinline__ void paged_meta_piece(int* meta, const PagedPiece& p) {
  int* m = meta + 4 * blockIdx.x;
  if (p.t0 > 0) {
    m[0] = p.t1 == p.cost;
  } else if (p.t1 < p.cost) {
    m[1] = p.b;
    m[2] = p.h;
    m[3] = p.u;
  }
}

// Visibility of 32 keys from key position `key0` on for the row of new token
// `node` (0 .. n-1): bit i set when it sees key0 + i. Keys at or past `len`
// are never seen; keys before the new tokens always are.
__device__ __forceinline__ unsigned paged_seen(const PagedArgs& a, const PagedReq& r, int node, int key0) {
  const int left = r.len - key0;
  if (left <= 0) return 0u;
  unsigned m = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
  const int at = key0 - (r.len - r.n);  // new token of the first key; below 0 for keys before them
  if (a.anc) {
    if (at <= -32) return m;
    const unsigned* w = a.anc + static_cast<long long>(r.tok0 + node) * a.anc_ld;
    if (at < 0) return m & ((w[0] << -at) | ((1u << -at) - 1u));
    const int i = at >> 5, sh = at & 31;
    const unsigned lo = i < a.words ? w[i] : 0u, hi = i + 1 < a.words ? w[i + 1] : 0u;
    return m & __funnelshift_r(lo, hi, sh);
  }
  const int vis = node - at + 1;
  if (vis <= 0) return 0u;
  return vis >= 32 ? m : m & ((1u << vis) - 1u);
}

}  // namespace afa
