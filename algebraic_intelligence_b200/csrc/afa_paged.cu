// AFA over a paged key/value cache: the new tokens of a batch of requests (one
// token each, chunks of prompts, or trees of drafted tokens) against the
// requests' cached keys. The math is pallas_afa_forward's
// (src/kernels/pallas_afa.py:104-151) with the keys read through a block table:
//
//   s = q.k / sqrt(D), p = rho(s)^8 where the row sees the key, else 0
//   out = sum p v / (sum p + sink), d_total = sum p + sink
//
// Row (token t, query head h) of a request of n new tokens and len keys sees
// key j < len when j < len - n (the tokens before), or when new token
// j - (len - n) is t or before it (causal), or its bit in t's ancestor words is
// set (a tree of drafted tokens), and when its block table entry names a page
// of the cache. The query heads h = kv_head * G + g of a group
// share the cache rows of their key head.
//
// This file: the CUDA-core kernel for float32 / float64 and for bf16 head
// dimensions the tensor-core kernel (afa_paged_tc.cu) does not take, the kernel
// that adds fragments, and the C entry point. The work split is in
// afa_paged.cuh.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

#include "afa_b200.h"
#include "afa_common.cuh"
#include "afa_internal.h"
#include "afa_paged.cuh"

namespace afa {
namespace {

constexpr int kSimtThreads = 256;

// rho(s)^8 with rho(|s|) = |s| + sqrt(1 + s^2) and rho(-s) = 1 / rho(s): sums of
// like signs only, every operation correctly rounded. In half steps of the type
// (relative): 1/2 of the fma's through the root, 1 the root's, 1 the sum's, and
// for s < 0 1 the reciprocal's, so rho is within 2.5 or 3.5 and a weight, with
// three squarings, within 8 times that plus 7: 27 or 35, 1.6e-6 or 2.1e-6 in
// float32 (25 seen over 4M scores; octic_ref's reciprocal root alone is off by
// up to 4).
__device__ __forceinline__ float recip(float x) { return __frcp_rn(x); }
__device__ __forceinline__ double recip(double x) { return __drcp_rn(x); }
template <typename A>
__device__ __forceinline__ A octic_even(A s) {
  const A t = s < A(0) ? -s : s;
  A rho = t + sqrt(fma(s, s, A(1)));
  if (s < A(0)) rho = recip(rho);
  const A k2 = rho * rho, k4 = k2 * k2;
  return k4 * k4;
}

// 16 bytes of accumulators.
template <typename A>
struct alignas(16) Quad {
  static constexpr int N = 16 / sizeof(A);
  A x[N];
};

// ROWS query rows x BN keys per step, 256 threads. Scores: a warp is LY rows x
// LX keys, a thread owns TR x TC of them; outputs: a thread owns RP rows of OC
// groups of 16 bytes of channels (with KS = 2 one of two halves of the keys as
// well), a warp 4 rows x 8 groups. Both ways a quarter warp's 16-byte reads of
// shared memory fall on different banks or are one broadcast, and there are few
// of them for each FMA (6 to 32, 8 to 64 with 32 rows): the FMAs bound 32 rows,
// the cache's bytes 8. Shared rows are DMAX channels padded by 16 bytes; several
// CTAs per SM cover the loads' latency. Outputs add up over BN keys in registers
// of their own before they join the row's, a thread's row sum takes TC weights a
// step: few enough additions that they do not show. Float32 outputs and d_total
// were 0.2e-6 to 2.6e-6 off (relative to sum p |v| and to d_total) from 64 to
// 300000 keys of 64 and 128 channels, also 32768 of them in one CTA, without a
// trend in the length (up to 1.3e-5 with 256 channels: a score's rounding counts
// eightfold in its weight).
template <typename A, int ROWS, int BN, int DMAX>
struct SimtCfg {
  static constexpr int V = Quad<A>::N;
  static constexpr int LX = ROWS == 8 && BN == 64 ? 8 : 4, LY = 32 / LX;
  static constexpr int TR = ROWS / LY, TC = BN / (8 * LX);
  static constexpr int CG = DMAX / V < 64 ? DMAX / V : 64, OC = DMAX / V / CG;  // channel groups across threads
  static constexpr int RG = kSimtThreads / CG;
  static constexpr int KS = RG > ROWS ? RG / ROWS : 1, RP = RG > ROWS ? 1 : ROWS / RG;
  static constexpr int LD = DMAX + V, PLD = BN + V;
  static constexpr size_t kSmem = sizeof(A) * (static_cast<size_t>(ROWS + 2 * BN) * LD + static_cast<size_t>(ROWS) * PLD);
  static_assert(TC >= 1 && TR >= 1 && KS <= 2 && CG % 8 == 0, "thread mapping");
  static_assert(KS == 1 || static_cast<size_t>(ROWS) * DMAX <= static_cast<size_t>(BN) * LD, "halves meet in the K tile");
};

template <typename T, typename A, int ROWS, int BN, int DMAX>
__global__ void __launch_bounds__(kSimtThreads) afa_paged_simt_kernel(const __grid_constant__ PagedArgs a) {
  using C = SimtCfg<A, ROWS, BN, DMAX>;
  constexpr int V = C::V, LX = C::LX, LY = C::LY, TR = C::TR, TC = C::TC, OC = C::OC, RP = C::RP, LD = C::LD,
                PLD = C::PLD;
  using Q4 = Quad<A>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ long long share_sm[kSimtThreads / 32 + 4];
  __shared__ long long k_row[BN], v_row[BN];  // offsets of the step's cache rows; below 0: none
  __shared__ A sums[8][ROWS];                 // row sums, by warp
  A* Qs = reinterpret_cast<A*>(smem_raw);
  A* Ks = Qs + ROWS * LD;
  A* Vs = Ks + BN * LD;
  A* Ps = Vs + BN * LD;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.D;
  const int kx = warp * LX + lane % LX, ry = lane / LX;  // scores: keys kx + 8 LX j, rows ry + LY i
  constexpr int WC = C::CG / 8;                          // warps along the channels
  const int cg = lane % 8 + 8 * (warp % WC), rg = lane / 8 + 4 * (warp / WC);
  const int ks = C::KS == 2 ? rg / ROWS : 0, ro = C::KS == 2 ? rg % ROWS : rg;  // outputs: rows ro + RG i
  const int dv = (D + V - 1) / V;  // 16-byte channel groups; the last is padded with zeros
  const T* q = static_cast<const T*>(a.q);
  T* out = static_cast<T*>(a.out);
  A* dtot = static_cast<A*>(a.dtot);
  const A scale = sizeof(A) == 8 ? static_cast<A>(a.scale_d) : static_cast<A>(a.scale);
  const A sink = sizeof(A) == 8 ? static_cast<A>(a.sink_d) : static_cast<A>(a.sink);
  A* frag = static_cast<A*>(a.frag) + static_cast<long long>(blockIdx.x) * 2 * a.frag_rows * (D + 1);
  // One group of channels of a row (zeros where p is null), in the accumulators' type.
  auto fetch = [&](const T* p, int c) {
    Q4 r;
    const int c0 = c * V;
    if (p && a.wide) {
      struct alignas(V * sizeof(T)) Run {
        T x[V];
      };
      const Run w = *reinterpret_cast<const Run*>(p + c0);
#pragma unroll
      for (int e = 0; e < V; ++e) r.x[e] = static_cast<A>(to_acc(w.x[e]));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) r.x[e] = p && c0 + e < D ? static_cast<A>(to_acc(p[c0 + e])) : A(0);
    }
    return r;
  };

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // see paged_combine_kernel
  PagedWalk<false> walk;
  walk.init(a, paged_share<kSimtThreads, false>(a, share_sm));
  if (tid == 0) paged_meta_clear(a.meta);
  PagedPiece p;
  while (walk.next(a, p)) {
    const int row0 = p.u * ROWS;
    const int rows = min(ROWS, p.r.n * a.G - row0);
    if (tid == 0) paged_meta_piece(a.meta, p);
    __syncthreads();
    for (int i = tid; i < ROWS * dv; i += kSimtThreads) {
      const int r = i / dv, c = i - r * dv;
      const T* src = nullptr;
      if (r < rows) {
        const int tok = (row0 + r) / a.G, g = row0 + r - tok * a.G;
        src = q + (static_cast<long long>(p.r.tok0) + tok) * a.q_st + (static_cast<long long>(p.h) * a.G + g) * a.q_sh;
      }
      *reinterpret_cast<Q4*>(Qs + r * LD + c * V) = fetch(src, c);
    }
    A rs[TR];
    A o[RP][OC][V];
#pragma unroll
    for (int i = 0; i < TR; ++i) rs[i] = A(0);
#pragma unroll
    for (int i = 0; i < RP; ++i)
#pragma unroll
      for (int j = 0; j < OC; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) o[i][j][e] = A(0);
    const int k_end = p.tiles == 0 ? 0 : min(p.t1 * kPagedTile, p.r.len);
    const int prefix = p.r.len - p.r.n;
    for (int k0 = p.t0 * kPagedTile; k0 < k_end; k0 += BN) {
      __syncthreads();
      bool missing = false;
      if (tid < BN) {
        const int key = k0 + tid;
        long long ko = -1, vo = -1;
        if (key < p.r.len) {
          const int page = a.table[p.b * a.table_ld + (key >> a.page_shift)];
          const long long in = key & ((1 << a.page_shift) - 1);
          if (page >= 0 && page < a.num_pages) {
            ko = page * a.k_sp + p.h * a.k_sh + in * a.k_sr;
            vo = page * a.v_sp + p.h * a.v_sh + in * a.v_sr;
          }
        }
        k_row[tid] = ko;
        v_row[tid] = vo;
        missing = ko < 0;
      }
      const bool all_seen = !__syncthreads_or(missing) && k0 + BN <= prefix;
#pragma unroll 4
      for (int i = tid; i < BN * dv; i += kSimtThreads) {
        const int r = i / dv, c = i - r * dv;
        const long long ko = k_row[r], vo = v_row[r];
        const Q4 x = fetch(ko < 0 ? nullptr : static_cast<const T*>(a.k) + ko, c);
        const Q4 y = fetch(ko < 0 ? nullptr : static_cast<const T*>(a.v) + vo, c);
        *reinterpret_cast<Q4*>(Ks + r * LD + c * V) = x;
        *reinterpret_cast<Q4*>(Vs + r * LD + c * V) = y;
      }
      __syncthreads();
      A s[TR][TC];
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < TC; ++j) s[i][j] = A(0);
#pragma unroll 4
      for (int c = 0; c < dv; ++c) {
        Q4 x[TR], y[TC];
#pragma unroll
        for (int i = 0; i < TR; ++i) x[i] = *reinterpret_cast<const Q4*>(Qs + (ry + LY * i) * LD + c * V);
#pragma unroll
        for (int j = 0; j < TC; ++j) y[j] = *reinterpret_cast<const Q4*>(Ks + (kx + 8 * LX * j) * LD + c * V);
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
          for (int i = 0; i < TR; ++i)
#pragma unroll
            for (int j = 0; j < TC; ++j) s[i][j] = fma(x[i].x[e], y[j].x[e], s[i][j]);
      }
#pragma unroll
      for (int i = 0; i < TR; ++i) {
        const int r = ry + LY * i;
#pragma unroll
        for (int j = 0; j < TC; ++j) {
          const int c = kx + 8 * LX * j;
          bool in = all_seen;
          if (!all_seen && r < rows && k_row[c] >= 0)
            in = (paged_seen(a, p.r, (row0 + r) / a.G, k0 + (c & ~31)) >> (c & 31)) & 1u;
          const A pr = in ? octic_even(s[i][j] * scale) : A(0);
          rs[i] += pr;
          Ps[r * PLD + c] = pr;
        }
      }
      __syncthreads();
      A ot[RP][OC][V];
#pragma unroll
      for (int i = 0; i < RP; ++i)
#pragma unroll
        for (int j = 0; j < OC; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) ot[i][j][e] = A(0);
#pragma unroll 2
      for (int kk = ks * V; kk < BN; kk += C::KS * V) {
        Q4 pv[RP];
#pragma unroll
        for (int i = 0; i < RP; ++i) pv[i] = *reinterpret_cast<const Q4*>(Ps + (ro + C::RG * i) * PLD + kk);
#pragma unroll
        for (int j = 0; j < OC; ++j) {
          const int c = cg + C::CG * j;
          if (c < dv) {
#pragma unroll
            for (int y = 0; y < V; ++y) {
              const Q4 vv = *reinterpret_cast<const Q4*>(Vs + (kk + y) * LD + c * V);
#pragma unroll
              for (int i = 0; i < RP; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) ot[i][j][e] = fma(pv[i].x[y], vv.x[e], ot[i][j][e]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RP; ++i)
#pragma unroll
        for (int j = 0; j < OC; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) o[i][j][e] += ot[i][j][e];
    }
    // Row sums: over the lanes of a row, then over the warps in order.
#pragma unroll
    for (int i = 0; i < TR; ++i) {
#pragma unroll
      for (int off = LX / 2; off > 0; off >>= 1) rs[i] += __shfl_xor_sync(0xffffffffu, rs[i], off);
      if (lane % LX == 0) sums[warp][ry + LY * i] = rs[i];
    }
    if (C::KS == 2) {  // the second half of the keys, through the K tile
      if (ks == 1)
#pragma unroll
        for (int e = 0; e < V; ++e) Ks[ro * DMAX + cg * V + e] = o[0][0][e];
    }
    __syncthreads();
    if (C::KS == 2) {
      if (ks == 0)
#pragma unroll
        for (int e = 0; e < V; ++e) o[0][0][e] += Ks[ro * DMAX + cg * V + e];
    }
    const bool whole = p.whole();
    A* f = frag + static_cast<long long>(paged_frag_slot(p)) * a.frag_rows * (D + 1);
#pragma unroll
    for (int i = 0; i < RP; ++i) {
      const int r = ro + C::RG * i;
      if (r >= rows || ks != 0) continue;
      A total = A(0);
#pragma unroll
      for (int w = 0; w < 8; ++w) total += sums[w][r];
      const int tok = (row0 + r) / a.G;
      const long long orow = (static_cast<long long>(p.r.tok0) + tok) * a.Hkv * a.G +
                             static_cast<long long>(p.h) * a.G + (row0 + r - tok * a.G);
      const A denom = total + sink;
#pragma unroll
      for (int j = 0; j < OC; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (cg + C::CG * j) * V + e;
          if (c >= D) continue;
          if (whole)
            out[orow * D + c] = from_acc<T>(denom > A(0) ? o[i][j][e] / denom : A(0));
          else
            f[static_cast<long long>(r) * D + c] = o[i][j][e];
        }
      if (cg == 0) {
        if (!whole)
          f[static_cast<long long>(a.frag_rows) * D + r] = total;
        else if (dtot)
          dtot[orow] = denom;
      }
    }
  }
}

// Adds the fragments of the unit that CTA blockIdx.x of the attention kernel
// began and did not end, in CTA order, and writes its rows: a warp per row,
// blockIdx.y spreads the rows. It is launched with the attention kernel still
// running (programmatic dependent launch) and waits for it here: the launch and
// the first instructions cost nothing then.
constexpr int kCombineWarps = 8;
template <typename T, typename A, int W>
__global__ void __launch_bounds__(kCombineWarps * 32) paged_combine_kernel(const __grid_constant__ PagedArgs a,
                                                                           int ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int4 meta = *reinterpret_cast<const int4*>(a.meta + 4 * c);
  const int b = meta.y, h = meta.z, u = meta.w, D = a.D;
  if (b < 0) return;
  const int lane = threadIdx.x & 31;
  int last = c + 1;  // the CTA that ends the unit: 32 are looked at in one step
  while (true) {
    const unsigned ends = __ballot_sync(0xffffffffu, last + lane >= ctas - 1 || a.meta[4 * (last + lane)] != 0);
    if (ends) {
      last += __ffs(ends) - 1;
      break;
    }
    last += 32;
  }
  const PagedReq req = paged_req(a, b);
  const long long row0 = static_cast<long long>(u) * a.unit_rows;
  const int rows = static_cast<int>(min(static_cast<long long>(a.unit_rows), static_cast<long long>(req.n) * a.G - row0));
  const long long size = static_cast<long long>(a.frag_rows) * (D + 1);
  // Fragment x of the unit: CTA c's fragment 1, then the next CTAs' fragments 0.
  const A* frag = static_cast<const A*>(a.frag) + 2LL * c * size;
  const int n = last - c + 1;
  const A sink = sizeof(A) == 8 ? static_cast<A>(a.sink_d) : static_cast<A>(a.sink);
  const long long den_at = static_cast<long long>(a.frag_rows) * D;
  // Four fragments' loads are under way at once, whatever their number: with few
  // query rows a latency for each CTA's entry and fragment was most of this
  // kernel (one token against 4000 keys of 8 heads: 18.4 us together, now 15.6;
  // against 65536: 59.4, now 55.1).
  auto each = [&](auto&& load) {
    for (int x0 = 0; x0 < n; x0 += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = x0 + i;
        load(frag + (x == 0 ? size : 2LL * x * size), x < n);
      }
  };
  for (int r = blockIdx.y * kCombineWarps + (threadIdx.x >> 5); r < rows; r += gridDim.y * kCombineWarps) {
    A den = sink;
    each([&](const A* f, bool in) { den += in ? f[den_at + r] : A(0); });
    const long long row = row0 + r, tok = row / a.G;
    const long long orow = (req.tok0 + tok) * a.Hkv * a.G + static_cast<long long>(h) * a.G + (row - tok * a.G);
    T* out = static_cast<T*>(a.out) + orow * D;
    for (int col = lane * W; col < D; col += 32 * W) {
      const long long at = static_cast<long long>(r) * D + col;
      A sum[W] = {};
      each([&](const A* f, bool in) {
        alignas(16) A v[W] = {};
        if (in) {
          if constexpr (W * sizeof(A) == 16)
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(f + at);
          else
            v[0] = f[at];
        }
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] += v[i];
      });
      alignas(16) T y[W];
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = from_acc<T>(den > A(0) ? sum[i] / den : A(0));
      if constexpr (W * sizeof(T) == 8) {
        *reinterpret_cast<uint2*>(out + col) = *reinterpret_cast<const uint2*>(y);
      } else if constexpr (W * sizeof(T) == 16) {
        *reinterpret_cast<uint4*>(out + col) = *reinterpret_cast<const uint4*>(y);
      } else {
        out[col] = y[0];
      }
    }
    if (lane == 0 && a.dtot) static_cast<A*>(a.dtot)[orow] = den;
  }
}

// CTAs of a launch per SM: one of the tensor-core kernels fills an SM, of the
// CUDA-core kernel up to four fit (float32, 64 channels).
constexpr int kMaxSms = 148, kSimtPerSm = 4;

// `ctas` comes as the number of SMs and leaves as the number of CTAs: all that
// are resident at once, since equal shares in a second round would take as long
// again.
template <typename T, typename A, int ROWS, int BN, int DMAX>
cudaError_t launch_simt(const PagedArgs& a, int* ctas, cudaStream_t stream) {
  constexpr size_t smem = SimtCfg<A, ROWS, BN, DMAX>::kSmem;
  static_assert(smem <= 220 * 1024, "shared memory per CTA");
  static PerDeviceOnce setup;
  static int per_sm[kMaxDevices] = {};
  auto kern = afa_paged_simt_kernel<T, A, ROWS, BN, DMAX>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = setup.run(dev, [&] {
      const cudaError_t r =
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      return r != cudaSuccess ? r
                              : cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[dev], kern, kSimtThreads, smem);
    });
  if (e != cudaSuccess) return e;
  *ctas *= std::max(1, std::min(per_sm[dev], kSimtPerSm));
  kern<<<*ctas, kSimtThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename A, int ROWS>
cudaError_t launch_simt_rows(const PagedArgs& a, int* ctas, cudaStream_t stream) {
  if constexpr (sizeof(A) == 8) {
    if (a.D <= 128) return launch_simt<T, A, ROWS, 32, 128>(a, ctas, stream);
    return launch_simt<T, A, ROWS, 32, 256>(a, ctas, stream);
  } else {
    if (a.D <= 64) return launch_simt<T, A, ROWS, 64, 64>(a, ctas, stream);
    if (a.D <= 128) return launch_simt<T, A, ROWS, 64, 128>(a, ctas, stream);
    return launch_simt<T, A, ROWS, 32, 256>(a, ctas, stream);
  }
}

template <typename T, typename A>
cudaError_t launch_simt_type(const PagedArgs& a, int* ctas, cudaStream_t stream) {
  return a.unit_rows == 8 ? launch_simt_rows<T, A, 8>(a, ctas, stream) : launch_simt_rows<T, A, 32>(a, ctas, stream);
}

template <typename T, typename A, int W>
cudaError_t launch_combine_w(const PagedArgs& a, int ctas, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  int y = (a.frag_rows + kCombineWarps - 1) / kCombineWarps;
  if (y > 8) y = 8;  // 147 x 8 CTAs fill the SMs once
  cfg.gridDim = dim3(ctas - 1, y);
  cfg.blockDim = dim3(kCombineWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_combine_kernel<T, A, W>, a, ctas);
}

// 16 bytes of sums per lane where rows start on 16 bytes in the fragments and
// on a lane's share of 16 bytes in `out`.
template <typename T, typename A>
cudaError_t launch_combine(const PagedArgs& a, int ctas, cudaStream_t stream) {
  if (ctas < 2) return cudaSuccess;
  constexpr int W = 16 / sizeof(A);
  if (a.D % W == 0 && reinterpret_cast<uintptr_t>(a.out) % (W * sizeof(T)) == 0)
    return launch_combine_w<T, A, W>(a, ctas, stream);
  return launch_combine_w<T, A, 1>(a, ctas, stream);
}

int sm_count() {
  static PerDeviceOnce setup;
  static int count[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const cudaError_t e =
      setup.run(dev, [&] { return cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev); });
  return e == cudaSuccess ? count[dev] : 0;
}

// Rows of a CUDA-core unit: 8 where requests have no more on average (single
// tokens), else 32.
int simt_unit_rows(int B, int T, int G) {
  return (static_cast<long long>(T) + B - 1) / B * G <= 8 ? 8 : 32;
}

// A multiple of four, so that fragments start on 16 bytes whatever D is.
int frag_rows_of(int unit_rows, int T, int G) {
  const long long all = static_cast<long long>(T) * G;
  return ((all < unit_rows ? static_cast<int>(all) : unit_rows) + 3) / 4 * 4;
}

// Workspace: meta (4 ints per CTA), then two fragments per CTA.
constexpr size_t kMetaBytes = (static_cast<size_t>(kMaxSms) * kSimtPerSm * 4 * sizeof(int) + 255) / 256 * 256;

size_t workspace_bytes(int T, int Hq, int Hkv, int D, int dtype) {
  const size_t acc = dtype == kF64 ? 8 : 4;
  const int G = Hq / Hkv;
  size_t rows = static_cast<size_t>(kMaxSms) * kSimtPerSm * frag_rows_of(32, T, G);
  if (dtype == kBF16 && (D == 64 || D == 128) && G <= 128)  // the tensor-core kernels may run
    rows = std::max(rows, static_cast<size_t>(kMaxSms) * frag_rows_of(paged_tc_unit_rows(G), T, G));
  return kMetaBytes + 2 * rows * (static_cast<size_t>(D) + 1) * acc;
}

int invalid(const char* msg) { return set_last_error(AFA_ERR_INVALID, msg); }

}  // namespace
}  // namespace afa

extern "C" size_t afa_paged_workspace_bytes(int tokens, int q_heads, int kv_heads, int D, int dtype) {
  if (tokens <= 0 || kv_heads <= 0 || q_heads < kv_heads || D <= 0) return 0;
  return afa::workspace_bytes(tokens, q_heads, kv_heads, D, dtype);
}

extern "C" int afa_paged(const void* q, const long long* q_strides, const void* k_cache, const void* v_cache,
                         const long long* k_strides, const long long* v_strides, void* out, void* d_total,
                         const int* block_table, long long table_stride, const int* seq_lens, const int* cu_tokens,
                         const void* ancestors, long long ancestors_stride, int ancestor_words, int batch, int tokens,
                         int q_heads, int kv_heads, int D, int table_cols, int page_size, int num_pages, int dtype,
                         double sink_omega, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace afa;
  if (dtype == AFA_F16)
    return set_last_error(AFA_ERR_DTYPE, "float16 is not supported: rho(s)^8 overflows float16 for s > 2.4; use "
                                         "bfloat16 or float32");
  if (dtype != AFA_F32 && dtype != AFA_BF16 && dtype != AFA_F64)
    return set_last_error(AFA_ERR_DTYPE, "afa_paged: unsupported dtype code");
  if (batch < 0 || tokens < 0 || q_heads <= 0 || kv_heads <= 0 || D <= 0 || table_cols <= 0 || num_pages <= 0)
    return invalid("afa_paged: invalid shape");
  if (D > 256) return invalid("head dimension above 256 is not supported");
  if (q_heads % kv_heads != 0) return invalid("query heads must be a multiple of the cache's heads");
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return invalid("page_size must be a power of two from 16 to 256");
  // In the type that the sums have: float64 keeps all of it.
  const float sink = static_cast<float>(sink_omega);
  if (!(sink_omega >= 0.0 && (dtype == AFA_F64 ? std::isfinite(sink_omega) : std::isfinite(sink))))
    return invalid("sink_omega must be finite and nonnegative");
  if (static_cast<long long>(table_cols) * page_size > INT_MAX - 65536)
    return invalid("afa_paged: a block table row may hold at most 2^31 - 65537 tokens");
  if (static_cast<long long>(tokens) * q_heads > INT_MAX / 2) return invalid("afa_paged: too many query rows");
  if (ancestors && ancestor_words <= 0) return invalid("ancestors needs at least one word per token");
  if (tokens == 0 || batch == 0) return AFA_OK;
  if (!q || !k_cache || !v_cache || !out || !block_table || !seq_lens || !cu_tokens || !q_strides || !k_strides ||
      !v_strides)
    return invalid("afa_paged: null pointer");
  const size_t need = afa_paged_workspace_bytes(tokens, q_heads, kv_heads, D, dtype);
  if (!workspace || workspace_bytes < need) {
    char msg[128];
    snprintf(msg, sizeof(msg), "afa_paged needs a workspace of %zu bytes (got %zu)", need, workspace_bytes);
    return invalid(msg);
  }
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return invalid("afa_paged: the workspace must start on a 16-byte boundary");
  PagedArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.dtot = d_total;
  a.table = block_table;
  a.lens = seq_lens;
  a.cu = cu_tokens;
  a.anc = static_cast<const unsigned*>(ancestors);
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.k_sp = k_strides[0];
  a.k_sh = k_strides[1];
  a.k_sr = k_strides[2];
  a.v_sp = v_strides[0];
  a.v_sh = v_strides[1];
  a.v_sr = v_strides[2];
  // The stride of an axis of one element says nothing: any that fits TMA does.
  if (tokens == 1) a.q_st = 8;
  if (q_heads == 1) a.q_sh = 8;
  if (num_pages == 1) a.k_sp = a.v_sp = 8;
  if (kv_heads == 1) a.k_sh = a.v_sh = 8;
  a.table_ld = table_stride;
  a.anc_ld = ancestors_stride;
  a.words = ancestor_words;
  a.B = batch;
  a.T = tokens;
  a.Hkv = kv_heads;
  a.G = q_heads / kv_heads;
  a.D = D;
  a.table_cols = table_cols;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
  a.num_pages = num_pages;
  a.scale_d = 1.0 / std::sqrt(static_cast<double>(D));
  a.scale = static_cast<float>(a.scale_d);
  a.sink_d = sink_omega;
  a.sink = sink;
  a.meta = static_cast<int*>(workspace);
  a.frag = static_cast<char*>(workspace) + kMetaBytes;
  a.status = device_status_ptr();
  int ctas = std::min(sm_count(), kMaxSms);
  if (!a.status || ctas <= 0) return set_last_error(AFA_ERR_CUDA, "afa_paged: device set-up failed");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool tc = paged_tc_supported(a, dtype);
  const int nt = tc ? paged_tr_rows(batch, tokens, a.G) : 0;
  a.unit_rows = nt ? nt / a.G * a.G : tc ? paged_tc_unit_rows(a.G) : simt_unit_rows(batch, tokens, a.G);
  // Tensor cores: two key tiles at least (of a pair of query tiles, if most units are pairs).
  a.min_share = !tc ? 1 : nt || static_cast<long long>(tokens) * a.G / batch <= a.unit_rows / 2 ? 2 : 4;
  if (!tc) {
    const size_t es = dtype_size(dtype), run = es * (dtype == kF64 ? 2 : 4);  // a channel group in memory
    a.wide = static_cast<size_t>(D) * es % run == 0;
    for (const void* x : {a.q, a.k, a.v}) a.wide = a.wide && reinterpret_cast<uintptr_t>(x) % run == 0;
    for (long long s : {a.q_st, a.q_sh, a.k_sp, a.k_sh, a.k_sr, a.v_sp, a.v_sh, a.v_sr})
      a.wide = a.wide && s * static_cast<long long>(es) % static_cast<long long>(run) == 0;
  }
  a.out_wide = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  a.frag_rows = frag_rows_of(a.unit_rows, tokens, a.G);
  const char* detail = "";
  cudaError_t e;
  if (tc) {
    e = nt ? launch_paged_tr(a, nt, ctas, st, &detail) : launch_paged_tc(a, ctas, st, &detail);
  } else switch (dtype) {
    case kF64: e = launch_simt_type<double, double>(a, &ctas, st); break;
    case kF32: e = launch_simt_type<float, float>(a, &ctas, st); break;
    default: e = launch_simt_type<__nv_bfloat16, float>(a, &ctas, st); break;
  }
  if (e == cudaSuccess) {
    switch (dtype) {
      case kF64: e = launch_combine<double, double>(a, ctas, st); break;
      case kF32: e = launch_combine<float, float>(a, ctas, st); break;
      default: e = launch_combine<__nv_bfloat16, float>(a, ctas, st); break;
    }
  }
  if (e != cudaSuccess) {
    char msg[200];
    snprintf(msg, sizeof(msg), "afa_paged launch: %s %s", cudaGetErrorString(e), detail);
    return set_last_error(AFA_ERR_CUDA, msg);
  }
  return AFA_OK;
}
