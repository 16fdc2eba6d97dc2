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
#include <climits>
#include <cmath>
#include <cstdio>

#include "afa_b200.h"
#include "afa_common.cuh"
#include "afa_internal.h"
#include "afa_paged.cuh"

namespace afa {
namespace {

constexpr int kSimtRows = 32;
constexpr int kSimtThreads = 256;

// 32 query rows x BN keys per step, 16 x 16 threads; thread (ty, tx) owns
// scores (ty + 16 i, tx + 16 j) and outputs (ty + 16 i, tx + 16 j'), so that
// shared-memory reads (row pitch DMAX + 1) are free of bank conflicts. Sums run
// over BN keys in registers of their own before they join the row's, which
// keeps float32 results near 1e-7 at any length.
template <typename T, typename A, int BN, int DMAX>
__global__ void __launch_bounds__(kSimtThreads) afa_paged_simt_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int LD = DMAX + 1, PLD = BN + 1, TR = kSimtRows / 16, TC = BN / 16, OC = DMAX / 16;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ long long share_sm[kSimtThreads / 32 + 4];
  __shared__ unsigned char in_cache[BN];
  A* Qs = reinterpret_cast<A*>(smem_raw);
  A* Ks = Qs + kSimtRows * LD;
  A* Vs = Ks + BN * LD;
  A* Ps = Vs + BN * LD;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, D = a.D;
  const T* q = static_cast<const T*>(a.q);
  const T* k = static_cast<const T*>(a.k);
  const T* v = static_cast<const T*>(a.v);
  T* out = static_cast<T*>(a.out);
  A* dtot = static_cast<A*>(a.dtot);
  const A scale = sizeof(A) == 8 ? static_cast<A>(a.scale_d) : static_cast<A>(a.scale);
  const A sink = sizeof(A) == 8 ? static_cast<A>(a.sink_d) : static_cast<A>(a.sink);
  A* frag = static_cast<A*>(a.frag) + static_cast<long long>(blockIdx.x) * 2 * a.frag_rows * (D + 1);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // see paged_combine_kernel
  PagedWalk walk;
  walk.init(a, paged_share<kSimtThreads>(a, share_sm));
  if (tid == 0) paged_meta_clear(a.meta);
  PagedPiece p;
  while (walk.next(a, p)) {
    const long long row0 = static_cast<long long>(p.u) * kSimtRows;
    const int rows = static_cast<int>(min(static_cast<long long>(kSimtRows), static_cast<long long>(p.r.n) * a.G - row0));
    if (tid == 0) paged_meta_piece(a.meta, p);
    __syncthreads();
    for (int i = tid; i < kSimtRows * D; i += kSimtThreads) {
      const int r = i / D, c = i - r * D;
      A x = A(0);
      if (r < rows) {
        const long long row = row0 + r;
        const long long tok = row / a.G;
        const int g = static_cast<int>(row - tok * a.G);
        x = static_cast<A>(to_acc(q[(p.r.tok0 + tok) * a.q_st + (static_cast<long long>(p.h) * a.G + g) * a.q_sh + c]));
      }
      Qs[r * LD + c] = x;
    }
    int node[TR];
    A o[TR][OC], rs[TR];
#pragma unroll
    for (int i = 0; i < TR; ++i) {
      const int r = ty + 16 * i;
      node[i] = r < rows ? static_cast<int>((row0 + r) / a.G) : -1;
      rs[i] = A(0);
#pragma unroll
      for (int j = 0; j < OC; ++j) o[i][j] = A(0);
    }
    const int k_end = min(p.t1 * kPagedTile, p.tiles == 0 ? 0 : p.r.len);
    for (int k0 = p.t0 * kPagedTile; k0 < k_end; k0 += BN) {
      __syncthreads();
      for (int i = tid; i < BN * D; i += kSimtThreads) {
        const int r = i / D, c = i - r * D, key = k0 + r;
        A kx = A(0), vx = A(0);
        if (key < p.r.len) {
          const int page = a.table[p.b * a.table_ld + (key >> a.page_shift)];
          const long long in = key & ((1 << a.page_shift) - 1);
          const bool ok = page >= 0 && page < a.num_pages;
          if (c == 0) in_cache[r] = ok;
          if (ok) {
            kx = static_cast<A>(to_acc(k[page * a.k_sp + p.h * a.k_sh + in * a.k_sr + c]));
            vx = static_cast<A>(to_acc(v[page * a.v_sp + p.h * a.v_sh + in * a.v_sr + c]));
          }
        }
        Ks[r * LD + c] = kx;
        Vs[r * LD + c] = vx;
      }
      __syncthreads();
      A s[TR][TC];
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < TC; ++j) s[i][j] = A(0);
      for (int d = 0; d < D; ++d) {
        A x[TR], y[TC];
#pragma unroll
        for (int i = 0; i < TR; ++i) x[i] = Qs[(ty + 16 * i) * LD + d];
#pragma unroll
        for (int j = 0; j < TC; ++j) y[j] = Ks[(tx + 16 * j) * LD + d];
#pragma unroll
        for (int i = 0; i < TR; ++i)
#pragma unroll
          for (int j = 0; j < TC; ++j) s[i][j] = fma(x[i], y[j], s[i][j]);
      }
#pragma unroll
      for (int i = 0; i < TR; ++i) {
        A part = A(0);
#pragma unroll
        for (int w = 0; w < (BN + 31) / 32; ++w) {
          const unsigned seen = node[i] < 0 ? 0u : paged_seen(a, p.r, node[i], k0 + 32 * w);
#pragma unroll
          for (int j = 0; j < TC; ++j) {
            const int c = tx + 16 * j;
            if (c / 32 != w) continue;
            const A pr = ((seen >> (c & 31)) & 1u) && in_cache[c] ? octic_ref(s[i][j] * scale) : A(0);
            part += pr;
            Ps[(ty + 16 * i) * PLD + c] = pr;
          }
        }
        rs[i] += part;
      }
      __syncthreads();
      A ot[TR][OC];
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < OC; ++j) ot[i][j] = A(0);
#pragma unroll 4
      for (int kk = 0; kk < BN; ++kk) {
        A pv[TR];
#pragma unroll
        for (int i = 0; i < TR; ++i) pv[i] = Ps[(ty + 16 * i) * PLD + kk];
#pragma unroll
        for (int j = 0; j < OC; ++j) {
          const int c = tx + 16 * j;
          if (c < D) {
            const A vv = Vs[kk * LD + c];
#pragma unroll
            for (int i = 0; i < TR; ++i) ot[i][j] = fma(pv[i], vv, ot[i][j]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < OC; ++j) o[i][j] += ot[i][j];
    }
    // The 16 threads of a half-warp share their rows.
#pragma unroll
    for (int i = 0; i < TR; ++i) {
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) rs[i] += __shfl_xor_sync(0xffffffffu, rs[i], off);
      const int r = ty + 16 * i;
      if (r >= rows) continue;
      if (p.whole()) {
        const long long row = row0 + r, tok = p.r.tok0 + row / a.G;
        const long long orow = tok * a.Hkv * a.G + static_cast<long long>(p.h) * a.G + row % a.G;
        const A denom = rs[i] + sink;
#pragma unroll
        for (int j = 0; j < OC; ++j) {
          const int c = tx + 16 * j;
          if (c < D) out[orow * D + c] = from_acc<T>(denom > A(0) ? o[i][j] / denom : A(0));
        }
        if (tx == 0 && dtot) dtot[orow] = denom;
      } else {
        A* f = frag + static_cast<long long>(paged_frag_slot(p)) * a.frag_rows * (D + 1);
#pragma unroll
        for (int j = 0; j < OC; ++j) {
          const int c = tx + 16 * j;
          if (c < D) f[r * D + c] = o[i][j];
        }
        if (tx == 0) f[a.frag_rows * D + r] = rs[i];
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
  int last = c + 1;
  while (last < ctas - 1 && a.meta[4 * last] == 0) ++last;
  const PagedReq req = paged_req(a, b);
  const long long row0 = static_cast<long long>(u) * a.unit_rows;
  const int rows = static_cast<int>(min(static_cast<long long>(a.unit_rows), static_cast<long long>(req.n) * a.G - row0));
  const long long size = static_cast<long long>(a.frag_rows) * (D + 1);
  const A* first = static_cast<const A*>(a.frag) + (2LL * c + 1) * size;
  const A* rest = static_cast<const A*>(a.frag) + 2LL * (c + 1) * size;  // of CTA c + 1; 2 * size apart
  const int nrest = last - c;
  const A sink = sizeof(A) == 8 ? static_cast<A>(a.sink_d) : static_cast<A>(a.sink);
  const int lane = threadIdx.x & 31;
  const long long den_at = static_cast<long long>(a.frag_rows) * D;
  for (int r = blockIdx.y * kCombineWarps + (threadIdx.x >> 5); r < rows; r += gridDim.y * kCombineWarps) {
    A den = first[den_at + r];
#pragma unroll 4
    for (int x = 0; x < nrest; ++x) den += rest[2LL * x * size + den_at + r];
    den += sink;
    const long long row = row0 + r, tok = row / a.G;
    const long long orow = (req.tok0 + tok) * a.Hkv * a.G + static_cast<long long>(h) * a.G + (row - tok * a.G);
    T* out = static_cast<T*>(a.out) + orow * D;
    for (int col = lane * W; col < D; col += 32 * W) {
      const long long at = static_cast<long long>(r) * D + col;
      A sum[W];
      auto add = [&](const A* f, bool set) {
        alignas(16) A v[W];
        if constexpr (W * sizeof(A) == 16)
          *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(f + at);
        else
          v[0] = f[at];
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] = set ? v[i] : sum[i] + v[i];
      };
      add(first, true);
#pragma unroll 4
      for (int x = 0; x < nrest; ++x) add(rest + 2LL * x * size, false);
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

template <typename T, typename A, int BN, int DMAX>
cudaError_t launch_simt(const PagedArgs& a, int ctas, cudaStream_t stream) {
  constexpr size_t smem = sizeof(A) * (static_cast<size_t>(kSimtRows + 2 * BN) * (DMAX + 1) +
                                       static_cast<size_t>(kSimtRows) * (BN + 1));
  static PerDeviceOnce setup;
  auto kern = afa_paged_simt_kernel<T, A, BN, DMAX>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = setup.run(dev, [&] {
      return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    });
  if (e != cudaSuccess) return e;
  kern<<<ctas, kSimtThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename A>
cudaError_t launch_simt_type(const PagedArgs& a, int ctas, cudaStream_t stream) {
  if constexpr (sizeof(A) == 8) {
    if (a.D <= 128) return launch_simt<T, A, 32, 128>(a, ctas, stream);
    return launch_simt<T, A, 32, 256>(a, ctas, stream);
  } else {
    if (a.D <= 64) return launch_simt<T, A, 64, 64>(a, ctas, stream);
    if (a.D <= 128) return launch_simt<T, A, 64, 128>(a, ctas, stream);
    return launch_simt<T, A, 32, 256>(a, ctas, stream);
  }
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

constexpr int kMaxPagedCtas = 148;

// Query rows per work unit and the workspace layout: meta, then fragments.
// Sized for the tensor-core kernel's units where it may run.
int max_unit_rows(int dtype, int G, int D) {
  return dtype == kBF16 && (D == 64 || D == 128) && G <= 128 ? paged_tc_unit_rows(G) : kSimtRows;
}
// A multiple of four, so that fragments start on 16 bytes whatever D is.
int frag_rows_of(int unit_rows, int T, int G) {
  const long long all = static_cast<long long>(T) * G;
  return ((all < unit_rows ? static_cast<int>(all) : unit_rows) + 3) / 4 * 4;
}
constexpr size_t kMetaBytes = (static_cast<size_t>(kMaxPagedCtas) * 4 * sizeof(int) + 255) / 256 * 256;

size_t workspace_bytes(int T, int Hq, int Hkv, int D, int dtype) {
  const size_t acc = dtype == kF64 ? 8 : 4;
  const size_t rows = frag_rows_of(max_unit_rows(dtype, Hq / Hkv, D), T, Hq / Hkv);
  return kMetaBytes + static_cast<size_t>(kMaxPagedCtas) * 2 * rows * (static_cast<size_t>(D) + 1) * acc;
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
                         float sink_omega, void* workspace, size_t workspace_bytes, void* stream) {
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
  if (!(std::isfinite(sink_omega) && sink_omega >= 0.f)) return invalid("sink_omega must be finite and nonnegative");
  if (static_cast<long long>(table_cols) * page_size > INT_MAX - 65536)
    return invalid("afa_paged: a block table row may hold at most 2^31 - 65537 tokens");
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
  a.sink_d = static_cast<double>(sink_omega);
  a.sink = sink_omega;
  a.meta = static_cast<int*>(workspace);
  a.frag = static_cast<char*>(workspace) + kMetaBytes;
  a.status = device_status_ptr();
  int ctas = sm_count();
  if (!a.status || ctas <= 0) return set_last_error(AFA_ERR_CUDA, "afa_paged: device set-up failed");
  if (ctas > kMaxPagedCtas) ctas = kMaxPagedCtas;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool tc = paged_tc_supported(a, dtype);
  const int nt = tc ? paged_tr_rows(batch, tokens, a.G) : 0;
  a.unit_rows = nt ? nt / a.G * a.G : tc ? paged_tc_unit_rows(a.G) : kSimtRows;
  a.frag_rows = frag_rows_of(a.unit_rows, tokens, a.G);
  const char* detail = "";
  cudaError_t e;
  if (tc) {
    e = nt ? launch_paged_tr(a, nt, ctas, st, &detail) : launch_paged_tc(a, ctas, st, &detail);
  } else switch (dtype) {
    case kF64: e = launch_simt_type<double, double>(a, ctas, st); break;
    case kF32: e = launch_simt_type<float, float>(a, ctas, st); break;
    default: e = launch_simt_type<__nv_bfloat16, float>(a, ctas, st); break;
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
