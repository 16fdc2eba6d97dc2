// Block tables, slot maps and tree masks of one serving step, built on the GPU
// from the requests' lengths.
//
// The pages of the cache are handed out from a stack (free_pages, free_count).
// Request b holds the pages block_table[b][0 .. page_counts[b]); it has
// seq_lens[b] tokens and appends new_lens[b]. With ps tokens to a page,
//
//   want_b = seq_lens_b + new_lens_b,  need_b = ceil(want_b / ps)
//   drop_b = max(held_b - need_b, 0)   pages released (a rejected draft, an ended request)
//   grow_b = max(need_b - held_b, 0)   pages taken
//
// Released pages join the top of the stack in request order, then the requests
// take theirs from the top in request order. A request whose tokens or pages
// do not fit is refused and keeps what it holds. Token i of request b goes to
// slot block_table[b][(seq_lens_b + i) / ps] * ps + (seq_lens_b + i) % ps; with
// a drafted tree its position is seq_lens_b + depth and its ancestor words name
// the new tokens on its path to the root.
//
// Everything is an exclusive sum over the requests (tokens, released pages,
// taken pages), so one launch does it: every CTA computes the sums by itself
// and then writes its share of the tokens and of the table and stack entries.
// No CTA reads what another writes: the page taken i-th is looked up in the
// stack or in the released part of a table row, both of which the launch leaves
// as they are, and the per-request results go to arrays of their own.
#include <climits>
#include <cstdio>

#include "afa_b200.h"
#include "afa_common.cuh"
#include "afa_internal.h"

namespace afa {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxBatch = 4096;
constexpr int kPlanMaxNodes = 256;

struct PlanArgs {
  int* table;
  const int* held;
  const int* lens;
  const int* add;
  int* stack;
  const int* free_count;
  const int* parents;
  long long* slots;
  int* rows;
  int* positions;
  int* cu;
  int* lens_out;
  int* held_out;
  int* free_out;
  unsigned char* granted;
  unsigned* ancestors;
  int B, M, shift, N, max_tokens, nodes, words;
};

struct PlanReq {
  int held, len, add, need;
  long long want;
  bool too_long;
};

__device__ __forceinline__ PlanReq plan_req(const PlanArgs& a, int b) {
  PlanReq r;
  r.held = min(max(a.held[b], 0), a.M);
  r.len = max(a.lens[b], 0);
  r.add = max(a.add[b], 0);
  r.want = static_cast<long long>(r.len) + r.add;
  r.need = static_cast<int>((r.want + (1 << a.shift) - 1) >> a.shift);
  r.too_long = r.want > (static_cast<long long>(a.M) << a.shift) || (a.parents && r.add > a.nodes);
  return r;
}

// Inclusive sum over the block's threads of (x, y); `sm` holds 2 * warps + 2
// words, the totals at its end. Callers separate two sums by __syncthreads().
__device__ __forceinline__ longlong2 block_scan(longlong2 v, longlong2* sm, longlong2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) {
      v.x += x;
      v.y += y;
    }
  }
  __syncthreads();
  if (lane == 31) sm[warp] = v;
  __syncthreads();
  longlong2 before = make_longlong2(0, 0);
  total = make_longlong2(0, 0);
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const longlong2 s = sm[w];
    if (w < warp) {
      before.x += s.x;
      before.y += s.y;
    }
    total.x += s.x;
    total.y += s.y;
  }
  v.x += before.x;
  v.y += before.y;
  return v;
}

// Largest i in [0, n) with at[i] <= x (at ascends, at[0] = 0 <= x).
__device__ __forceinline__ int find(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int sm_plan[];
  __shared__ longlong2 sm_scan[kPlanThreads / 32];
  int* cu = sm_plan;             // B + 1: tokens before request b
  int* gone = cu + a.B + 1;      // B: pages released before request b
  int* grown = gone + a.B;       // B: pages taken before request b
  const int tid = threadIdx.x;
  const int fc = min(max(a.free_count[0], 0), a.N);

  // Tokens asked for, then pages, request by request.
  longlong2 total;
  long long tok = 0, drops = 0, grows = 0;
  for (int c0 = 0; c0 < a.B; c0 += kPlanThreads) {
    const int b = c0 + tid;
    PlanReq r{};
    if (b < a.B) r = plan_req(a, b);
    const long long ask = b < a.B && !r.too_long ? r.add : 0;
    const longlong2 t = block_scan(make_longlong2(ask, 0), sm_scan, total);
    const bool off = b >= a.B || r.too_long || (ask > 0 && tok + t.x > a.max_tokens);
    tok += total.x;
    const longlong2 d = make_longlong2(off ? 0 : max(r.held - r.need, 0), off ? 0 : max(r.need - r.held, 0));
    const longlong2 p = block_scan(d, sm_scan, total);
    if (b < a.B) {
      gone[b] = static_cast<int>(drops + p.x - d.x);
      // Refused: marked by the sign; the sum stays below 2^31 (checked on the host).
      grown[b] = static_cast<int>(grows + p.y - d.y);
      cu[b] = off ? -1 : static_cast<int>(d.y);
    }
    drops += total.x;
    grows += total.y;
  }
  __syncthreads();
  const int F = static_cast<int>(drops);
  const long long supply = static_cast<long long>(fc) + F;
  long long before = 0, taken = 0;
  for (int c0 = 0; c0 < a.B; c0 += kPlanThreads) {
    const int b = c0 + tid;
    int n = 0, take = 0;
    if (b < a.B) {
      const PlanReq r = plan_req(a, b);
      const int grow = cu[b];
      const bool ok = grow >= 0 && (grow == 0 || static_cast<long long>(grown[b]) + grow <= supply);
      n = ok ? r.add : 0;
      take = ok ? grow : 0;
      if (blockIdx.x == 0) {
        a.granted[b] = ok;
        a.lens_out[b] = ok ? static_cast<int>(r.want) : r.len;
        a.held_out[b] = ok ? r.need : r.held;
      }
    }
    const longlong2 t = block_scan(make_longlong2(n, take), sm_scan, total);
    if (b < a.B) {
      cu[b] = static_cast<int>(before + t.x - n);
      if (blockIdx.x == 0) a.cu[b] = cu[b];
    }
    before += total.x;
    taken += total.y;
  }
  const int T = static_cast<int>(before), A = static_cast<int>(taken);
  if (tid == 0) {
    cu[a.B] = T;
    if (blockIdx.x == 0) {
      a.cu[a.B] = T;
      a.free_out[0] = min(fc + F - A, a.N);  // what finds no room on the stack is not on it
    }
  }
  __syncthreads();

  // e-th released page; i-th taken one, from the top of stack + released.
  auto released = [&](int e) {
    const int b = find(gone, a.B, e);
    return a.table[static_cast<long long>(b) * a.M + plan_req(a, b).need + (e - gone[b])];
  };
  auto taken_page = [&](int i) {
    const int s = fc + F - 1 - i;
    return s < fc ? a.stack[s] : released(s - fc);
  };
  const int step = gridDim.x * kPlanThreads;
  const int id = blockIdx.x * kPlanThreads + tid;
  for (int e = id; e < A; e += step) {
    const int b = find(grown, a.B, e);
    a.table[static_cast<long long>(b) * a.M + min(max(a.held[b], 0), a.M) + (e - grown[b])] = taken_page(e);
  }
  for (int e = id; e < F - A; e += step)
    if (fc + e < a.N) a.stack[fc + e] = released(e);
  for (int t = id; t < a.max_tokens; t += step) {
    long long slot = -1;
    int row = -1, pos = 0;
    if (t < T) {
      row = find(cu, a.B, t);
      const int len = max(a.lens[row], 0), node = t - cu[row];
      const int held = min(max(a.held[row], 0), a.M);
      const int at = (len + node) >> a.shift;
      const int page = at < held ? a.table[static_cast<long long>(row) * a.M + at] : taken_page(grown[row] + at - held);
      slot = (static_cast<long long>(page) << a.shift) + ((len + node) & ((1 << a.shift) - 1));
      pos = len + node;
      if (a.parents) {
        const int* par = a.parents + static_cast<long long>(row) * a.nodes;
        unsigned w[kPlanMaxNodes / 32] = {};
        int depth = 0, i = node;
        while (true) {
#pragma unroll
          for (int k = 0; k < kPlanMaxNodes / 32; ++k) w[k] |= (i >> 5) == k ? 1u << (i & 31) : 0u;
          const int up = par[i];
          if (up < 0 || up >= i) break;
          i = up;
          ++depth;
        }
        pos = len + depth;
#pragma unroll
        for (int k = 0; k < kPlanMaxNodes / 32; ++k)
          if (k < a.words) a.ancestors[static_cast<long long>(t) * a.words + k] = w[k];
      }
    } else if (a.parents) {
      for (int k = 0; k < a.words; ++k) a.ancestors[static_cast<long long>(t) * a.words + k] = 0u;
    }
    a.slots[t] = slot;
    a.rows[t] = row;
    a.positions[t] = pos;
  }
}

int invalid(const char* msg) { return set_last_error(AFA_ERR_INVALID, msg); }

}  // namespace
}  // namespace afa

extern "C" int afa_paged_plan(int* block_table, const int* page_counts, const int* seq_lens, const int* new_lens,
                              int* free_pages, const int* free_count, const int* parents, long long* slots, int* rows,
                              int* positions, int* cu_tokens, int* seq_lens_out, int* page_counts_out,
                              int* free_count_out, unsigned char* granted, void* ancestors, int batch, int table_cols,
                              int page_size, int num_free, int max_tokens, int nodes, void* stream) {
  using namespace afa;
  if (batch <= 0 || batch > kPlanMaxBatch) return invalid("afa_paged_plan: batch must be in [1, 4096]");
  if (table_cols <= 0 || num_free <= 0 || max_tokens < 0 || max_tokens > (1 << 30))
    return invalid("afa_paged_plan: invalid shape");
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return invalid("page_size must be a power of two from 16 to 256");
  if (static_cast<long long>(table_cols) * page_size > INT_MAX - 65536 ||
      static_cast<long long>(table_cols) * batch > INT_MAX - num_free)
    return invalid("afa_paged_plan: block table too large");
  if (parents && (nodes <= 0 || nodes > kPlanMaxNodes)) return invalid("a tree may have at most 256 nodes");
  if (!block_table || !page_counts || !seq_lens || !new_lens || !free_pages || !free_count || !cu_tokens ||
      !seq_lens_out || !page_counts_out || !free_count_out || !granted ||
      (max_tokens > 0 && (!slots || !rows || !positions || (parents && !ancestors))))
    return invalid("afa_paged_plan: null pointer");
  PlanArgs a{block_table, page_counts, seq_lens, new_lens, free_pages, free_count, parents, slots, rows, positions,
             cu_tokens, seq_lens_out, page_counts_out, free_count_out, granted, static_cast<unsigned*>(ancestors),
             batch, table_cols, __builtin_ctz(static_cast<unsigned>(page_size)), num_free, max_tokens,
             parents ? nodes : 0, parents ? (nodes + 31) / 32 : 0};
  const size_t smem = (3 * static_cast<size_t>(batch) + 1) * sizeof(int);
  long long blocks = (static_cast<long long>(max_tokens) + kPlanThreads - 1) / kPlanThreads;
  if (blocks > 148) blocks = 148;
  if (blocks < 1) blocks = 1;
  static PerDeviceOnce setup;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = setup.run(dev, [&] {
      return cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>((3 * kPlanMaxBatch + 1) * sizeof(int)));
    });
  if (e == cudaSuccess) {
    paged_plan_kernel<<<static_cast<int>(blocks), kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) {
    char msg[200];
    snprintf(msg, sizeof(msg), "afa_paged_plan launch: %s", cudaGetErrorString(e));
    return set_last_error(AFA_ERR_CUDA, msg);
  }
  return AFA_OK;
}
