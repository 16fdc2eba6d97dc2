// Rotary positions with several axes, the write of new keys and values into a
// paged cache, and the move of a drafted tree's accepted path to its front.
//
//   afa_ago_rotate_axes  AGO Cayley rotations (src/attention.py:142-152,
//                   :210-240) where every axis of a token's position (time,
//                   height, width) turns channel pairs of its own: pair p of
//                   axis a(p) at positions[a(p)][token] = m becomes
//                   (c x0 - s x1, s x0 + c x1) with c, s = tables[m][p]. A
//                   rotation's inverse is its transpose, so the gradient is the
//                   same pass with -s. Pairs behind the last axis stay.
//   afa_paged_append     the same for new keys on their way into the cache
//                   (row slots[token] of it) beside their values, and for the
//                   queries: one launch between the projection and attention.
//   afa_paged_commit     cache row base + i <- row base + accepted[i].
//
// All are bound by HBM: each element is read once and written once in 16-byte
// accesses; a thread keeps the cosines and sines of its channel pairs in
// registers over kHeadsPerThread heads of its token, since reading them for
// every head would move more table than data.
#include <climits>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "afa_b200.h"
#include "afa_common.cuh"
#include "afa_internal.h"

namespace afa {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kHeadsPerThread = 4;
constexpr int kRowThreads = 256;
constexpr int kRowCtas = 148 * 4;  // resident at once

// One of the row sets of a launch: heads x D of every token, from src to dst.
struct RowSet {
  const void* src;
  void* dst;
  long long s_b, s_t, s_h;  // source strides (elements): batch, token, head
  long long d_b, d_t, d_h;  // destination strides; in the cache: page, row, head
  int heads, groups;        // groups = ceil(heads / kHeadsPerThread)
  int turn, cache;          // rotate; write to cache row slots[token]
};

struct RowArgs {
  RowSet set[3];
  int sets;
  const void* c;
  const void* s;
  const void* positions;  // [axis][batch][token], strides p_a, p_b, p_t
  const long long* slots;
  long long p_a, p_b, p_t;
  long long rows;         // cache rows: pages << page_shift
  int pos64, batch, tokens, D, table_len, page_shift, groups, backward, table_runs;
  int end[kMaxAxes];      // pairs [end[a-1], end[a]) belong to axis a; unused axes end at the last
};

__device__ __forceinline__ long long load_index(const void* p, long long i, int is64) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// NaN for a position the tables do not hold.
template <typename A> __device__ __forceinline__ A not_a_number();
template <> __device__ __forceinline__ float not_a_number<float>() { return __int_as_float(0x7fffffff); }
template <> __device__ __forceinline__ double not_a_number<double>() { return __longlong_as_double(0x7fffffffffffffffll); }

template <typename TT, int P>
struct alignas(sizeof(TT) * P < 16 ? sizeof(TT) * P : 16) TableRun {
  TT x[P];
};

// E elements (E / 2 channel pairs) of a row per thread: 16 bytes, or one pair
// when rows are not 16-byte aligned. Consecutive threads take the chunks of a
// row and then the next token, so that a warp's accesses are contiguous where
// rows of a head follow each other (the attention layout), and whole rows
// otherwise. A thread reads its cosines and sines once and walks every
// gridDim.y-th group of kHeadsPerThread heads, whose loads go out together.
template <typename T, typename TT, typename A, int E, typename V>
__global__ void __launch_bounds__(kRowThreads, 4) paged_rows_kernel(const __grid_constant__ RowArgs a) {
  constexpr int P = E / 2;
  const int chunks = a.D / E, pairs = a.D / 2;
  const int idx = blockIdx.x * kRowThreads + threadIdx.x;
  const int t = idx / chunks;
  if (t >= a.tokens) return;
  const int e0 = (idx - t * chunks) * E, p0 = e0 / 2;
  const int end = a.end[kMaxAxes - 1];  // pairs from here on are not turned
  for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
    A cc[P], ss[P];
    if (p0 < end) {
      auto axis_of = [&](int pair) { return (pair >= a.end[0]) + (pair >= a.end[1]) + (pair >= a.end[2]); };
      auto position = [&](int axis) {
        return load_index(a.positions, axis * a.p_a + b * a.p_b + t * a.p_t, a.pos64);
      };
      const int first = axis_of(p0);
      if (P > 1 && a.table_runs && p0 + P <= end && axis_of(p0 + P - 1) == first) {
        // The usual case: all pairs of the chunk belong to one axis.
        const long long m = position(first);
        if (m >= 0 && m < a.table_len) {
          const auto cr = *reinterpret_cast<const TableRun<TT, P>*>(static_cast<const TT*>(a.c) + m * pairs + p0);
          const auto sr = *reinterpret_cast<const TableRun<TT, P>*>(static_cast<const TT*>(a.s) + m * pairs + p0);
#pragma unroll
          for (int p = 0; p < P; ++p) {
            cc[p] = static_cast<A>(to_acc(cr.x[p]));
            ss[p] = static_cast<A>(to_acc(sr.x[p]));
          }
        } else {
#pragma unroll
          for (int p = 0; p < P; ++p) cc[p] = ss[p] = not_a_number<A>();
        }
      } else {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (p0 + p >= end) continue;
          const long long m = position(axis_of(p0 + p));
          const bool in_table = m >= 0 && m < a.table_len;
          const long long i = m * pairs + p0 + p;
          cc[p] = in_table ? static_cast<A>(to_acc(static_cast<const TT*>(a.c)[i])) : not_a_number<A>();
          ss[p] = in_table ? static_cast<A>(to_acc(static_cast<const TT*>(a.s)[i])) : not_a_number<A>();
        }
      }
      if (a.backward) {
#pragma unroll
        for (int p = 0; p < P; ++p) ss[p] = -ss[p];
      }
    }
    for (int x = blockIdx.y; x < a.groups; x += gridDim.y) {
      int group = x, si = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (si == i && i + 1 < a.sets && group >= a.set[i].groups) {
          group -= a.set[i].groups;
          ++si;
        }
      const RowSet& S = a.set[si];
      long long at = 0;
      if (S.cache) {
        const long long slot = a.slots[t];
        if (slot < 0 || slot >= a.rows) continue;
        at = (slot >> a.page_shift) * S.d_b + (slot & ((1 << a.page_shift) - 1)) * S.d_t;
      } else {
        at = b * S.d_b + t * S.d_t;
      }
      const int h0 = group * kHeadsPerThread, nh = S.heads - h0;
      const T* src = static_cast<const T*>(S.src) + b * S.s_b + t * S.s_t + h0 * S.s_h + e0;
      T* dst = static_cast<T*>(S.dst) + at + h0 * S.d_h + e0;
      V in[kHeadsPerThread];
#pragma unroll
      for (int j = 0; j < kHeadsPerThread; ++j) {
        if (j < nh) in[j] = *reinterpret_cast<const V*>(src);
        src += S.s_h;
      }
      const bool turn = S.turn && p0 < end;
#pragma unroll
      for (int j = 0; j < kHeadsPerThread; ++j) {
        if (turn) {
          T y[E];
          memcpy(y, &in[j], sizeof(V));
#pragma unroll
          for (int p = 0; p < P; ++p) {
            if (p0 + p >= end) continue;
            const A x0 = static_cast<A>(to_acc(y[2 * p])), x1 = static_cast<A>(to_acc(y[2 * p + 1]));
            // Which product is rounded is said here, not left to the compiler: the wide
            // and the narrow kernel give the same bits.
            y[2 * p] = from_acc<T>(fma(cc[p], x0, -(ss[p] * x1)));
            y[2 * p + 1] = from_acc<T>(fma(ss[p], x0, cc[p] * x1));
          }
          memcpy(&in[j], y, sizeof(V));
        }
        if (j < nh) *reinterpret_cast<V*>(dst) = in[j];
        dst += S.d_h;
      }
    }
  }
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = uint32_t; };
template <> struct Pair<float> { using type = uint2; };
template <> struct Pair<double> { using type = uint4; };

template <typename T, typename TT, typename A>
cudaError_t launch_rows_tt(RowArgs a, bool wide, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  if (a.batch == 0 || a.tokens == 0) return cudaSuccess;
  const long long items = static_cast<long long>(a.tokens) * (a.D / (wide ? E : 2));
  if (items > INT_MAX - kRowThreads) return cudaErrorInvalidConfiguration;
  // Heads are spread over CTAs as far as it takes to have kRowCtas of them.
  const long long x = (items + kRowThreads - 1) / kRowThreads, z = a.batch < 65535 ? a.batch : 65535;
  long long y = (kRowCtas + x * z - 1) / (x * z);
  if (y > a.groups) y = a.groups;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y), static_cast<unsigned>(z));
  // A chunk's table values in one or two loads, where its run of pairs is aligned.
  const size_t run = sizeof(TT) * (E / 2) < 16 ? sizeof(TT) * (E / 2) : 16;
  a.table_runs = (a.D / 2) % (E / 2) == 0 && reinterpret_cast<uintptr_t>(a.c) % run == 0 &&
                 reinterpret_cast<uintptr_t>(a.s) % run == 0;
  if (wide)
    paged_rows_kernel<T, TT, A, E, uint4><<<grid, kRowThreads, 0, stream>>>(a);
  else
    paged_rows_kernel<T, TT, A, 2, typename Pair<T>::type><<<grid, kRowThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename A>
cudaError_t launch_rows_t(const RowArgs& a, int table_dtype, bool wide, cudaStream_t stream) {
  switch (table_dtype) {
    case kF32: return launch_rows_tt<T, float, A>(a, wide, stream);
    case kBF16: return launch_rows_tt<T, __nv_bfloat16, A>(a, wide, stream);
    case kF64: return launch_rows_tt<T, double, A>(a, wide, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_rows(const RowArgs& a, int dtype, int table_dtype, bool wide, cudaStream_t stream) {
  switch (dtype) {
    case kF64: return launch_rows_t<double, double>(a, table_dtype, wide, stream);
    case kF32: return launch_rows_t<float, float>(a, table_dtype, wide, stream);
    case kBF16: return launch_rows_t<__nv_bfloat16, float>(a, table_dtype, wide, stream);
    default: return cudaErrorInvalidValue;
  }
}

bool ok_dtype(int dt) { return dt == kF32 || dt == kBF16 || dt == kF64; }
int invalid(const char* msg) { return set_last_error(AFA_ERR_INVALID, msg); }
int fail_cuda(const char* what, cudaError_t e) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return set_last_error(AFA_ERR_CUDA, msg);
}

// Whether rows at these addresses can be accessed `unit` bytes at a time.
bool aligned(const void* p, size_t unit, size_t esize, std::initializer_list<long long> strides) {
  if (reinterpret_cast<uintptr_t>(p) % unit != 0) return false;
  for (long long s : strides)
    if (static_cast<unsigned long long>(s) * esize % unit != 0) return false;
  return true;
}

// The stride of an axis of one entry says nothing and is never multiplied by
// anything but 0: it does not count against the alignment of rows.
long long used(long long stride, int entries) { return entries > 1 ? stride : 0; }

// The axes' channel pairs as running ends; false when they do not fit.
bool set_axes(RowArgs& a, const int* sections, int axes) {
  int at = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < axes) {
      if (sections[i] < 0 || sections[i] > a.D / 2 - at) return false;
      at += sections[i];
    }
    a.end[i] = at;
  }
  return true;
}

// ---------------------------------------------------------------------------
// Commit
// ---------------------------------------------------------------------------
constexpr int kCommitThreads = 256;
constexpr int kMaxPath = 256;
constexpr int kCommitBatch = 8;  // rows in flight per thread

struct CommitArgs {
  void* k;
  void* v;
  const int* table;
  const int* base;
  const int* lens;
  const int* accepted;
  int* lens_out;
  long long k_l, k_p, k_h, k_r, v_l, v_p, v_h, v_r;  // strides in units of V
  long long table_ld, acc_ld;
  int layers, heads, chunks, cols, path, shift, num_pages;
};

// One CTA row (blockIdx.x) per request; its threads and blockIdx.y share the
// columns (cache, layer, head, chunk of a row). A column's rows move in order:
// accepted[i] ascends, so accepted[i] >= i and a row is written only after it,
// and every row before it, has been read; kCommitBatch loads go out together,
// and the rows they read lie at or behind those the stores before wrote.
template <typename V>
__global__ void __launch_bounds__(kCommitThreads) paged_commit_kernel(const __grid_constant__ CommitArgs a) {
  __shared__ int s_page[2][kMaxPath];  // source, destination
  __shared__ int s_row[2][kMaxPath];
  __shared__ int s_count;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int base = max(a.base[b], 0);
  const long long cap = min(static_cast<long long>(a.lens[b]), static_cast<long long>(a.cols) << a.shift);
  if (tid == 0) s_count = a.path;
  __syncthreads();
  for (int i = tid; i < a.path; i += kCommitThreads) {
    const int node = a.accepted[b * a.acc_ld + i];
    const int prev = i > 0 ? a.accepted[b * a.acc_ld + i - 1] : -1;
    const long long src = static_cast<long long>(base) + node, dst = static_cast<long long>(base) + i;
    bool ok = node >= 0 && node > prev && src < cap && dst < cap;
    int ps = 0, pd = 0;
    if (ok) {
      ps = a.table[b * a.table_ld + (src >> a.shift)];
      pd = a.table[b * a.table_ld + (dst >> a.shift)];
      ok = ps >= 0 && ps < a.num_pages && pd >= 0 && pd < a.num_pages;
    }
    if (!ok) atomicMin(&s_count, i);
    s_page[0][i] = ps;
    s_page[1][i] = pd;
    s_row[0][i] = static_cast<int>(src) & ((1 << a.shift) - 1);
    s_row[1][i] = static_cast<int>(dst) & ((1 << a.shift) - 1);
  }
  __syncthreads();
  const int n = s_count;
  if (tid == 0 && blockIdx.y == 0) a.lens_out[b] = base + n;
  const long long cols = 2LL * a.layers * a.heads * a.chunks;
  for (long long c = static_cast<long long>(blockIdx.y) * kCommitThreads + tid; c < cols;
       c += static_cast<long long>(gridDim.y) * kCommitThreads) {
    long long x = c / a.chunks;
    const int chunk = static_cast<int>(c - x * a.chunks);
    const int h = static_cast<int>(x % a.heads);
    x /= a.heads;
    const int layer = static_cast<int>(x % a.layers);
    const bool is_v = x / a.layers != 0;
    V* p = static_cast<V*>(is_v ? a.v : a.k) + layer * (is_v ? a.v_l : a.k_l) + h * (is_v ? a.v_h : a.k_h) + chunk;
    const long long sp = is_v ? a.v_p : a.k_p, sr = is_v ? a.v_r : a.k_r;
    for (int i0 = 0; i0 < n; i0 += kCommitBatch) {
      V r[kCommitBatch];
#pragma unroll
      for (int j = 0; j < kCommitBatch; ++j)
        if (i0 + j < n) r[j] = p[s_page[0][i0 + j] * sp + s_row[0][i0 + j] * sr];
#pragma unroll
      for (int j = 0; j < kCommitBatch; ++j)
        if (i0 + j < n) p[s_page[1][i0 + j] * sp + s_row[1][i0 + j] * sr] = r[j];
    }
  }
}

template <typename V>
cudaError_t launch_commit(CommitArgs a, int batch, int row_bytes, size_t esize, cudaStream_t stream) {
  a.chunks = row_bytes / static_cast<int>(sizeof(V));
  const long long q = static_cast<long long>(sizeof(V) / esize);
  for (long long* s : {&a.k_l, &a.k_p, &a.k_h, &a.k_r, &a.v_l, &a.v_p, &a.v_h, &a.v_r}) *s /= q;
  const long long cols = 2LL * a.layers * a.heads * a.chunks;
  long long y = (cols + kCommitThreads - 1) / kCommitThreads;
  if (y > 1024) y = 1024;
  paged_commit_kernel<V><<<dim3(batch, static_cast<unsigned>(y)), kCommitThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace afa

extern "C" int afa_ago_rotate_axes(const void* q, const long long* q_strides, void* q_out, int q_heads, const void* k,
                                   const long long* k_strides, void* k_out, int k_heads, const void* c, const void* s,
                                   int table_dtype, int table_len, const void* positions,
                                   const long long* position_strides, int positions_64, const int* sections, int axes,
                                   int token_major, int batch, int tokens, int dim, int backward, int dtype,
                                   void* stream) {
  using namespace afa;
  if (!ok_dtype(dtype) || !ok_dtype(table_dtype))
    return set_last_error(AFA_ERR_DTYPE, "afa_ago_rotate_axes: dtypes must be float32, bfloat16 or float64");
  if (dim <= 0 || dim % 2 != 0) return invalid("Feature dimension must be even");
  if (batch < 0 || tokens < 0 || q_heads <= 0 || (k && k_heads <= 0) || table_len <= 0)
    return invalid("afa_ago_rotate_axes: invalid shape");
  if (axes < 1 || axes > kMaxAxes || !sections) return invalid("between one and four position axes are supported");
  RowArgs a{};
  a.D = dim;
  if (!set_axes(a, sections, axes)) return invalid("sections must be nonnegative and sum to at most dim / 2");
  if (batch == 0 || tokens == 0) return AFA_OK;
  if (!q || !q_strides || !q_out || !c || !s || !positions || !position_strides || (k && (!k_strides || !k_out)))
    return invalid("afa_ago_rotate_axes: null pointer");
  a.sets = k ? 2 : 1;
  bool wide = dim * dtype_size(dtype) % 16 == 0;
  for (int i = 0; i < a.sets; ++i) {
    const long long* st = i ? k_strides : q_strides;
    const int heads = i ? k_heads : q_heads;
    RowSet& S = a.set[i];
    S.src = i ? k : q;
    S.dst = i ? k_out : q_out;
    S.s_b = used(st[0], batch);
    S.s_t = used(st[1], tokens);
    S.s_h = used(st[2], heads);
    S.d_b = static_cast<long long>(heads) * tokens * dim;
    S.d_t = token_major ? static_cast<long long>(heads) * dim : dim;
    S.d_h = token_major ? dim : static_cast<long long>(tokens) * dim;
    S.heads = heads;
    S.groups = (heads + kHeadsPerThread - 1) / kHeadsPerThread;
    S.turn = 1;
    a.groups += S.groups;
    wide = wide && aligned(S.src, 16, dtype_size(dtype), {S.s_b, S.s_t, S.s_h}) && aligned(S.dst, 16, 1, {});
    if (!aligned(S.src, 2 * dtype_size(dtype), dtype_size(dtype), {S.s_b, S.s_t, S.s_h}) ||
        !aligned(S.dst, 2 * dtype_size(dtype), 1, {}))
      return invalid("afa_ago_rotate_axes: rows must start at a channel pair's alignment");
  }
  a.c = c;
  a.s = s;
  a.table_len = table_len;
  a.positions = positions;
  a.pos64 = positions_64;
  a.p_a = position_strides[0];
  a.p_b = position_strides[1];
  a.p_t = position_strides[2];
  a.batch = batch;
  a.tokens = tokens;
  a.backward = backward;
  const cudaError_t e = launch_rows(a, dtype, table_dtype, wide, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? AFA_OK : fail_cuda("afa_ago_rotate_axes launch", e);
}

extern "C" int afa_paged_append(const void* k, const long long* k_strides, const void* v, const long long* v_strides,
                                void* k_cache, const long long* k_cache_strides, void* v_cache,
                                const long long* v_cache_strides, const long long* slots, const void* q,
                                const long long* q_strides, void* q_out, int q_heads, const void* c, const void* s,
                                int table_dtype, int table_len, const void* positions,
                                const long long* position_strides, int positions_64, const int* sections, int axes,
                                int tokens, int kv_heads, int dim, int num_pages, int page_size, int dtype,
                                void* stream) {
  using namespace afa;
  if (!ok_dtype(dtype) || (c && !ok_dtype(table_dtype)))
    return set_last_error(AFA_ERR_DTYPE, "afa_paged_append: dtypes must be float32, bfloat16 or float64");
  if (dim <= 0 || dim % 2 != 0) return invalid("Feature dimension must be even");
  if (tokens < 0 || kv_heads <= 0 || num_pages <= 0 || (q && q_heads <= 0))
    return invalid("afa_paged_append: invalid shape");
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return invalid("page_size must be a power of two from 16 to 256");
  RowArgs a{};
  a.D = dim;
  if (c) {
    if (!s || table_len <= 0) return invalid("afa_paged_append: invalid tables");
    if (axes < 1 || axes > kMaxAxes || !sections) return invalid("between one and four position axes are supported");
    if (!set_axes(a, sections, axes)) return invalid("sections must be nonnegative and sum to at most dim / 2");
  } else if (q) {
    return invalid("q is only rotated: it needs rotary tables");
  }
  if (tokens == 0) return AFA_OK;
  if (!k || !v || !k_strides || !v_strides || !k_cache || !v_cache || !k_cache_strides || !v_cache_strides || !slots ||
      (q && (!q_strides || !q_out)) || (c && (!positions || !position_strides)))
    return invalid("afa_paged_append: null pointer");
  const size_t es = dtype_size(dtype);
  bool wide = dim * es % 16 == 0, pairs = true;
  a.sets = q ? 3 : 2;
  for (int i = 0; i < a.sets; ++i) {  // k, v, q
    const long long* st = i == 0 ? k_strides : i == 1 ? v_strides : q_strides;
    const long long* cs = i == 0 ? k_cache_strides : v_cache_strides;
    RowSet& S = a.set[i];
    S.src = i == 0 ? k : i == 1 ? v : q;
    S.dst = i == 0 ? k_cache : i == 1 ? v_cache : q_out;
    S.s_b = 0;
    S.heads = i == 2 ? q_heads : kv_heads;
    S.s_t = used(st[0], tokens);
    S.s_h = used(st[1], S.heads);
    S.d_b = i == 2 ? 0 : used(cs[0], num_pages);
    S.d_t = i == 2 ? static_cast<long long>(q_heads) * dim : cs[2];
    S.d_h = i == 2 ? dim : used(cs[1], kv_heads);
    S.groups = (S.heads + kHeadsPerThread - 1) / kHeadsPerThread;
    S.turn = i != 1 && c;
    S.cache = i != 2;
    a.groups += S.groups;
    for (size_t unit : {size_t(16), 2 * es}) {
      const bool fits = aligned(S.src, unit, es, {S.s_t, S.s_h}) && aligned(S.dst, unit, es, {S.d_b, S.d_t, S.d_h});
      (unit == 16 ? wide : pairs) &= fits;
    }
  }
  if (!pairs) return invalid("afa_paged_append: rows must start at a channel pair's alignment");
  a.c = c;
  a.s = s;
  a.table_len = table_len;
  a.positions = positions;
  if (c) {
    a.pos64 = positions_64;
    a.p_a = position_strides[0];
    a.p_t = position_strides[1];
  }
  a.slots = slots;
  a.rows = static_cast<long long>(num_pages) * page_size;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
  a.batch = 1;
  a.tokens = tokens;
  const cudaError_t e = launch_rows(a, dtype, c ? table_dtype : static_cast<int>(kF32), wide,
                                    static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? AFA_OK : fail_cuda("afa_paged_append launch", e);
}

extern "C" int afa_paged_commit(void* k_cache, const long long* k_strides, void* v_cache, const long long* v_strides,
                                const int* block_table, long long table_stride, const int* base_lens,
                                const int* seq_lens, const int* accepted, long long accepted_stride, int* lens_out,
                                int batch, int path, int layers, int kv_heads, int dim, int table_cols, int num_pages,
                                int page_size, int dtype, void* stream) {
  using namespace afa;
  if (!ok_dtype(dtype))
    return set_last_error(AFA_ERR_DTYPE, "afa_paged_commit: dtypes must be float32, bfloat16 or float64");
  if (batch < 0 || path < 0 || layers <= 0 || kv_heads <= 0 || dim <= 0 || table_cols <= 0 || num_pages <= 0)
    return invalid("afa_paged_commit: invalid shape");
  if (path > kMaxPath) return invalid("an accepted path may have at most 256 tokens");
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return invalid("page_size must be a power of two from 16 to 256");
  if (static_cast<long long>(table_cols) * page_size > INT_MAX - 65536)
    return invalid("afa_paged_commit: a block table row may hold at most 2^31 - 65537 tokens");
  if (batch == 0) return AFA_OK;
  if (!k_cache || !v_cache || !k_strides || !v_strides || !block_table || !base_lens || !seq_lens || !lens_out ||
      (path > 0 && !accepted))
    return invalid("afa_paged_commit: null pointer");
  CommitArgs a{};
  a.k = k_cache;
  a.v = v_cache;
  a.table = block_table;
  a.base = base_lens;
  a.lens = seq_lens;
  a.accepted = accepted;
  a.lens_out = lens_out;
  a.k_l = used(k_strides[0], layers);
  a.k_p = used(k_strides[1], num_pages);
  a.k_h = used(k_strides[2], kv_heads);
  a.k_r = k_strides[3];
  a.v_l = used(v_strides[0], layers);
  a.v_p = used(v_strides[1], num_pages);
  a.v_h = used(v_strides[2], kv_heads);
  a.v_r = v_strides[3];
  a.table_ld = table_stride;
  a.acc_ld = accepted_stride;
  a.layers = layers;
  a.heads = kv_heads;
  a.cols = table_cols;
  a.path = path;
  a.shift = __builtin_ctz(static_cast<unsigned>(page_size));
  a.num_pages = num_pages;
  const size_t es = dtype_size(dtype);
  const int row_bytes = dim * static_cast<int>(es);
  const bool wide = row_bytes % 16 == 0 && aligned(k_cache, 16, es, {a.k_l, a.k_p, a.k_h, a.k_r}) &&
                    aligned(v_cache, 16, es, {a.v_l, a.v_p, a.v_h, a.v_r});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (wide)
    e = launch_commit<uint4>(a, batch, row_bytes, es, st);
  else if (es == 2)
    e = launch_commit<unsigned short>(a, batch, row_bytes, es, st);
  else if (es == 4)
    e = launch_commit<unsigned>(a, batch, row_bytes, es, st);
  else
    e = launch_commit<unsigned long long>(a, batch, row_bytes, es, st);
  return e == cudaSuccess ? AFA_OK : fail_cuda("afa_paged_commit launch", e);
}
