// Arguments and host interfaces of the attention over a paged key/value cache
// (afa_paged.cu, afa_paged_tc.cu).
#pragma once

#include <cstddef>
#include <cuda_runtime.h>

namespace afa {

// Keys per tile: the unit the work is counted and split in.
constexpr int kPagedTile = 128;

// Strides are in elements.
struct PagedArgs {
  const void* q;            // (tokens, Hkv * G, D): q_st between tokens, q_sh between heads
  const void* k;            // (pages, Hkv, page size, D): k_sp / k_sh / k_sr
  const void* v;
  void* out;                // (tokens, Hkv * G, D), contiguous
  void* dtot;               // (tokens, Hkv * G) accumulation dtype, may be null
  const int* table;         // (B, table_cols), rows table_ld apart
  const int* lens;          // (B,) keys of each request, its new tokens included
  const int* cu;            // (B + 1,) first token of each request
  const unsigned* anc;      // (tokens, words) visible new tokens, or null: causal
  long long q_st, q_sh, k_sp, k_sh, k_sr, v_sp, v_sh, v_sr, table_ld, anc_ld;
  int B, T, Hkv, G, D, table_cols, page_shift, num_pages, words;
  int unit_rows;            // query rows (token, head of the group) per work unit
  int frag_rows;            // rows of a fragment: unit_rows, or all rows there can be if fewer
  int min_share;            // cost of a CTA's share below which fewer CTAs run
  int wide;                 // CUDA cores: rows can be read a channel group at a time
  int out_wide;             // out starts on 16 bytes
  double scale_d, sink_d;
  float scale, sink;
  int* meta;                // workspace: 4 ints per CTA (see PagedPiece)
  void* frag;               // workspace: two fragments of frag_rows * (D + 1) sums per CTA
  int* status;
};

bool paged_tc_supported(const PagedArgs& a, int dtype);
// The tensor-core kernel's launch shape: query rows per work unit, CTAs.
int paged_tc_unit_rows(int G);
// Query rows per unit of the transposed kernel for this batch (16 or 32; a
// unit has the largest multiple of G up to it), or 0 when the rows a request
// has on average are too many for it.
int paged_tr_rows(int B, int T, int G);
cudaError_t launch_paged_tr(const PagedArgs& a, int nt, int ctas, cudaStream_t stream, const char** detail);
cudaError_t launch_paged_tc(const PagedArgs& a, int ctas, cudaStream_t stream, const char** detail);

}  // namespace afa
