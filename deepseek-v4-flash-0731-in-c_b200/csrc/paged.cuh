// paged.cuh - the latent cache in pages: tables, reference counts, page copies.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace dsv4 {

constexpr int kPagedMaxLayers = 64;   // caches that share one set of tables
constexpr int kPagedMaxSeqs = 4096;   // slots, and ops of one call

// Bits of the status word.
constexpr unsigned kPagedExhausted = 1u;  // an op did not find the free pages it needs
constexpr unsigned kPagedBadOp = 2u;      // an op that is not one (slot out of range, named twice, ...)
constexpr unsigned kPagedBounds = 4u;     // a sequence beyond the bounds given to the attention call

// Passed to the kernels by value. All layers have rows of the same size;
// cache row of position p of slot s = table[s][p / page] * page + p % page.
struct PagedState {
  uint8_t* codes[kPagedMaxLayers];
  uint8_t* scales[kPagedMaxLayers];
  uint16_t* rope[kPagedMaxLayers];
  int layers, nope, rope_dim;
  int page, n_pages, n_seqs, max_pages;
  int* table;        // [n_seqs][max_pages], -1 = no page
  int* length;       // [n_seqs]
  int* refs;         // [n_pages] table entries that name the page, 0 (or less) = free
  unsigned* status;  // may be null
  void* ws;          // paged_workspace_bytes()
};

size_t paged_workspace_bytes(int n_pages, int n_seqs);

// Slot dst[i] takes the place of a copy of slot src[i] (-1, or src null:
// emptied).
cudaError_t paged_fork(const PagedState& p, const int* dst, const int* src, int n,
                       cudaStream_t st);
// Slot slots[i] grows by counts[i] tokens; rows (may be null) receives the
// cache rows of the new tokens, op after op, and -1 behind them.
cudaError_t paged_append(const PagedState& p, const int* slots, const int* counts, int n,
                         long long* rows, long long n_rows, cudaStream_t st);
// Pages in use move to the lowest page numbers; table_out / refs_out may be
// the state's own.
cudaError_t paged_compact(const PagedState& p, int* table_out, int* refs_out, cudaStream_t st);

}  // namespace dsv4
