// paged_attn.cuh - attention of new tokens over the paged latent cache.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"

namespace dsv4 {

// One layer's cache and the tables, as the attention kernels take them.
struct PagedLayer {
  const uint8_t* codes;
  const uint8_t* scales;
  const uint16_t* rope;
  int nope, rope_dim;
  int page, n_pages, n_seqs, max_pages;
  const int* table;
  const int* length;
  unsigned* status;
};

struct PagedAttnProblem {
  PagedLayer pages;
  const void* q = nullptr;          // [total][H][d] BF16 or fp32 (BF16-valued)
  void* out = nullptr;              // as q
  bool bf16 = true;
  long long q_stride = 0;           // elements between tokens of q / out
  long long out_stride = 0;
  const int* q_start = nullptr;     // [n_seqs + 1] first row of each slot's new tokens
  const float* sink = nullptr;      // [H] or null
  const float* rope_cos = nullptr;  // [total][rope_out / 2] or null (no inverse RoPE)
  const float* rope_sin = nullptr;
  int rope_out = 0;                 // inverse RoPE on the last rope_out dims
  float* lse = nullptr;             // [total][H] or null
  int total = 0, H = 0;
  int max_new = 0, max_len = 0;     // bounds of one slot's new tokens and length
  int window = 0;                   // 0: every earlier position
  long long max_keys = 0;           // bound of the positions seen, all slots together
  float scale = 0.f;
  unsigned* err = nullptr;          // device error word
  bool out_32 = false;              // rows of out (BF16) are 32-byte aligned
  bool rope_vec = false;            // RoPE factors of 32 dims are whole, aligned vectors
};

size_t paged_attn_workspace_bytes(const PagedAttnProblem& p);
cudaError_t paged_attn_forward(const PagedAttnProblem& p, void* ws, cudaStream_t st);

}  // namespace dsv4
