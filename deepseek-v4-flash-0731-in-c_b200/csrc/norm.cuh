// norm.cuh - RMS norm of rows with an 8-bit output, and new latents on their
// way into the pages.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "attn.cuh"

namespace dsv4 {

constexpr int kNormMaxWidth = 32768;

struct NormProblem {
  int rows = 0, width = 0;
  bool bf16 = true;                 // x, residual, sum, out
  const void* x = nullptr;          // rows, x_stride elements apart
  const void* residual = nullptr;   // or null
  void* sum = nullptr;              // x + residual, or null; may be x or residual
  void* out = nullptr;              // the normalised rows, or null
  long long x_stride = 0, residual_stride = 0, sum_stride = 0, out_stride = 0;
  const uint16_t* gain = nullptr;   // [width] BF16 or null
  float eps = 0.f;
  uint8_t* codes = nullptr;         // [rows][width] E4M3
  uint8_t* scales = nullptr;        // [rows][ceil(width / 128)] E8M0
};
cudaError_t norm_quant(const NormProblem& p, cudaStream_t st);

struct LatentWrite {
  Fp8KvCache cache;
  const void* kv = nullptr;         // n rows of nope + rope_dim values, stride elements apart
  bool bf16 = true;
  long long stride = 0;
  const long long* rows = nullptr;  // [n] cache rows; outside the cache: left out
  int n = 0;
  const uint16_t* gain = nullptr;   // [nope + rope_dim] BF16, or null: no norm
  float eps = 0.f;
  const float* rope_cos = nullptr;  // [n][rope_dim / 2] or null: no rotation
  const float* rope_sin = nullptr;
};
cudaError_t latent_write(const LatentWrite& p, cudaStream_t st);

}  // namespace dsv4
