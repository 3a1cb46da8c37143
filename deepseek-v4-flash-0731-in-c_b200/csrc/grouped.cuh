// grouped.cuh - products of many rows grouped by expert, and the routed
// experts of a MoE layer built from them.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace dsv4 {

constexpr int kGroupedMaxExperts = 1024;

// Row r of group e (offsets[e] <= r < offsets[e + 1]) is multiplied with
// matrix e. All device pointers.
struct GroupedProblem {
  int experts = 0, rows = 0;  // groups; bound of offsets
  int outs = 0, width = 0;    // outputs and inputs of a matrix
  bool fp8 = false;           // weights: E4M3 with E8M0 per 128 x 128, else E2M1 per 32
  const uint8_t* w[2] = {nullptr, nullptr};   // [experts][outs][width] (E2M1: width / 2)
  const uint8_t* ws[2] = {nullptr, nullptr};  // the second pair: the up matrix of a gated product
  const uint8_t* xq = nullptr;     // [x_rows][width] E4M3
  const uint8_t* xs = nullptr;     // [x_rows][width / 128] E8M0
  int x_rows = 0;
  const int* offsets = nullptr;    // [experts + 1]
  const int* src = nullptr;        // [rows] row of xq, or null: r
  const int* dst = nullptr;        // [rows] row of out, or null: r
  int out_rows = 0;
  void* out = nullptr;             // [out_rows] rows of outs, fp32 or BF16
  bool bf16 = true;
  long long out_stride = 0;
  // gated (w[1] given): E4M3 codes and E8M0 scales per 128 of
  // silu(min(g, limit)) * clamp(u, -limit, limit) * weight[r], row r
  float limit = 0.f;
  const float* weight = nullptr;   // [rows] or null
  uint8_t* hq = nullptr;           // [rows][outs]
  uint8_t* hs = nullptr;           // [rows][outs / 128]
  unsigned* err = nullptr;         // device error word
};

// The workspace starts with counters that have to be zero; grouped_reset
// makes them so.
size_t grouped_workspace_bytes(const GroupedProblem& p);
cudaError_t grouped_reset(void* ws, cudaStream_t st);
cudaError_t grouped_forward(const GroupedProblem& p, void* ws, cudaStream_t st);

// The routed experts of n tokens: gate and up products, SwiGLU, route weight
// and quantisation, down products, and each token's sum in route order.
struct ExpertsProblem {
  int n = 0, topk = 0, hidden = 0, inter = 0;
  int lo = 0, experts = 0;  // this device's experts are lo .. lo + experts - 1
  const uint8_t *w1 = nullptr, *s1 = nullptr, *w3 = nullptr, *s3 = nullptr, *w2 = nullptr,
                *s2 = nullptr;
  float limit = 0.f;
  const uint8_t *xq = nullptr, *xs = nullptr;  // [n][hidden], [n][hidden / 128]
  const int* idx = nullptr;                    // [n][topk]
  const float* wt = nullptr;                   // [n][topk]
  uint16_t* out = nullptr;                     // [n][hidden] BF16
  unsigned* err = nullptr;
};
size_t experts_workspace_bytes(const ExpertsProblem& p);
cudaError_t experts_forward(const ExpertsProblem& p, void* ws, cudaStream_t st);

}  // namespace dsv4
