// logprob.cuh - log probabilities of given tokens, entropy and top alternatives.
#pragma once
#include <cuda_runtime.h>

namespace dsv4 {

constexpr int kMaxTopAlternatives = 32;

struct LogprobProblem {
  const void* logits = nullptr;  // [rows] rows of vocab values, fp32 or BF16
  bool bf16 = false;
  int rows = 0, vocab = 0;
  long long stride = 0;          // elements between rows
  const int* tokens = nullptr;   // [rows]; outside [0, vocab): none asked for
  float* logprob = nullptr;      // [rows]
  float* entropy = nullptr;      // [rows] or null
  int* rank = nullptr;           // [rows] or null
  int top = 0;                   // 0 .. kMaxTopAlternatives
  int* top_id = nullptr;         // [rows][top]
  float* top_logprob = nullptr;  // [rows][top]
};

cudaError_t token_logprobs(const LogprobProblem& p, cudaStream_t st);

}  // namespace dsv4
