// beam.cuh - selection of beams over their continuations, and the slots that
// the chosen ones take.
#pragma once
#include <cuda_runtime.h>

namespace dsv4 {

constexpr int kMaxBeams = 32;
constexpr int kMaxBeamCandidates = 32;

struct BeamProblem {
  const void* logits = nullptr;  // [groups * beams] rows of vocab values, fp32 or BF16
  bool bf16 = false;
  int groups = 0, beams = 0, vocab = 0;
  long long stride = 0;          // elements between rows
  const float* score = nullptr;  // [groups][beams]
  int cands = 0;
  int* parent = nullptr;         // [groups][cands] beam, -1: none
  int* token = nullptr;
  float* total = nullptr;
  int eos = -1;
  int* next = nullptr;           // [groups][beams] candidate, -1: none
  const int* slot = nullptr;     // [groups][beams], or null
  int* dst = nullptr;            // [groups][beams]
  int* src = nullptr;
};

cudaError_t beam_select(const BeamProblem& p, cudaStream_t st);

}  // namespace dsv4
