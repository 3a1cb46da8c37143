// logprob.cu - log probabilities of given tokens over rows of logits.
//
// Per row x[V] with m = max x, Z = sum e^(x - m):
//   logprob = x_t - m - log Z
//   entropy = log Z - sum e^(x - m) (x - m) / Z        (a masked -inf adds 0)
//   rank    = #(x > x_t) + #(x == x_t at a lower index)
//   top     = the k largest, the lower index first among equals (-0 == 0)
// A row that is all -inf gives -inf log probabilities and entropy 0; a NaN
// or +inf in a row makes its log probabilities and entropy NaN. NaN never
// competes for the top alternatives: a place left over holds id -1 and NaN.
#include "logprob.cuh"

#include <climits>
#include <cmath>
#include <cuda_bf16.h>

namespace dsv4 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load(const LogprobProblem& p, int row, int i) {
  const long long at = row * p.stride + i;
  return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at])
                : static_cast<const float*>(p.logits)[at];
}

template <class T, class F>
__device__ T block_fold(T v, F f) {
  __shared__ T part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < kThreads / 32; ++w) v = f(v, part[w]);
  return v;
}

__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobProblem p) {
  const int row = blockIdx.x;
  const int t = p.tokens[row];
  const bool asked = t >= 0 && t < p.vocab;
  const float xt = asked ? load(p, row, t) : 0.f;
  float m = -INFINITY;
  int above = 0, nan = 0;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
    const float x = load(p, row, i);
    m = fmaxf(m, x);
    above += x > xt || (x == xt && i < t);
    nan |= x != x;
  }
  m = block_fold(m, [](float a, float b) { return fmaxf(a, b); });
  above = block_fold(above, [](int a, int b) { return a + b; });
  nan = block_fold(nan, [](int a, int b) { return a | b; });
  const float ref = m == -INFINITY ? 0.f : m;
  float z = 0.f, xz = 0.f;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
    const float d = load(p, row, i) - ref, e = expf(d);
    z += e;
    if (e > 0.f) xz = fmaf(e, d, xz);
  }
  auto add = [](float a, float b) { return a + b; };
  z = block_fold(z, add);
  xz = block_fold(xz, add);
  const bool undefined = nan || m == INFINITY;
  const float lz = m == -INFINITY ? 0.f : logf(z);
  if (threadIdx.x == 0) {
    p.logprob[row] = !asked ? 0.f : undefined ? NAN : xt - ref - lz;
    if (p.entropy) p.entropy[row] = undefined ? NAN : m == -INFINITY ? 0.f : lz - xz / z;
    if (p.rank) p.rank[row] = asked ? above : -1;
  }
  // k rounds, each the largest behind the last one taken
  float lx = INFINITY;
  int li = -1;
  for (int k = 0; k < p.top; ++k) {
    float bx = -INFINITY;
    int bi = INT_MAX;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
      const float x = load(p, row, i);
      const bool left = x < lx || (x == lx && i > li);
      if (left && (x > bx || bi == INT_MAX)) { bx = x; bi = i; }
    }
    const float best = block_fold(bi == INT_MAX ? -INFINITY : bx,
                                  [](float a, float b) { return fmaxf(a, b); });
    const int at = block_fold(bi != INT_MAX && bx == best ? bi : INT_MAX,
                              [](int a, int b) { return min(a, b); });
    if (threadIdx.x == 0) {
      p.top_id[static_cast<long long>(row) * p.top + k] = at == INT_MAX ? -1 : at;
      p.top_logprob[static_cast<long long>(row) * p.top + k] =
          at == INT_MAX || undefined ? NAN : best - ref - lz;
    }
    lx = best;
    li = at == INT_MAX ? INT_MAX : at;
  }
}

}  // namespace

cudaError_t token_logprobs(const LogprobProblem& p, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  logprob_kernel<<<p.rows, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dsv4
