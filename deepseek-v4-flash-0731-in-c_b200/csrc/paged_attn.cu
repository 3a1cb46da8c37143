// paged_attn.cu - attention of new tokens over the paged latent cache.
//
// Token i of slot s is at position p = length[s] - new_s + i and sees the
// positions t <= p (with a window: t > p - window) whose page the table
// names. With k_t = v_t the latent row:
//   x_t = scale * q . k_t,  M = max(max_t x_t, sink)
//   den = exp(sink - M) + sum_t exp(x_t - M)
//   o   = sum_t exp(x_t - M) k_t / den,  lse = M + log den
// then the inverse RoPE of the last dims in fp32 and one rounding to BF16.
// A token that sees nothing and has no sink gets o = 0, lse = -inf. A seen
// row that holds a NaN or an infinity makes the token's output NaN; rows that
// a token does not see have no effect on it, whatever they hold.
#include "paged_attn.cuh"

#include <cmath>
#include <cuda_bf16.h>

#include "attn.cuh"
#include "dsv4_common.cuh"

namespace dsv4 {
namespace {

constexpr int kMaxDim = 1024;              // of the general kernel
constexpr int kLaneDims = kMaxDim / 32;
constexpr int kSimtWarps = 8;

__device__ __forceinline__ float latent_value(const PagedState& c, int layer, long long r, int i) {
  if (i < c.nope) {
    const float v = e4m3_decode(c.codes[layer][r * c.nope + i]) *
                    e8m0_decode(c.scales[layer][r * kKvScaleSlots + i / 64]);
    return isfinite(v) ? bf16_round(v) : v;  // the rounding's carry would turn a NaN into a zero
  }
  return bf16_widen(c.rope[layer][r * c.rope_dim + (i - c.nope)]);
}

// The slot whose rows hold row `row`: the last s with q_start[s] <= row that
// is not empty. -1: none.
__device__ __forceinline__ int slot_of(const int* q_start, int n_seqs, int row) {
  int lo = 0, hi = n_seqs;  // first s with q_start[s + 1] > row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid + 1] > row) hi = mid;
    else lo = mid + 1;
  }
  return lo < n_seqs && q_start[lo] <= row ? lo : -1;
}

__device__ __forceinline__ float load_q(const PagedAttnProblem& p, long long at) {
  return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[at])
                : bf16_round(static_cast<const float*>(p.q)[at]);
}
__device__ __forceinline__ void store_out(const PagedAttnProblem& p, long long at, float v) {
  if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(p.out)[at] = __bfloat162float(__float2bfloat16_rn(v));
}

// General form: one block per (head, token), a warp per key, the running
// maximum and sum of a softmax per warp, merged at the end.
__global__ void __launch_bounds__(32 * kSimtWarps) paged_attn_simt_kernel(
    const __grid_constant__ PagedAttnProblem p) {
  const PagedState& c = p.pages;
  const int row = blockIdx.x, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = c.nope + c.rope_dim;
  __shared__ float sm_m[kSimtWarps], sm_den[kSimtWarps];
  __shared__ float sm_o[kMaxDim];
  __shared__ int sm_bad;
  const int s = slot_of(p.q_start, c.n_seqs, row);
  if (threadIdx.x == 0) sm_bad = 0;
  for (int i = threadIdx.x; i < d; i += blockDim.x) sm_o[i] = 0.f;
  __syncthreads();
  float m = -INFINITY, den = 0.f;
  float q[kLaneDims], o[kLaneDims];
#pragma unroll
  for (int u = 0; u < kLaneDims; ++u) {
    const int i = u * 32 + lane;
    q[u] = i < d ? load_q(p, row * p.q_stride + static_cast<long long>(h) * d + i) : 0.f;
    o[u] = 0.f;
  }
  if (s >= 0) {
    const int last = c.length[s] - p.q_start[s + 1] + row;
    const int first = p.window > 0 ? max(0, last - p.window + 1) : 0;
    const int* table = c.table + static_cast<size_t>(s) * c.max_pages;
    for (int t = first + warp; t <= last && t / c.page < c.max_pages; t += kSimtWarps) {
      const int page = table[t / c.page];
      if (page < 0 || page >= c.n_pages) continue;
      const long long r = static_cast<long long>(page) * c.page + t % c.page;
      float k[kLaneDims], dot = 0.f;
      bool fine = true;
#pragma unroll
      for (int u = 0; u < kLaneDims; ++u) {
        const int i = u * 32 + lane;
        k[u] = i < d ? latent_value(c, p.layer, r, i) : 0.f;
        fine = fine && isfinite(k[u]);
        dot = fmaf(q[u], k[u], dot);
      }
      if (!__all_sync(0xffffffffu, fine)) {
        if (lane == 0) sm_bad = 1;
        continue;
      }
#pragma unroll
      for (int u = 16; u > 0; u >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, u);
      const float x = dot * p.scale;
      const float mx = fmaxf(m, x);
      const float a = m == -INFINITY ? 0.f : expf(m - mx), w = expf(x - mx);
      den = den * a + w;
#pragma unroll
      for (int u = 0; u < kLaneDims; ++u) o[u] = o[u] * a + w * k[u];
      m = mx;
    }
  }
  if (lane == 0) sm_m[warp] = m;
  __syncthreads();
  float M = p.sink ? p.sink[h] : -INFINITY;
  for (int w = 0; w < kSimtWarps; ++w) M = fmaxf(M, sm_m[w]);
  const float f = m == -INFINITY ? 0.f : expf(m - M);
  if (lane == 0) sm_den[warp] = den * f;
#pragma unroll
  for (int u = 0; u < kLaneDims; ++u) o[u] *= f;
  for (int w = 0; w < kSimtWarps; ++w) {  // in warp order: the sum does not depend on timing
    if (warp == w) {
#pragma unroll
      for (int u = 0; u < kLaneDims; ++u) {
        const int i = u * 32 + lane;
        if (i < d) sm_o[i] += o[u];
      }
    }
    __syncthreads();
  }
  float total = p.sink && M != -INFINITY ? expf(p.sink[h] - M) : 0.f;
  for (int w = 0; w < kSimtWarps; ++w) total += sm_den[w];
  const bool bad = sm_bad != 0;
  const float inv = bad ? NAN : (total == 0.f ? 0.f : 1.f / total);
  const int r0 = d - p.rope_out;
  for (int i = 2 * threadIdx.x; i < d; i += 2 * blockDim.x) {
    float x0 = sm_o[i] * inv, x1 = i + 1 < d ? sm_o[i + 1] * inv : 0.f;
    if (p.rope_cos && i >= r0) {
      const long long at = static_cast<long long>(row) * (p.rope_out / 2) + (i - r0) / 2;
      const float cs = p.rope_cos[at], sn = p.rope_sin[at];
      const float y0 = x0 * cs + x1 * sn, y1 = x1 * cs - x0 * sn;
      x0 = y0;
      x1 = y1;
    }
    const long long at = row * p.out_stride + static_cast<long long>(h) * d + i;
    store_out(p, at, x0);
    if (i + 1 < d) store_out(p, at + 1, x1);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[static_cast<size_t>(row) * p.H + h] = bad ? NAN : (total == 0.f ? -INFINITY : M + logf(total));
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnProblem&) { return 0; }

cudaError_t paged_attn_forward(const PagedAttnProblem& p, void*, cudaStream_t st) {
  if (p.total <= 0) return cudaSuccess;
  if (p.pages.nope + p.pages.rope_dim > kMaxDim) return cudaErrorInvalidValue;
  paged_attn_simt_kernel<<<dim3(p.total, p.H), 32 * kSimtWarps, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dsv4
