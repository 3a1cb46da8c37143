// beam.cu - selection of beams: per prompt, the best of its beams'
// continuations,
//   total[b, t] = score[b] + x[b, t] - log sum_t' e^x[b, t']
// the lower (beam, token) first among equals, those that go on, and the slot
// that each takes.
//
// Only a beam's `cands` largest logits can be among the prompt's `cands` best,
// so the first kernel keeps, of every part of a row, that many values and the
// part's maximum and sum of exponentials: one read, the part in registers. The
// second merges a prompt's parts. Within a beam the logits alone decide, so
// nothing is rounded there; between beams the totals are compared in 64 bits
// (the sums behind them are fp32 over 32 values and 64 bits beyond).
// Which thread adds which value depends on the value's index alone, whatever
// the row's alignment, so that beams with equal rows have equal totals and tie.
#include "beam.cuh"

#include <climits>
#include <cmath>

#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPer = 32;                  // values of a thread
constexpr int kSpan = kThreads * kPer;    // of a part
constexpr int kCap = 2048;                // candidates held
using Key = unsigned long long;           // ordered value above inverted index; 0: nothing

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 -> +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ Key make_key(float x, int i) {
  return (static_cast<Key>(ordered(x)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_index(Key k) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k));
}

struct Part {
  double z;  // sum of e^(x - m)
  float m;   // maximum
};

struct Work {
  Part* part;  // [rows][parts]
  Key* key;    // [rows][parts][cands], descending, 0 behind the last
};

struct BeamArgs {
  BeamProblem p;
  int parts;
  bool wide;  // 16-byte aligned rows
  Work w;
};

template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 4) beam_parts_kernel(const BeamArgs a) {
  __shared__ Key cand[kCap];
  __shared__ float warp_m[kWarps], warp_t[kWarps];
  __shared__ double warp_z[kWarps];
  __shared__ Key best[kWarps];
  __shared__ int held;
  const BeamProblem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  constexpr int kN = kBf16 ? 8 : 4, kVecs = kPer / kN;  // values of 16 bytes
  const long long at = row * p.stride;
  const int i0 = part * kSpan;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) held = 0;
  // value k of vector u: index i0 + (u * kThreads + tid) * kN + k
  float v[kPer];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int i = i0 + (u * kThreads + tid) * kN;
    if (a.wide && i + kN <= p.vocab) {
      uint4 r;
      const void* q = kBf16 ? static_cast<const void*>(static_cast<const uint16_t*>(p.logits) + at + i)
                            : static_cast<const void*>(static_cast<const float*>(p.logits) + at + i);
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(q));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int k = 0; k < kN; ++k)
        v[u * kN + k] = !kBf16 ? __uint_as_float(w[k & 3])
                               : __uint_as_float((k & 1) ? w[k >> 1] & 0xFFFF0000u : w[k >> 1] << 16);
    } else {
#pragma unroll
      for (int k = 0; k < kN; ++k)
        v[u * kN + k] = i + k >= p.vocab ? -INFINITY
                        : kBf16 ? bf16_widen(static_cast<const uint16_t*>(p.logits)[at + i + k])
                                : static_cast<const float*>(p.logits)[at + i + k];
    }
  }
  float mine = v[0];
#pragma unroll
  for (int k = 1; k < kPer; ++k) mine = fmaxf(mine, v[k]);
  mine = fmaxf(mine, -INFINITY);  // NaN where every value is one
  // Every warp has `each` threads whose largest value reaches the each-th
  // largest of them, so each * kWarps >= cands values reach the smallest of
  // these.
  float top = warp_max(mine), kth = top, left = mine;
  for (int each = kWarps; each < p.cands; each += kWarps) {
    const unsigned who = __ballot_sync(0xffffffffu, left == kth);
    if (lane == __ffs(who) - 1) left = -INFINITY;
    kth = warp_max(left);
  }
  if (lane == 0) {
    warp_m[warp] = top;
    warp_t[warp] = kth;
  }
  __syncthreads();
  float m = warp_m[0], limit = warp_t[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    m = fmaxf(m, warp_m[w]);
    limit = fminf(limit, warp_t[w]);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float each_z = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) each_z += ex2_approx((v[k] - ref) * kLog2e);
  double z = each_z;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  if (lane == 0) warp_z[warp] = z;
  if (mine >= limit) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (v[k] >= limit && v[k] > -INFINITY) {
        const int n = atomicAdd(&held, 1);
        if (n < kCap)
          cand[n] = make_key(v[k], i0 + ((k / kN) * kThreads + tid) * kN + k % kN);
      }
  }
  __syncthreads();
  const int n = held;
  Key* out = a.w.key + static_cast<long long>(blockIdx.x) * p.cands;
  if (tid == 0) {
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += warp_z[w];
    a.w.part[blockIdx.x] = {sum, m};
  }
  if (n <= kCap) {
    // a key's place is the number of larger ones (keys differ)
    for (int i = tid; i < n; i += kThreads) {
      const Key k = cand[i];
      int rank = 0;
      for (int j = 0; j < n && rank < p.cands; ++j) rank += cand[j] > k;
      if (rank < p.cands) out[rank] = k;
    }
    for (int i = n + tid; i < p.cands; i += kThreads) out[i] = 0;
    return;
  }
  // More values reach the limit than fit (a row of equal values): one of the
  // block's best after the other.
  Key before = ~0ull;
  for (int r = 0; r < p.cands; ++r) {
    Key k = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const Key q = v[j] > -INFINITY
                        ? make_key(v[j], i0 + ((j / kN) * kThreads + tid) * kN + j % kN) : 0;
      if (q < before && q > k) k = q;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Key q = __shfl_xor_sync(0xffffffffu, k, o);
      k = q > k ? q : k;
    }
    if (lane == 0) best[warp] = k;
    __syncthreads();
    k = best[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) k = best[w] > k ? best[w] : k;
    if (tid == 0) out[r] = k;
    before = k;
    __syncthreads();
  }
}

// A candidate of the second kernel: what it is compared by, larger first, then
// its place among the prompt's continuations, smaller first. place < 0: none.
struct Cand {
  double total;
  long long place;
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  if (a.place < 0 || b.place < 0) return b.place < 0 && a.place >= 0;
  return a.total != b.total ? a.total > b.total : a.place < b.place;
}
__device__ __forceinline__ Cand shfl_xor(const Cand& c, int j) {
  return {__shfl_xor_sync(0xffffffffu, c.total, j), __shfl_xor_sync(0xffffffffu, c.place, j)};
}
// The 32 best of two descending sequences, one element a lane.
__device__ __forceinline__ Cand best_of(Cand a, Cand b) {
  const int lane = threadIdx.x & 31;
  const Cand r = shfl_xor(b, 31);  // reversed
  if (better(r, a)) a = r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const Cand o = shfl_xor(a, j);
    if (better(o, a) == ((lane & j) == 0)) a = o;
  }
  return a;
}
__device__ __forceinline__ Key best_of(Key a, Key b) {
  const int lane = threadIdx.x & 31;
  const Key r = __shfl_xor_sync(0xffffffffu, b, 31);
  if (r > a) a = r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const Key o = __shfl_xor_sync(0xffffffffu, a, j);
    if ((o > a) == ((lane & j) == 0)) a = o;
  }
  return a;
}

// The n-th (from 0) set bit's number; 32: there are fewer.
__device__ __forceinline__ int nth_bit(unsigned mask, int n) {
  for (int i = 0; i < n; ++i) mask &= mask - 1;
  return mask ? __ffs(mask) - 1 : 32;
}

__global__ void __launch_bounds__(kThreads) beam_group_kernel(const BeamArgs a) {
  __shared__ Cand list[kWarps][32];
  const BeamProblem& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  Cand mine = {0.0, -1};
  for (int b = warp; b < p.beams; b += kWarps) {
    const long long row = static_cast<long long>(g) * p.beams + b;
    const Part* part = a.w.part + row * a.parts;
    const Key* key = a.w.key + row * a.parts * p.cands;
    float m = -INFINITY;
    for (int i = lane; i < a.parts; i += 32) m = fmaxf(m, part[i].m);
    m = warp_max(m);
    double z = 0.0;
    for (int i = lane; i < a.parts; i += 32) {
      const Part q = part[i];
      // (NaN stays; a part of nothing has z 0)
      z += q.m == -INFINITY ? q.z : q.z * exp(static_cast<double>(q.m) - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    Key k = lane < p.cands ? key[lane] : 0;
    for (int i = 1; i < a.parts; ++i)
      k = best_of(k, lane < p.cands ? key[static_cast<long long>(i) * p.cands + lane] : 0);
    const double off = static_cast<double>(p.score[row]) - (m + log(z));
    Cand c = {0.0, -1};
    if (k) {
      c.total = key_value(k) + off;
      // a dead beam, or a row with a NaN or +inf, has no candidates
      if (fabs(c.total) <= 1.7e308) c.place = static_cast<long long>(b) * p.vocab + key_index(k);
    }
    mine = best_of(mine, c);
  }
  list[warp][lane] = mine;
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < min(kWarps, p.beams); ++w) mine = best_of(mine, list[w][lane]);
  const bool live = lane < p.cands && mine.place >= 0;
  const int parent = live ? static_cast<int>(mine.place / p.vocab) : -1;
  const int token = live ? static_cast<int>(mine.place - static_cast<long long>(parent) * p.vocab) : -1;
  if (lane < p.cands) {
    const long long at = static_cast<long long>(g) * p.cands + lane;
    p.parent[at] = parent;
    p.token[at] = token;
    p.total[at] = live ? static_cast<float>(mine.total) : -INFINITY;
  }
  // the best that have not ended go on
  const unsigned on = __ballot_sync(0xffffffffu, live && token != p.eos);
  const bool beam = lane < p.beams;
  const int follow = nth_bit(on, lane);
  const int mother_of = __shfl_sync(0xffffffffu, parent, follow & 31);
  const int mother = beam && follow < 32 ? mother_of : -1;
  const long long at = static_cast<long long>(g) * p.beams + lane;
  if (beam) p.next[at] = follow < 32 ? follow : -1;
  if (!p.slot) return;
  // A beam's first child stays in its slot; the others take those of the beams
  // without one, so that no slot that is copied from is overwritten.
  const unsigned same = __match_any_sync(0xffffffffu, mother);
  const bool stays = mother >= 0 && lane == __ffs(same) - 1;
  const unsigned mothers = __reduce_or_sync(0xffffffffu, mother >= 0 ? 1u << mother : 0u);
  const unsigned lost = ~mothers & (p.beams == 32 ? 0xffffffffu : (1u << p.beams) - 1);
  const unsigned moves = __ballot_sync(0xffffffffu, beam && !stays);
  if (!beam) return;
  const int home = stays ? mother : nth_bit(lost, __popc(moves & ((1u << lane) - 1)));
  const long long row = static_cast<long long>(g) * p.beams;
  p.dst[at] = p.slot[row + home];
  p.src[at] = mother >= 0 ? p.slot[row + mother] : -1;
}

int parts_of(const BeamProblem& p) { return (p.vocab + kSpan - 1) / kSpan; }

}  // namespace

size_t beam_workspace_bytes(const BeamProblem& p) {
  const size_t parts = static_cast<size_t>(p.groups) * p.beams * parts_of(p);
  return parts * (sizeof(Part) + sizeof(Key) * p.cands);
}

cudaError_t beam_select(const BeamProblem& p, void* ws, cudaStream_t st) {
  if (p.groups <= 0) return cudaSuccess;
  BeamArgs a;
  a.p = p;
  a.parts = parts_of(p);
  const int size = p.bf16 ? 2 : 4;
  a.wide = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.stride * size % 16 == 0;
  const long long blocks = static_cast<long long>(p.groups) * p.beams * a.parts;
  if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  a.w.key = static_cast<Key*>(ws);
  a.w.part = reinterpret_cast<Part*>(a.w.key + blocks * p.cands);
  cudaError_t e = launch_pdl(p.bf16 ? beam_parts_kernel<true> : beam_parts_kernel<false>,
                             dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(beam_group_kernel, dim3(p.groups), dim3(kThreads), 0, st, a);
}

}  // namespace dsv4
