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
//
// One pass over the row: every thread keeps a running maximum and the two
// sums relative to it. A candidate for the top is one 64-bit key, the value
// in an order-preserving form above the inverted index, so that the larger
// key is the better one, ties included. The block keeps the k best so far;
// what comes later has a higher index and therefore has to exceed the k-th
// strictly, which after the first step few values do (ties of any number
// never do). Rows are cut over a cluster where there are too few of them to
// fill the GPU; the parts meet in the first CTA's shared memory.
#include "logprob.cuh"

#include <climits>
#include <cmath>
#include <cuda_bf16.h>

#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRound = 4 * kThreads; // candidates of four values a thread
constexpr int kCap = 2 * kRound;     // candidates held
// More candidates than kThin are thinned out to the best 32, looked at every
// kWindow steps: a tighter limit keeps later values out, a look costs two
// barriers. (2048 rows of 129280 fp32 values, top 8: 211 us; 226 with 256, 213
// with windows of 4.)
constexpr int kThin = 64;
constexpr int kWindow = 8;
constexpr int kTop = kMaxTopAlternatives;
constexpr int kMaxCluster = 16;
constexpr float kLn2 = 0.69314718055994531f;
using Key = unsigned long long;      // 0: nothing

__device__ __forceinline__ Key make_key(float x, int i) {
  uint32_t u = __float_as_uint(x + 0.0f);  // -0 -> +0
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<Key>(u) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_index(Key k) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k));
}

// One key per lane, descending over the lanes.
__device__ __forceinline__ Key swap_step(Key k, int j, bool keep_max) {
  const Key o = __shfl_xor_sync(0xffffffffu, k, j);
  return keep_max ? (o > k ? o : k) : (o < k ? o : k);
}
__device__ __forceinline__ Key merge_sorted(Key k) {  // a bitonic sequence to descending
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) k = swap_step(k, j, (lane & j) == 0);
  return k;
}
__device__ __forceinline__ Key sort_lanes(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int j = n >> 1; j > 0; j >>= 1) k = swap_step(k, j, ((lane & j) == 0) == ((lane & n) == 0));
  return k;
}
// The 32 best of two descending sequences.
__device__ __forceinline__ Key best_of(Key a, Key b) {
  const Key r = __shfl_xor_sync(0xffffffffu, b, 31);  // reversed
  return merge_sorted(a > r ? a : r);
}

struct alignas(16) Shared {
  Key cand[kCap];
  Key list[kWarps][kTop];
  float4 part_sums[kMaxCluster];  // the parts of a cluster, in its first CTA
  Key part[kMaxCluster][kTop];
  float m[kWarps], z[kWarps], s[kWarps];
  int above[kWarps];
  int n;                       // candidates held
  Key limit;                   // the k-th best so far, 0: fewer than k
};

// Warp 0: the best of the first `used` warps' sequences, by pairs, then pairs
// of pairs. Whole block.
__device__ Key best_of_warps(Shared& sh, Key best, int used) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int s = 1; s < used; s <<= 1) {
    if (warp & s) sh.list[warp][lane] = best;
    __syncthreads();
    if ((warp & (2 * s - 1)) == 0 && warp + s < used) best = best_of(best, sh.list[warp + s][lane]);
  }
  return best;
}

// The best 32 of the n candidates, descending, to cand[0 .. 31]; the k-th is
// the new limit. Whole block.
__device__ void compact(Shared& sh, int k) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __syncthreads();
  const int n = sh.n;
  if (n <= kThreads) {
    // a thread a key: its place is the number of larger ones (keys differ).
    // Shorter than the sort below where there are no more keys than threads (1
    // row: 10.3 us, 11.6 to 12.0 with the sort alone).
    const Key mine = tid < n ? sh.cand[tid] : 0;
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) rank += sh.cand[i] > mine;
    __syncthreads();
    if (tid < n && rank < kTop) {
      sh.cand[rank] = mine;
      if (rank == k - 1) sh.limit = mine;
    }
    if (tid == 0) sh.n = min(n, kTop);
    __syncthreads();
    return;
  }
  Key best = 0;
  for (int base = warp * 32; base < n; base += kThreads) {
    const int i = base + lane;
    const Key next = sort_lanes(i < n ? sh.cand[i] : 0);
    best = base == warp * 32 ? next : best_of(best, next);
  }
  best = best_of_warps(sh, best, kWarps);
  if (warp == 0) {
    sh.cand[lane] = best;
    const Key kth = __shfl_sync(0xffffffffu, best, k - 1);
    if (lane == 0) {
      sh.limit = kth;
      sh.n = kTop;
    }
  }
  __syncthreads();
}

// 1 where a > b (a >= b), else 0: counts of up to 2^24 in a register
__device__ __forceinline__ float gt1(float a, float b) {
  float r;
  asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ge1(float a, float b) {
  float r;
  asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Running sums in natural units relative to m: sum e^(x - m) and
// sum e^(x - m) log2 e (x - m). (Plain fp32 arithmetic: with the packed kind
// more instructions went into pairing registers than it saved.)
struct Sums {
  float m, z, s;
};

__device__ __forceinline__ void raise_max(Sums& t, float bm) {
  if (bm > t.m) {
    if (t.m != -INFINITY) {  // (nothing but zeros, or NaN, so far)
      const float d = fmaxf((t.m - bm) * kLog2e, -1e4f);  // finite: it meets a zero
      const float f = ex2_approx(d);
      t.s = f * fmaf(d, t.z, t.s);
      t.z = f * t.z;
    }
    t.m = bm;
  }
}

__device__ __forceinline__ void add_value(Sums& t, float ref, float x) {
  // x - ref first: exact where it matters, whatever the size of the logits
  const float d = (x - ref) * kLog2e, e = ex2_approx(d);
  t.z += e;
  t.s = fmaf(e, fmaxf(d, -256.f), t.s);  // e = 0 below 2^-126: a masked value adds 0
}

// 16 bytes that are read once.
__device__ __forceinline__ uint4 ldg_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool kBf16>
struct Vec {
  static constexpr int kN = kBf16 ? 8 : 4;  // values of 16 bytes
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t w = kBf16 ? (i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w)
                             : (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
    if (!kBf16) return __uint_as_float(w);
    return __uint_as_float((i & 1) ? w & 0xFFFF0000u : w << 16);
  }
  // 16 bytes that hold -inf everywhere
  static __device__ __forceinline__ uint4 none() {
    const uint32_t w = kBf16 ? 0xFF80FF80u : 0xFF800000u;
    return make_uint4(w, w, w, w);
  }
};

// kStep: values a thread reads per step; kBlocks: blocks of an SM.
//
// 2048 rows of 129280 fp32 values, top 8: 211 us, 5.0 TB/s of the 6.5 that a
// copy reaches. Instructions bound it: an exponential, two FMAs, compares, a
// share of a maximum and of the bookkeeping are 20 a value, and 77% of the
// issue slots are taken (600 rows, start and end included; memory 46%, in BF16
// rows, whose bytes are half, 25% at 95% of the time). 256 threads, four blocks
// an SM: 9% less than with two of 512. 1 row: 10.3 us, a chain of one read, the
// choice among 32 values a thread, the cluster's meeting and the final merge.
template <bool kBf16, int kStep, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) logprob_kernel(const LogprobProblem p, int parts) {
  using V = Vec<kBf16>;
  constexpr int kN = V::kN, kVecs = kStep / kN;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (parts > 1) cluster_arrive();
  const int row = blockIdx.x / parts, part = blockIdx.x % parts;
  constexpr int kSize = kBf16 ? 2 : 4;
  const uint8_t* x_row = static_cast<const uint8_t*>(p.logits) + row * p.stride * kSize;
  auto value_at = [&](int i) {
    return kBf16 ? bf16_widen(reinterpret_cast<const uint16_t*>(x_row)[i])
                 : reinterpret_cast<const float*>(x_row)[i];
  };
  // values before the first 16-byte boundary, whole vectors, values behind the last
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x_row) & 15);
  const int head = min(p.vocab, off ? (16 - off) / kSize : 0);
  const int vecs = (p.vocab - head) / kN;
  const int tail0 = head + vecs * kN;
  const int v0 = static_cast<int>(static_cast<long long>(vecs) * part / parts);
  const int v1 = static_cast<int>(static_cast<long long>(vecs) * (part + 1) / parts);
  const uint4* src = reinterpret_cast<const uint4*>(x_row + head * kSize);

  if (tid == 0) {
    sh.n = 0;
    sh.limit = 0;
  }
  Sums sum = {-INFINITY, 0.f, 0.f}, odd = sum;
  float above = 0.f;
  uint4 cur[kVecs], buf[kVecs];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = base + u * kThreads + tid;
      buf[u] = v < v1 ? ldg_stream(src + v) : V::none();
    }
  };
  constexpr int kStride = kVecs * kThreads;  // vectors of a step
  // A value of this thread's step at `base` joins the candidates if its key
  // exceeds the limit. Past the capacity they are only counted.
  auto join = [&](int base, int u, int i, Key limit, float lv) {
    const float x = V::get(cur[u], i);
    if (x >= lv || limit == 0) {
      const int v = base + u * kThreads + tid;
      const Key k = make_key(x, head + v * kN + i);
      if (v < v1 && x == x && k > limit) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kCap) sh.cand[at] = k;
      }
    }
  };
  load(v0);
  const int t = p.tokens[row];
  const bool asked = t >= 0 && t < p.vocab;
  const float xt = asked ? value_at(t) : NAN;  // NaN: nothing is above it
  __syncthreads();
  bool first = true;
  int held = 0;  // candidates from before the window
  for (int w0 = v0; w0 < v1; w0 += kWindow * kStride) {
    const int w1 = min(v1, w0 + kWindow * kStride);
    const int before = held;
    for (int base = w0; base < w1; base += kStride) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) cur[u] = buf[u];
      if (base + kStride < v1) load(base + kStride);
      float vm[kVecs];  // the best of each vector
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        vm[u] = fmaxf(V::get(cur[u], 0), V::get(cur[u], 1));
#pragma unroll
        for (int i = 2; i < kN; i += 2) vm[u] = max3(vm[u], V::get(cur[u], i), V::get(cur[u], i + 1));
      }
      float bm = vm[0];
#pragma unroll
      for (int u = 1; u < kVecs; ++u) bm = fmaxf(bm, vm[u]);
      bm = fmaxf(bm, -INFINITY);  // NaN where every value is one
      raise_max(odd, bm);  // (the two chains of sums have one maximum)
      raise_max(sum, bm);
      const float ref = sum.m == -INFINITY ? 0.f : sum.m;
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          Sums& q = (i & 1) ? odd : sum;
          add_value(q, ref, V::get(cur[u], i));
        }
      // Values above the token's; equal ones count where they come before it.
      // Most steps lie on one side of it.
      const int i_lo = head + base * kN, i_hi = i_lo + kStride * kN;
      if (base + kStride <= v1 && i_hi <= t) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
          for (int i = 0; i < kN; ++i) above += ge1(V::get(cur[u], i), xt);
      } else {
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
          for (int i = 0; i < kN; ++i) above += gt1(V::get(cur[u], i), xt);
        if (i_lo < t) {
#pragma unroll
          for (int u = 0; u < kVecs; ++u) {
            const int v = base + u * kThreads + tid, i0 = head + v * kN;
            if (v < v1 && i0 < t) {
#pragma unroll
              for (int i = 0; i < kN; ++i)
                if (i0 + i < t && V::get(cur[u], i) == xt) above += 1.f;
            }
          }
        }
      }
      if (p.top > 0) {
        if (first) {
          // Every warp has `each` threads whose best value reaches the each-th
          // best of them, so each * kWarps >= k values reach the smallest of
          // these.
          float mine = bm, kth = warp_max(mine);
          for (int each = kWarps; each < p.top; each += kWarps) {
            const unsigned at_top = __ballot_sync(0xffffffffu, mine == kth);
            if (lane == __ffs(at_top) - 1) mine = -INFINITY;
            kth = warp_max(mine);
          }
          if (lane == 0) sh.m[warp] = kth;
          __syncthreads();
          kth = sh.m[lane % kWarps];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            kth = fminf(kth, __shfl_xor_sync(0xffffffffu, kth, o));
          // just below every key of that value
          if (kth > -INFINITY) {
            if (tid == 0) sh.limit = make_key(kth, -1);
          } else {
            // A warp without so many values (a short row, a masked range): the
            // k-th best of all threads' best, if there are k (1404 rows of 1260
            // BF16 values, top 12: 25 us, 43 where every value was let in). If
            // not, most values are -inf, of which the first k alone can be among
            // the best: none behind the first 32 vectors, should k of their
            // values not be NaN (48 rows of 129280, 999 of 1000 masked: 24
            // us, 48 where every -inf was let in).
            Key best = sort_lanes(bm > -INFINITY ? make_key(bm, tid) : 0);
            best = best_of_warps(sh, best, kWarps);
            if (warp == 0) {
              const Key at = __shfl_sync(0xffffffffu, best, p.top - 1);
              int values = 0;
#pragma unroll
              for (int i = 0; i < kN; ++i) values += V::get(cur[0], i) == V::get(cur[0], i);
              values = __reduce_add_sync(0xffffffffu, values);
              if (lane == 0) {
                if (at) sh.limit = make_key(key_value(at), -1);
                else if (v1 - v0 >= 32 && values >= p.top)
                  sh.limit = make_key(-INFINITY, head + (v0 + 32) * kN);
              }
            }
          }
          __syncthreads();
        }
        const Key limit = *static_cast<volatile Key*>(&sh.limit);  // an old one only lets more in
        const float lv = limit ? key_value(limit) : -INFINITY;
        // (equal values can count in the first step alone: later ones come
        // behind)
        if (limit == 0 || (first ? bm >= lv : bm > lv)) {
#pragma unroll
          for (int u = 0; u < kVecs; ++u)
            if (limit == 0 || vm[u] >= lv) {
#pragma unroll
              for (int i = 0; i < kN; ++i) join(base, u, i, limit, lv);
            }
        }
        if (first) {
          __syncthreads();
          const int n = sh.n;
          __syncthreads();  // nobody adds to it before all have read it
          // (worth it where enough is still to come)
          if (n > p.top && n <= kCap && v1 - v0 > 2 * kStride) compact(sh, p.top);
          first = false;
        }
      }
    }
    if (p.top > 0) {
      __syncthreads();
      const int n = sh.n;
      __syncthreads();
      held = n;
      if (n > kThin) held = kTop;
      if (n > kCap) {
        // more than fit (values in ascending order, say): the window again,
        // four values a thread at a time, thinned out in between (the limit
        // may be a value of this window, which has to come in again)
        if (tid == 0) {
          sh.n = before;
          if (sh.limit) sh.limit -= 1;
        }
        __syncthreads();
        for (int base = w0; base < w1; base += kStride) {
#pragma unroll
          for (int u = 0; u < kVecs; ++u) {
            const int v = base + u * kThreads + tid;
            cur[u] = v < v1 ? ldg_stream(src + v) : V::none();
          }
#pragma unroll
          for (int u = 0; u < kVecs; ++u)
#pragma unroll
            for (int i = 0; i < kN; ++i) {
              const Key limit = sh.limit;
              join(base, u, i, limit, limit ? key_value(limit) : -INFINITY);
              if (i % 4 == 3) {
                __syncthreads();
                const int m = sh.n;
                __syncthreads();
                if (m > kCap - kRound) compact(sh, p.top);
              }
            }
        }
        compact(sh, p.top);
      } else if (n > kThin) {
        compact(sh, p.top);
      }
    }
  }
  // the values outside whole vectors: at most one a thread
  {
    const int n_head = part == 0 ? head : 0, n_tail = part == parts - 1 ? p.vocab - tail0 : 0;
    const int i = tid < n_head ? tid : tid - n_head < n_tail ? tail0 + tid - n_head : -1;
    if (n_head + n_tail > 0) {
      const float x = i >= 0 ? value_at(i) : -INFINITY;
      if (i >= 0) {
        raise_max(odd, x);
        raise_max(sum, x);
        add_value(sum, sum.m == -INFINITY ? 0.f : sum.m, x);
        if (x > xt || (x == xt && i < t)) above += 1.f;
        if (p.top > 0 && x == x) sh.cand[atomicAdd(&sh.n, 1)] = make_key(x, i);
      }
    }
  }
  if (p.top > 0) compact(sh, p.top);  // sorted, whatever their number

  int n_above = static_cast<int>(above);
  sum.z += odd.z;
  sum.s += odd.s;
  auto warp_sums = [&] {
    raise_max(sum, warp_max(sum.m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o);
      sum.s += __shfl_xor_sync(0xffffffffu, sum.s, o);
    }
    n_above = __reduce_add_sync(0xffffffffu, n_above);
  };
  warp_sums();
  if (lane == 0) {
    sh.m[warp] = sum.m;
    sh.z[warp] = sum.z;
    sh.s[warp] = sum.s;
    sh.above[warp] = n_above;
  }
  __syncthreads();
  Key best = 0;
  if (warp == 0) {
    const bool in = lane < kWarps;
    sum = {in ? sh.m[lane] : -INFINITY, in ? sh.z[lane] : 0.f, in ? sh.s[lane] : 0.f};
    n_above = in ? sh.above[lane] : 0;
    warp_sums();
    if (p.top > 0) best = lane < sh.n ? sh.cand[lane] : 0;
  }
  if (parts > 1) {
    static_assert(kMaxCluster <= 2 * kWarps && kMaxCluster <= 32, "two parts a warp");
    // every part writes into the first CTA's shared memory, which is there
    // since all have arrived at the barrier of the start
    cluster_wait();
    if (warp == 0) {
      auto remote = [&](const void* q) {
        uint32_t a;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(q)));
        return a;
      };
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&sh.part[part][lane])), "l"(best)
                   : "memory");
      if (lane == 0)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                         remote(&sh.part_sums[part])),
                     "f"(sum.m), "f"(sum.z), "f"(sum.s), "f"(__int_as_float(n_above))
                     : "memory");
    }
    cluster_arrive();
    if (part != 0) return;
    cluster_wait();
    if (p.top > 0) {
      best = warp < parts ? sh.part[warp][lane] : 0;
      if (warp + kWarps < parts) best = best_of(best, sh.part[warp + kWarps][lane]);
      best = best_of_warps(sh, best, min(parts, kWarps));
    }
    if (warp == 0) {
      const float4 q = sh.part_sums[lane % parts];
      const bool in = lane < parts;
      sum = {in ? q.x : -INFINITY, in ? q.y : 0.f, in ? q.z : 0.f};
      n_above = in ? __float_as_int(q.w) : 0;
      warp_sums();
    }
  }
  if (part != 0 || warp != 0) return;
  const float z = sum.z, ref = sum.m == -INFINITY ? 0.f : sum.m;
  const bool undefined = z != z || sum.m == INFINITY;
  const float lz = sum.m == -INFINITY ? 0.f : logf(z);
  if (lane == 0) {
    p.logprob[row] = !asked ? 0.f : undefined ? NAN : xt - ref - lz;
    if (p.entropy)
      p.entropy[row] =
          undefined ? NAN : sum.m == -INFINITY ? 0.f : fmaxf(lz - kLn2 * (sum.s / z), 0.f);
    if (p.rank) p.rank[row] = asked ? n_above : -1;
  }
  if (lane < p.top) {
    const long long at = static_cast<long long>(row) * p.top + lane;
    p.top_id[at] = best ? key_index(best) : -1;
    p.top_logprob[at] = !best || undefined ? NAN : key_value(best) - ref - lz;
  }
}

}  // namespace

cudaError_t token_logprobs(const LogprobProblem& p, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  // Few rows: each is cut over a cluster so that a thread's 32 values are all
  // it reads, and the k best are picked once (1 row of 129280: 10.3 us where
  // the kernel of many rows takes 14.3). More rows than that leave room for: steps of
  // 16 values, four blocks to an SM, rows cut while SMs idle (48 rows: 16.4 us,
  // 32 uncut).
  constexpr int kShort = 32, kLong = 16;
  int parts = 1;
  while (parts < kMaxCluster && p.vocab > parts * kThreads * kShort) parts *= 2;
  const bool few = static_cast<long long>(p.rows) * parts <= 2 * sms;
  if (!few) {
    parts = 1;
    while (parts < 8 && static_cast<long long>(p.rows) * parts * 2 <= 4 * sms &&
           p.vocab / (parts * 2) >= kThreads * kLong / 2)
      parts *= 2;
  }
  if (static_cast<long long>(p.rows) * parts > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  auto kernel = few ? (p.bf16 ? logprob_kernel<true, kShort, 2> : logprob_kernel<false, kShort, 2>)
                    : (p.bf16 ? logprob_kernel<true, kLong, 4> : logprob_kernel<false, kLong, 4>);
  const void* fn = reinterpret_cast<const void*>(kernel);
  e = set_max_dynamic_smem(fn, static_cast<int>(sizeof(Shared)));
  if (e == cudaSuccess && parts > 8)  // more than every device has to take
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * parts);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p, parts);
}

}  // namespace dsv4
