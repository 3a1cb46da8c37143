// beam.cu - selection of beams: per prompt, the best of its beams'
// continuations,
//   total[b, t] = score[b] + x[b, t] - log sum_t' e^x[b, t']
// the lower (beam, token) first among equals, those that go on, and the slot
// that each takes.
//
// Only a beam's `cands` largest logits can be among the prompt's `cands` best,
// so a block keeps, of every part of a row, that many values and the part's
// maximum and sum of exponentials, in one read. The parts of a prompt are dealt
// out over a cluster of blocks, whose first one merges them out of the others'
// shared memory. Within a beam the logits alone decide, so nothing is rounded
// there; between beams the totals are compared in 64 bits (the sums behind them
// are fp32 over a step's values of a thread and 64 bits beyond: the log of one errs
// by less than 2^-17, and totals of two beams that are nearer may change places).
// Which thread adds which value depends on the value's index alone, whatever
// the row's alignment, so that beams with equal rows have equal totals and tie.
#include "beam.cuh"

#include <climits>
#include <cmath>

#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

// Many rows: 256 threads, four blocks an SM. Few prompts, whose clusters do not
// fill the GPU: 512 threads, a block an SM, and more of a row on its way at once.
template <bool kFew>
constexpr int kThreads = kFew ? 512 : 256;
template <bool kFew>
constexpr int kBlocks = kFew ? 1 : 4;
constexpr int kCap = 512;                 // candidates held
// Candidates beyond the best are thinned out once there are this many more.
constexpr int kThin = 48;
constexpr int kMaxParts = 64;             // of a row
constexpr int kJobs = 512;                // threads with candidates, between two looks
constexpr int kMaxWarps = 16;
using Key = unsigned long long;           // ordered value above inverted index; 0: nothing

constexpr double kLn2 = 0.69314718055994530942;
constexpr double kLog2e64 = 1.4426950408889634074;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__constant__ double kReciprocal[12] = {0.0, 1.0, 1.0 / 2, 1.0 / 3, 1.0 / 4, 1.0 / 5,
                                        1.0 / 6, 1.0 / 7, 1.0 / 8, 1.0 / 9, 1.0 / 10, 1.0 / 11};
// e^x for x <= 0 to 1e-13 of itself (0 below 2^-1000), as 2^(x log2 e): Taylor's
// series around the nearest whole number. One copy of it, since it is seldom run.
__device__ __noinline__ double exp_down(double x) {
  x *= kLog2e64;
  if (!(x > -1000.0)) return x == x ? 0.0 : x;
  const double n = rint(x), t = (x - n) * kLn2;
  double r = 1.0;
#pragma unroll
  for (int k = 11; k > 0; --k) r = fma(r * t, kReciprocal[k], 1.0);
  return r * __hiloint2double((1023 + static_cast<int>(n)) << 20, 0);
}

// Values of a thread in a step.
template <bool kBf16, bool kFew>
constexpr int kPer = kBf16 || kFew ? 32 : 16;

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

// The next smaller value of a finite one (or of +inf).
__device__ __forceinline__ float below(float x) {
  const uint32_t u = ordered(x) - (x == 0.f ? 2 : 1);  // (-0 is not below 0)
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}

struct Part {
  double z;  // sum of e^(x - m)
  float m;   // -inf: of nothing
};

struct BeamArgs {
  BeamProblem p;
  int parts, steps;  // of a row; steps of a part
  int blocks;        // of a prompt: part u of its beams * parts is block u % blocks's
  bool wide;         // 16-byte aligned rows
};

template <bool kBf16, bool kFew>
struct Values {
  static constexpr int kN = kBf16 ? 8 : 4, kVecs = kPer<kBf16, kFew> / kN;  // values of 16 bytes
  uint4 v[kVecs];
  __device__ __forceinline__ float get(int k) const {
    const uint4& r = v[k / kN];
    const int i = k % kN, w = kBf16 ? i / 2 : i;
    const uint32_t u = w == 0 ? r.x : w == 1 ? r.y : w == 2 ? r.z : r.w;
    if (!kBf16) return __uint_as_float(u);
    return __uint_as_float((i & 1) ? u & 0xFFFF0000u : u << 16);
  }
  // value k of the step at i0: index i0 + (k / kN * kThreads + tid) * kN + k % kN
  static __device__ __forceinline__ int index(int i0, int k) {
    return i0 + ((k / kN) * kThreads<kFew> + static_cast<int>(threadIdx.x)) * kN + k % kN;
  }
  // Rows off the 16-byte boundary, by their stride or the first one's address, are
  // read value by value (512 BF16 rows of 50,257: 47 us, 41 where they lie 50,264
  // apart).
  __device__ __forceinline__ void load(const void* row, int i0, int vocab, bool wide) {
    if (wide && i0 + kThreads<kFew> * kPer<kBf16, kFew> <= vocab) {
      const char* q = static_cast<const char*>(row) + static_cast<size_t>(index(i0, 0)) * (kBf16 ? 2 : 4);
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w)
                     : "l"(q + u * kThreads<kFew> * 16));
      return;
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int i = index(i0, u * kN);
      const uint32_t none = kBf16 ? 0xFF80FF80u : 0xFF800000u;  // -inf
      v[u] = make_uint4(none, none, none, none);
      if (wide && i + kN <= vocab) {
        const void* q = static_cast<const char*>(row) + static_cast<size_t>(i) * (kBf16 ? 2 : 4);
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w) : "l"(q));
      } else if (i < vocab) {
        uint32_t w[4] = {none, none, none, none};
#pragma unroll
        for (int k = 0; k < kN; ++k)
          if (i + k < vocab) {
            if (!kBf16) {
              w[k & 3] = static_cast<const uint32_t*>(row)[i + k];
            } else {
              const uint32_t h = static_cast<const uint16_t*>(row)[i + k];
              w[k / 2] = (k & 1) ? (w[k / 2] & 0xFFFFu) | (h << 16) : (w[k / 2] & 0xFFFF0000u) | h;
            }
          }
        v[u] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

struct Held {
  Key cand[2][kCap];
  Key best[kMaxWarps];
  double z[kMaxWarps];
  float m[kMaxWarps], t[kMaxWarps];
  uint32_t job[kJobs];         // step and thread
  int n, jobs;
};

// The best `keep` of cand[from][0 .. n), descending, to the other list; a key's
// place is the number of larger ones (keys differ). Whole block; n is the same
// for all.
__device__ __forceinline__ void thin(Held& h, int from, int n, int keep) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const Key k = h.cand[from][i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += h.cand[from][j] > k;
    if (rank < keep) h.cand[from ^ 1][rank] = k;
  }
  if (threadIdx.x == 0) h.n = min(n, keep);
  __syncthreads();
}

// Part `part` of row `row`: its best `cands` values, descending (0 behind the
// last), its maximum and sum. Whole block.
template <bool kBf16, bool kFew>
__device__ __forceinline__ void take_part(Held& h, const BeamArgs& a, long long row, int part,
                                          Part* out, Key* keys) {
  constexpr int kEach = kPer<kBf16, kFew>, kTids = kThreads<kFew>, kSpan = kTids * kEach;
  constexpr int kWarps = kTids / 32, kTidBits = kFew ? 9 : 8;
  const BeamProblem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const void* x = static_cast<const char*>(p.logits) + row * p.stride * (kBf16 ? 2 : 4);
  int i0 = part * a.steps * kSpan;
  const int i1 = min(p.vocab, i0 + a.steps * kSpan);
  Values<kBf16, kFew> next;
  next.load(x, i0, i1, a.wide);
  __syncthreads();  // the part before has been written down
  if (tid == 0) h.n = h.jobs = 0;
  // The sum is of e^(v - ref): ref is a maximum of some values of this thread, moved
  // when one exceeds it by more than 8 (some thread of a warp has a new maximum at
  // every step). The difference is taken before it is scaled: v log2 e - ref log2 e
  // keeps the rounding of its second product, 2^18 where a row's masked values
  // are -1e9, and nothing is left of a sum that is moved by such powers.
  float ref = -INFINITY, base = 0.f;  // base: ref, or 0 before there is one
  float above = -INFINITY;  // candidates exceed it; -inf never is one
  double z = 0.0;
  const int part_i0 = i0;
  int list = 0, kept = 0, w0 = i0, step = 0;
  for (; i0 < i1; i0 += kSpan, ++step) {
    float v[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) v[k] = next.get(k);
    if (i0 + kSpan < i1) next.load(x, i0 + kSpan, i1, a.wide);
    float top = fmaxf(v[0], -INFINITY);  // (stays so where every value is NaN)
#pragma unroll
    for (int k = 1; k + 1 < kEach; k += 2) top = max3(top, v[k], v[k + 1]);
    top = fmaxf(top, v[kEach - 1]);
    if (top > ref + 8.f) {
      if (ref != -INFINITY) z *= exp_down(static_cast<double>(ref) - top);
      ref = base = top;
    }
    float z0 = 0.f, z1 = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; k += 2) {
      z0 += ex2_approx((v[k] - base) * kLog2e);
      z1 += ex2_approx((v[k + 1] - base) * kLog2e);
    }
    z += z0 + z1;
    if (step == 0) {
      // Every warp has `each` threads whose largest value reaches the each-th
      // largest of them, so each * kWarps >= cands values reach the smallest
      // of these.
      float kth = warp_max(top), left = top;
      for (int each = kWarps; each < p.cands; each += kWarps) {
        const unsigned who = __ballot_sync(0xffffffffu, left == kth);
        if (lane == __ffs(who) - 1) left = -INFINITY;
        kth = warp_max(left);
      }
      if (lane == 0) h.t[warp] = kth;
      __syncthreads();
      float limit = h.t[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) limit = fminf(limit, h.t[w]);
      above = limit > -INFINITY ? below(limit) : limit;
    }
    // A thread with a candidate only says so: what runs seldom costs more in
    // instruction fetches than it does (a loop over the values here took 1,000
    // clocks each time that one was found).
    if (top > above) {
      const int at = atomicAdd(&h.jobs, 1);
      if (at < kJobs) h.job[at] = static_cast<uint32_t>(step) << kTidBits | tid;
    }
    // looked at after one step, two, four, eight and so on, as the limit's next
    // tightening takes twice the values (of two steps both at once)
    if (i0 + kSpan < i1 && i0 + 2 * kSpan >= i1 && step == 0) continue;
    if ((step & (step + 1)) != 0 && i0 + kSpan < i1) continue;
    __syncthreads();
    const int jobs = h.jobs;
    if (jobs <= kJobs) {
      // a warp a thread's values of a step, read again, four threads' at a time
      constexpr int kN = Values<kBf16, kFew>::kN, kAtOnce = 4;
      const int in_step = (lane / kN) * kTids * kN + lane % kN;
#pragma unroll 1
      for (int j = warp; j < jobs; j += kAtOnce * kWarps) {
        float y[kAtOnce];
        int i[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const uint32_t job = j + q * kWarps < jobs ? h.job[j + q * kWarps] : 0;
          i[q] = part_i0 + static_cast<int>(job >> kTidBits) * kSpan + in_step +
                 static_cast<int>(job & (kTids - 1)) * kN;
          y[q] = -INFINITY;
          if (j + q * kWarps < jobs && lane < kEach && i[q] < i1)
            y[q] = kBf16 ? bf16_widen(static_cast<const uint16_t*>(x)[i[q]])
                         : static_cast<const float*>(x)[i[q]];
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
          if (y[q] > above) {
            const int at = atomicAdd(&h.n, 1);
            if (at < kCap) h.cand[list][at] = make_key(y[q], i[q]);
          }
      }
    }
    __syncthreads();
    const int n = jobs <= kJobs ? h.n : kCap + 1;
    __syncthreads();  // nobody adds to either before all have read them
    if (tid == 0) h.jobs = 0;
    if (n > kCap) {
      // more values exceed the limit than fit (equal ones, or ascending): the
      // block's best, one after the other, of the values since the last look,
      // read again, and those kept
      Key before = ~0ull;
#pragma unroll 1
      for (int r = 0; r < p.cands; ++r) {
        Key k = tid < kept ? h.cand[list][tid] : 0;
        if (k >= before) k = 0;
#pragma unroll 1
        for (int i = w0 + tid; i < min(i1, i0 + kSpan); i += kTids) {
          const float y = kBf16 ? bf16_widen(static_cast<const uint16_t*>(x)[i])
                                : static_cast<const float*>(x)[i];
          const Key q = y > -INFINITY ? make_key(y, i) : 0;
          if (q < before && q > k) k = q;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Key q = __shfl_xor_sync(0xffffffffu, k, o);
          k = q > k ? q : k;
        }
        if (lane == 0) h.best[warp] = k;
        __syncthreads();
        k = h.best[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) k = h.best[w] > k ? h.best[w] : k;
        if (tid == 0) h.cand[list ^ 1][r] = k;
        before = k;
        __syncthreads();
      }
      list ^= 1;
      kept = p.cands;  // (at least so many: n > kCap)
      if (tid == 0) h.n = kept;
      above = key_value(h.cand[list][p.cands - 1]);
      __syncthreads();
    } else if (n > p.cands + (step == 0 ? 0 : kThin)) {  // (the first limit is loose)
      thin(h, list, n, p.cands);
      list ^= 1;
      kept = p.cands;
      above = key_value(h.cand[list][p.cands - 1]);
    } else {
      kept = n;
      __syncthreads();  // jobs
    }
    w0 = i0 + kSpan;
  }
  thin(h, list, kept, p.cands);  // sorted
  list ^= 1;
  // the block's sum, relative to its largest ref (NaN stays)
  const float top = warp_max(ref);
  if (ref != -INFINITY) z *= exp_down(static_cast<double>(ref) - top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  if (lane == 0) {
    h.m[warp] = top;
    h.z[warp] = z;
  }
  __syncthreads();
  if (warp == 0) {
    const bool in = lane < kWarps;
    const float one = in ? h.m[lane] : -INFINITY, all = warp_max(one);
    z = in ? h.z[lane] : 0.0;
    if (one != -INFINITY) z *= exp_down(static_cast<double>(one) - all);
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) *out = {z, all};
    if (lane < p.cands) keys[lane] = lane < h.n ? h.cand[list][lane] : 0;
  }
}

// A candidate of the merge: what it is compared by, larger first, then its place
// (beam, then token), smaller first. place < 0: none.
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

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 8 bytes of block `rank`'s shared memory, at the place that q has here.
__device__ __forceinline__ unsigned long long ld_block(const void* q, int rank) {
  uint32_t at;
  unsigned long long v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(q)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}

struct Merge {
  Cand list[kMaxWarps][32];
  double top[kMaxBeams], rest[kMaxBeams];
};

// One prompt's parts: the block that merges them.
template <bool kFew>
__device__ __forceinline__ void merge_group(Merge& sh, const BeamArgs& a, int g, const Part* part,
                                            const Key* keys) {
  constexpr int kWarps = kThreads<kFew> / 32;
  const BeamProblem& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto key_of = [&](int u) { return ld_block(keys + (u / a.blocks) * p.cands + lane, u % a.blocks); };
  auto part_of = [&](int u) {
    const Part* q = part + u / a.blocks;
    const int rank = u % a.blocks;
    return Part{__longlong_as_double(ld_block(&q->z, rank)),
                __uint_as_float(static_cast<uint32_t>(ld_block(&q->m, rank)))};
  };
  // Eight parts of a row at a time: their lists are asked for together and
  // merged by pairs, the first ones while the rows' sums are on their way.
  constexpr int kTake = 8;
  const int takes = (a.parts + kTake - 1) / kTake, units = p.beams * takes;
  Key k[kTake];
  auto load_keys = [&](int u) {
    const int b = u / takes, first = (u - b * takes) * kTake;
#pragma unroll
    for (int i = 0; i < kTake; ++i)
      k[i] = first + i < a.parts && lane < p.cands ? key_of(b * a.parts + first + i) : 0;
  };
  auto best_key = [&](int u) {
    const int first = (u % takes) * kTake;
#pragma unroll
    for (int w = 1; w < kTake; w *= 2)
#pragma unroll
      for (int i = 0; i < kTake; i += 2 * w)
        if (first + i + w < a.parts) k[i] = best_of(k[i], k[i + w]);
  };
  if (warp < units) load_keys(warp);
  // A row's total is (x - top) + rest: top its maximum, rest the score less the log
  // of the sum beside it. (Added up first, both would be lost beside a large top.)
  for (int b = warp; b < p.beams; b += kWarps) {
    const long long row = static_cast<long long>(g) * p.beams + b;
    const double score = p.score[row];
    Part q[kMaxParts / 32];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) {
      q[i] = i * 32 + lane < a.parts ? part_of(b * a.parts + i * 32 + lane) : Part{0.0, -INFINITY};
      m = fmaxf(m, q[i].m);
    }
    m = warp_max(m);
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i)  // (NaN stays; a part of nothing has z 0)
      if (i * 32 < a.parts) z += q[i].m == -INFINITY ? q[i].z : q[i].z * exp_down(static_cast<double>(q[i].m) - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) {
      sh.top[b] = m;
      sh.rest[b] = score - log2(z) * kLn2;
    }
  }
  if (warp < units) best_key(warp);
  __syncthreads();
  Cand mine = {0.0, -1};
  for (int u = warp; u < units; u += kWarps) {
    if (u != warp) {
      load_keys(u);
      best_key(u);
    }
    const int b = u / takes;
    Cand c = {0.0, -1};
    if (k[0]) {
      c.total = (static_cast<double>(key_value(k[0])) - sh.top[b]) + sh.rest[b];
      // a dead beam, or a row with a NaN or +inf, has no candidates
      if (fabs(c.total) <= 1.7e308) c.place = static_cast<long long>(b) << 32 | key_index(k[0]);
    }
    mine = u == warp ? c : best_of(mine, c);
  }
  sh.list[warp][lane] = mine;
  const int used = min(kWarps, units);
  for (int s = 1; s < used; s <<= 1) {
    __syncthreads();
    if ((warp & (2 * s - 1)) == 0 && warp + s < used) {
      mine = best_of(mine, sh.list[warp + s][lane]);
      sh.list[warp][lane] = mine;
    }
  }
  if (warp != 0) return;
  const bool live = lane < p.cands && mine.place >= 0;
  const int parent = live ? static_cast<int>(mine.place >> 32) : -1;
  const int token = live ? static_cast<int>(mine.place) : -1;
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
  // (dst may be slot itself: read by all before it is written)
  const int home = stays ? mother : nth_bit(lost, __popc(moves & ((1u << lane) - 1)));
  const long long row = static_cast<long long>(g) * p.beams;
  const int to = p.slot[row + home], from = mother >= 0 ? p.slot[row + mother] : -1;
  __syncwarp(p.beams == 32 ? 0xffffffffu : (1u << p.beams) - 1);
  p.dst[at] = to;
  p.src[at] = from;
}

constexpr int kMaxBlocks = 16;  // of a cluster

__host__ __device__ inline int slots_of(int beams, int parts, int blocks) {
  return (beams * parts + blocks - 1) / blocks;
}

// 64 prompts of eight beams, 129,280 BF16 logits, 112 of the 512 beams dead: 66 us,
// 1.6 TB/s of the 104 MB that are read (floor 16 us). No unit is near its limit
// (DRAM 19%, exponentials 24%, issue slots 32%): a block's steps, its looks at
// candidates, a part's end and the merge (5 us) come one after the other, and
// warps wait at the barriers between them; some 50 to 80 bytes a thread go through
// local memory at 64 registers. One prompt of four beams, fp32: 16 us, of which the
// host's call is 10, reading and choosing 5 and the merge 6 overlapped with the next
// call's start (14.6 us in two launches, one for the parts and one for the merge,
// where the batch took 106).
template <bool kBf16, bool kFew>
__global__ void __launch_bounds__(kThreads<kFew>, kBlocks<kFew>) beam_kernel(const BeamArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];  // this block's parts, then their keys
  __shared__ union {
    Held held;
    Merge merge;
  } sh;
  const int slots = slots_of(a.p.beams, a.parts, a.blocks), units = a.p.beams * a.parts;
  Part* part = reinterpret_cast<Part*>(smem);
  Key* keys = reinterpret_cast<Key*>(part + slots);
  const int g = blockIdx.x / a.blocks, rank = blockIdx.x - g * a.blocks;
  pdl_wait();
  pdl_trigger();
  for (int u = rank, slot = 0; u < units; u += a.blocks, ++slot) {
    const int b = u / a.parts;
    // nothing of a dead beam's row is read (of a prompt just begun all but one)
    if (!(fabsf(a.p.score[static_cast<long long>(g) * a.p.beams + b]) < INFINITY)) {
      if (threadIdx.x == 0) part[slot] = {0.0, -INFINITY};
      if (threadIdx.x < a.p.cands) keys[slot * a.p.cands + threadIdx.x] = 0;
      continue;
    }
    take_part<kBf16, kFew>(sh.held, a, static_cast<long long>(g) * a.p.beams + b, u - b * a.parts,
                           part + slot, keys + slot * a.p.cands);
  }
  cluster_arrive();
  cluster_wait();
  if (rank == 0) merge_group<kFew>(sh.merge, a, g, part, keys);
  __syncwarp();
  cluster_arrive();  // until then the others' shared memory is read
  cluster_wait();
}

// How rows are cut and over how many blocks a prompt's parts are dealt out: what
// the slowest place of the GPU takes in steps, a part's start, choice and end
// counted as three, and the merge of eight parts as one.
void deal(const BeamProblem& p, int span, int places, BeamArgs* a) {
  const int steps = (p.vocab - 1) / span + 1;
  const int most = steps < kMaxParts ? steps : kMaxParts;
  double least = 0.0;
  a->parts = 0;
  for (int n = 1; n <= most; ++n) {
    const int each = (steps + n - 1) / n;
    if (n > 1 && (steps + n - 2) / (n - 1) == each) continue;  // no shorter
    for (int blocks = 1; blocks <= kMaxBlocks && blocks < 2 * p.beams * n; blocks *= 2) {
      const double waves =
          static_cast<double>((static_cast<long long>(p.groups) * blocks + places - 1) / places);
      const double cost = waves * slots_of(p.beams, n, blocks) * (each + 3) + p.beams * n / 64 + n / 8;
      if (a->parts == 0 || cost < least) {
        least = cost;
        a->parts = n;
        a->steps = each;
        a->blocks = blocks;
      }
    }
  }
}

}  // namespace

cudaError_t beam_select(const BeamProblem& p, cudaStream_t st) {
  if (p.groups <= 0) return cudaSuccess;
  BeamArgs a;
  a.p = p;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const bool few = p.groups * static_cast<long long>(kMaxBlocks) <= sms;
  if (few)
    deal(p, kThreads<true> * (p.bf16 ? kPer<true, true> : kPer<false, true>), kBlocks<true> * sms, &a);
  else
    deal(p, kThreads<false> * (p.bf16 ? kPer<true, false> : kPer<false, false>), kBlocks<false> * sms, &a);
  const int size = p.bf16 ? 2 : 4;
  a.wide = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.stride * size % 16 == 0;
  if (static_cast<long long>(p.groups) * a.blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  auto kernel = few ? (p.bf16 ? beam_kernel<true, true> : beam_kernel<false, true>)
                    : (p.bf16 ? beam_kernel<true, false> : beam_kernel<false, false>);
  const void* fn = reinterpret_cast<const void*>(kernel);
  const int bytes = slots_of(p.beams, a.parts, a.blocks) *
                    static_cast<int>(sizeof(Part) + sizeof(Key) * p.cands);
  prefer_max_shared(fn);
  e = set_max_dynamic_smem(fn, 160 * 1024);
  if (e == cudaSuccess && bytes > 160 * 1024) e = cudaErrorInvalidValue;
  if (e == cudaSuccess && a.blocks > 8)  // more than every device has to take
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.groups * a.blocks));
  cfg.blockDim = dim3(few ? kThreads<true> : kThreads<false>);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(a.blocks), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace dsv4
