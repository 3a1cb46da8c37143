// paged.cu - page bookkeeping of the latent cache, on the device.
//
// Sequences hold their latents in pages of the cache's rows and may share
// them (samples forked off one prompt). Which pages a slot holds changes
// inside a captured step (a verify step accepts a number of tokens that the
// host does not know), so tables, lengths and reference counts live in
// device memory and every operation is a function of that state alone:
// free pages are taken in ascending order, op after op, so a call gives the
// same tables whatever order its threads run in.
#include "paged.cuh"

#include <climits>

#include "launch.cuh"

namespace dsv4 {
namespace {

constexpr int kMetaThreads = 1024;

struct PageJob {
  int src, dst, rows;  // rows [0, rows) of page src to page dst, every layer
};

// Workspace: job count and live count, jobs, then per-page maps.
struct Ws {
  int* head;      // [0] jobs, [1] pages in use
  PageJob* jobs;  // [max(n_seqs, n_pages)]
  long long* first;  // [n_seqs + 1] first token of each op
  int* map;          // [n_pages]
};

__host__ __device__ inline int max_jobs(int n_pages, int n_seqs) {
  return n_pages > n_seqs ? n_pages : n_seqs;
}

__host__ __device__ inline Ws carve(void* ws, int n_pages, int n_seqs) {
  Ws w;
  w.head = static_cast<int*>(ws);
  w.jobs = reinterpret_cast<PageJob*>(w.head + 64);
  // (12-byte jobs: rounded up to whole 16 bytes)
  w.first = reinterpret_cast<long long*>(reinterpret_cast<char*>(w.jobs) +
                                         ((sizeof(PageJob) * max_jobs(n_pages, n_seqs) + 15) & ~15ull));
  w.map = reinterpret_cast<int*>(w.first + n_seqs + 1);
  return w;
}

// Exclusive prefix sum over the block's threads; *total = the block's sum.
template <class T>
__device__ T block_scan(T v, T* total) {
  __shared__ T part[32];
  __shared__ T sum;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  T incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();  // the previous call's reads of part and sum
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const T w = lane < nw ? part[lane] : 0;
    T wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T u = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += u;
    }
    part[lane] = wi - w;
    if (lane == 31) sum = wi;
  }
  __syncthreads();
  *total = sum;
  return part[warp] + incl - v;
}

__device__ __forceinline__ bool in_range(int v, int n) { return v >= 0 && v < n; }

__device__ void raise(const PagedState& p, unsigned bits) {
  if (p.status) atomicOr(p.status, bits);
}

// Four counts of pages from q on; pages that there are not are in use.
__device__ __forceinline__ int4 refs4(const PagedState& p, int q) {
  if (q + 3 < p.n_pages && (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0)
    return *reinterpret_cast<const int4*>(p.refs + q);
  return make_int4(q < p.n_pages ? p.refs[q] : 1, q + 1 < p.n_pages ? p.refs[q + 1] : 1,
                   q + 2 < p.n_pages ? p.refs[q + 2] : 1, q + 3 < p.n_pages ? p.refs[q + 3] : 1);
}

// The lowest `want` free pages (a count below 0 is no use either), ascending,
// into page[]; returns how many there are. Whole block: four pages a thread, the
// next four on their way.
__device__ int take_free(const PagedState& p, int want, int* page) {
  int have = 0;
  const int q0 = 4 * threadIdx.x;
  int4 next = want > 0 ? refs4(p, q0) : make_int4(1, 1, 1, 1);
  for (int base = 0; base < p.n_pages && have < want; base += 4 * blockDim.x) {
    const int q = base + q0;
    const int4 r = next;
    if (base + 4 * static_cast<int>(blockDim.x) < p.n_pages) next = refs4(p, q + 4 * blockDim.x);
    const int f[4] = {r.x <= 0, r.y <= 0, r.z <= 0, r.w <= 0};
    int total;
    int at = have + block_scan(f[0] + f[1] + f[2] + f[3], &total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f[i]) {
        if (at < want) page[at] = q + i;
        ++at;
      }
    have += total;
  }
  __syncthreads();
  return have < want ? have : want;
}

// This lane's next entries of a table row, all on their way at once; -1
// behind its end.
constexpr int kAhead = 4;
__device__ __forceinline__ void load_pages(const int* row, int j0, int n, int (&q)[kAhead]) {
#pragma unroll
  for (int k = 0; k < kAhead; ++k) q[k] = j0 + 32 * k < n ? row[j0 + 32 * k] : -1;
}

// ops' first claims on a slot: owner[s] = the lowest op that names it.
__device__ void claim(const PagedState& p, const int* slots, int n, int* owner) {
  for (int s = threadIdx.x; s < p.n_seqs; s += blockDim.x) owner[s] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (in_range(slots[i], p.n_seqs)) atomicMin(&owner[slots[i]], i);
  __syncthreads();
}

// One block: the ops depend on one another through the free pages, and what
// they touch is small (64 ops on 96 slots of 15 pages: 8 us), so what counts
// is the chain of dependent accesses: lengths and tables, the pages given
// back, the scan of the counts, the new tables. A
// warp has an op and asks for 128 entries of a table row at once (one entry a
// lane and round: 9.5 us instead of 5 where 48 slots hold 125 pages each).
__global__ void __launch_bounds__(kMetaThreads) fork_kernel(const __grid_constant__ PagedState p,
                                                            const int* __restrict__ dst,
                                                            const int* __restrict__ src, int n) {
  extern __shared__ int sm[];
  int* owner = sm;                 // [n_seqs]
  int* rank = owner + p.n_seqs;    // [n] place among the ops that need a page; -1 none, -2 no op
  int* page = rank + n;            // [n] the pages taken
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  claim(p, dst, n, owner);
  // Which ops are done, and which of them need a page of their own: the
  // source's last page where it is not full.
  int needs = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0, state = -2;
    if (i < n) {
      const int d = dst[i], s = src ? src[i] : -1;
      bool ok = in_range(d, p.n_seqs) && s >= -1 && s < p.n_seqs && owner[d] == i;
      // a source that another op replaces is no longer what was asked for
      if (ok && s >= 0 && s != d && owner[s] != INT_MAX && src[owner[s]] != s) ok = false;
      if (!ok) {
        raise(p, kPagedBadOp);
      } else if (s != d) {
        state = -1;
        if (s >= 0) {
          const int len = min(max(p.length[s], 0), p.max_pages * p.page);
          const int f = len / p.page;
          need = len % p.page != 0 &&
                 in_range(p.table[static_cast<size_t>(s) * p.max_pages + f], p.n_pages);
        }
      }
    }
    int total;
    const int r = needs + block_scan(need, &total);
    if (i < n) rank[i] = need ? r : state;
    needs += total;
  }
  __syncthreads();
  // The destinations give back what they held.
  for (int i = warp; i < n; i += nw) {
    if (rank[i] == -2) continue;
    int* row = p.table + static_cast<size_t>(dst[i]) * p.max_pages;
    for (int j0 = lane; j0 < p.max_pages; j0 += 32 * kAhead) {
      int q[kAhead];
      load_pages(row, j0, p.max_pages, q);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (in_range(q[k], p.n_pages)) atomicSub(&p.refs[q[k]], 1);
        if (j0 + 32 * k < p.max_pages) row[j0 + 32 * k] = -1;
      }
    }
  }
  __syncthreads();
  const int got = take_free(p, needs, page);
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  if (threadIdx.x == 0) w.head[0] = got;
  for (int i = warp; i < n; i += nw) {
    const int r = rank[i];
    if (r == -2) continue;
    const int d = dst[i], s = src ? src[i] : -1;
    if (s < 0 || r >= got) {  // emptied, or no page left for it
      if (lane == 0) {
        p.length[d] = 0;
        if (s >= 0) raise(p, kPagedExhausted);
      }
      continue;
    }
    const int len = min(max(p.length[s], 0), p.max_pages * p.page);
    const int f = len / p.page;
    const int* from = p.table + static_cast<size_t>(s) * p.max_pages;
    int* row = p.table + static_cast<size_t>(d) * p.max_pages;
    for (int j0 = lane; j0 < f; j0 += 32 * kAhead) {
      int q[kAhead];
      load_pages(from, j0, f, q);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (in_range(q[k], p.n_pages)) {
          atomicAdd(&p.refs[q[k]], 1);
          row[j0 + 32 * k] = q[k];
        }
    }
    if (lane == 0) {
      p.length[d] = len;
      if (r >= 0) {
        row[f] = page[r];
        p.refs[page[r]] = 1;
        w.jobs[r] = {from[f], page[r], len % p.page};
      }
    }
  }
}

// One block, as the fork: the ops' needs, prefix sums of them (so the pages of
// an op do not depend on timing; an op that finds none keeps its place, so that
// no later one overtakes it), the lowest free pages in one scan of the
// counts, four a thread, the next four on their way (48 ops that take 3,400
// of 16,384 pages: 9 us).
__global__ void __launch_bounds__(kMetaThreads) append_kernel(const __grid_constant__ PagedState p,
                                                              const int* __restrict__ slots,
                                                              const int* __restrict__ counts, int n,
                                                              long long* __restrict__ rows,
                                                              long long n_rows) {
  extern __shared__ int sm[];
  int* owner = sm;               // [n_seqs]
  int* start = owner + p.n_seqs; // [n] pages that the ops before this one need; -1 no op
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  int* page = w.map;
  pdl_trigger();
  claim(p, slots, n, owner);
  int needs = 0;
  long long out = 0;  // tokens of the ops before: where an op's rows begin
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0;
    bool ok = false;
    long long tokens;
    const long long begin = out + block_scan(i < n ? max(counts[i], 0) + 0ll : 0ll, &tokens);
    out += tokens;
    if (i < n) {
      const int s = slots[i], c = counts[i];
      w.first[i] = begin;
      ok = in_range(s, p.n_seqs) && c >= 0 && owner[s] == i && (!rows || begin + c <= n_rows);
      if (ok) {
        const int len = p.length[s], cap = p.max_pages * p.page;
        ok = len >= 0 && len <= cap && c <= cap - len;
        // tokens go behind the last one, so its page must be this slot's alone
        if (ok && c > 0 && len % p.page != 0) {
          const int q = p.table[static_cast<size_t>(s) * p.max_pages + len / p.page];
          ok = in_range(q, p.n_pages) && p.refs[q] == 1;
        }
        if (ok) need = (len + c + p.page - 1) / p.page - (len + p.page - 1) / p.page;
      }
      if (!ok) raise(p, kPagedBadOp);
    }
    int total;
    const int r = needs + block_scan(need, &total);
    if (i < n) start[i] = ok ? r : -1;
    needs += total;
  }
  const int got = take_free(p, min(needs, p.n_pages), page);
  for (int i = warp; i < n; i += nw) {
    const int r = start[i];
    int len = -1;  // not done
    if (r >= 0) {
      const int s = slots[i], c = counts[i];
      len = p.length[s];
      const int have = (len + p.page - 1) / p.page, want = (len + c + p.page - 1) / p.page;
      if (want > have && r + want - have > got) {
        len = -1;
        if (lane == 0) raise(p, kPagedExhausted);
      } else {
        int* row = p.table + static_cast<size_t>(s) * p.max_pages;
        for (int j = lane; j < want - have; j += 32) {
          row[have + j] = page[r + j];
          p.refs[page[r + j]] = 1;
        }
        __syncwarp();
        if (lane == 0) p.length[s] = len + c;
      }
    }
    if (lane == 0) w.jobs[i].src = len;
  }
  if (threadIdx.x == 0) w.first[n] = out;
}

// The cache row of each new token, -1 behind the last one (a captured step has
// rows for the most tokens that it may bring, and what it does not bring must
// not be written where the step before had its own): a thread per token finds
// its op by a search in shared memory (the ops' starts are loaded once a block; in global
// memory every probe costs an L2 access), 54,000 tokens of 48 ops in 3.4 us.
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ PagedState p,
                                                   const int* __restrict__ slots, int n,
                                                   long long* __restrict__ rows, long long n_rows) {
  extern __shared__ long long first[];  // [n + 1]
  pdl_wait();
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  for (int i = threadIdx.x; i <= n; i += 256) first[i] = w.first[i];
  __syncthreads();
  const long long total = first[n];
  for (long long t = blockIdx.x * 256ll + threadIdx.x; t < n_rows; t += gridDim.x * 256ll) {
    int lo = 0, hi = n;  // the last op with first <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int len = t < total ? w.jobs[lo].src : -1;
    long long row = -1;
    if (len >= 0) {
      const int pos = len + static_cast<int>(t - first[lo]);
      row = static_cast<long long>(
                p.table[static_cast<size_t>(slots[lo]) * p.max_pages + pos / p.page]) * p.page +
            pos % p.page;
    }
    rows[t] = row;
  }
}

// The i-th page in use beyond the live count moves to the i-th hole below
// it: no page is both, so all moves can run at once, and their number is
// the smallest that makes the pool dense. (A page is in use or a hole whatever
// its count, one below 0 too: there are as many holes as moves in any state.)
__global__ void __launch_bounds__(kMetaThreads) compact_kernel(
    const __grid_constant__ PagedState p, int* refs_out) {
  pdl_trigger();
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  int live = 0;
  for (int q = 4 * threadIdx.x; q < p.n_pages; q += 4 * blockDim.x) {
    const int4 r = refs4(p, q);
    live += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0);
    if (q + 3 >= p.n_pages)  // (the ones that there are not)
      live -= min(3, q + 4 - p.n_pages);
  }
  block_scan(live, &live);
  int holes = 0, moves = 0;
  for (int base = 0; base < p.n_pages; base += 4 * blockDim.x) {
    const int q = base + 4 * threadIdx.x;
    const int4 r4 = refs4(p, q);
    const int r[4] = {r4.x, r4.y, r4.z, r4.w};
    int h = 0, m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = q + i < p.n_pages;
      h += in && q + i < live && r[i] <= 0;
      m += in && q + i >= live && r[i] > 0;
    }
    // both counts in one scan: below 2^16 a block's step
    int total;
    const int before = block_scan(h | (m << 16), &total);
    int ha = holes + (before & 0xFFFF), ma = moves + (before >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (q + i >= p.n_pages) continue;
      if (q + i < live) {
        if (r[i] <= 0) w.jobs[ha++].dst = q + i;
      } else if (r[i] > 0) {
        w.jobs[ma].src = q + i;
        w.jobs[ma].rows = p.page;
        w.map[q + i] = ma++;
      } else {
        w.map[q + i] = -1;  // free: no table names it
      }
    }
    holes += total & 0xFFFF;
    moves += total >> 16;
  }
  __syncthreads();
  // (refs_out may be refs: a move's two pages are one thread's)
  for (int i = threadIdx.x; i < moves; i += blockDim.x) {
    const PageJob j = w.jobs[i];
    const int r = p.refs[j.src];
    w.map[j.src] = j.dst;
    refs_out[j.dst] = r;
    refs_out[j.src] = 0;
  }
  __syncthreads();
  if (refs_out != p.refs)
    for (int q = threadIdx.x; q < p.n_pages; q += blockDim.x) {
      const int r = p.refs[q];
      if (q < live ? r > 0 : r <= 0) refs_out[q] = r;
    }
  if (threadIdx.x == 0) {
    w.head[0] = moves;
    w.head[1] = live;
  }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 10;  // 16-byte vectors in flight per thread: a page of 64 rows at once

// `bytes` from src to dst in pieces of T, whose size divides all three.
template <class T>
__device__ __forceinline__ void copy_pieces(uint8_t* dst, const uint8_t* src, size_t bytes) {
  const size_t n = bytes / sizeof(T);
  for (size_t i = threadIdx.x; i < n; i += kCopyThreads)
    reinterpret_cast<T*>(dst)[i] = reinterpret_cast<const T*>(src)[i];
}

__device__ void copy_any(uint8_t* dst, const uint8_t* src, size_t bytes) {
  const uintptr_t a =
      reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src) | bytes;
  if (a % 16 == 0) copy_pieces<uint4>(dst, src, bytes);
  else if (a % 8 == 0) copy_pieces<uint2>(dst, src, bytes);
  else if (a % 4 == 0) copy_pieces<uint32_t>(dst, src, bytes);
  else copy_pieces<uint16_t>(dst, src, bytes);  // rows of BF16 values
}

// The rows of one (job, layer) per block and round. A move is read and
// written once, so the memory bounds it: all of a page's vectors are loaded
// before the first is stored, in whole vectors over the row boundaries (codes,
// then RoPE values, of a page are contiguous). 43 layers, pages of 64 rows:
// 275 MB moved by the compaction in 107 us, 5.1 TB/s read and written; 64
// forks' last pages, 41 MB, in 13 us, where the start and the end weigh.
// (Rows one after the other, scales and RoPE values in their own loops: 538 us
// for the compaction.)
__device__ void copy_jobs(const PagedState& p, long long block, long long blocks) {
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  const long long n = static_cast<long long>(w.head[0]) * p.layers;
  for (long long b = block; b < n; b += blocks) {
    const PageJob j = w.jobs[b / p.layers];
    const int l = static_cast<int>(b % p.layers);
    const size_t from = static_cast<size_t>(j.src) * p.page, to = static_cast<size_t>(j.dst) * p.page;
    const size_t rows = j.rows;
    const uint8_t* codes = p.codes[l] + from * p.nope;
    uint8_t* codes_to = p.codes[l] + to * p.nope;
    const uint8_t* rope = reinterpret_cast<const uint8_t*>(p.rope[l] + from * p.rope_dim);
    uint8_t* rope_to = reinterpret_cast<uint8_t*>(p.rope[l] + to * p.rope_dim);
    const uint2* scales = reinterpret_cast<const uint2*>(p.scales[l] + from * 8);
    uint2* scales_to = reinterpret_cast<uint2*>(p.scales[l] + to * 8);
    const size_t rope_bytes = rows * p.rope_dim * 2;
    const bool wide =
        ((reinterpret_cast<uintptr_t>(rope) | reinterpret_cast<uintptr_t>(rope_to) | rope_bytes) &
         15) == 0;
    // codes (64 a group: always whole vectors), then RoPE values
    const int nc = static_cast<int>(rows * p.nope / 16);
    const int nv = nc + (wide ? static_cast<int>(rope_bytes / 16) : 0);
    uint2 sc = make_uint2(0, 0);
    const bool one_scale = rows <= kCopyThreads;
    if (one_scale && threadIdx.x < rows) sc = __ldg(scales + threadIdx.x);
    for (int v0 = threadIdx.x; v0 < nv; v0 += kCopyVecs * kCopyThreads) {
      uint4 x[kCopyVecs];
#pragma unroll
      for (int u = 0; u < kCopyVecs; ++u) {
        const int v = v0 + u * kCopyThreads;
        if (v < nv)
          x[u] = v < nc ? __ldg(reinterpret_cast<const uint4*>(codes) + v)
                        : __ldg(reinterpret_cast<const uint4*>(rope) + (v - nc));
      }
#pragma unroll
      for (int u = 0; u < kCopyVecs; ++u) {
        const int v = v0 + u * kCopyThreads;
        if (v < nv) {
          if (v < nc) reinterpret_cast<uint4*>(codes_to)[v] = x[u];
          else reinterpret_cast<uint4*>(rope_to)[v - nc] = x[u];
        }
      }
    }
    if (one_scale) {
      if (threadIdx.x < rows) scales_to[threadIdx.x] = sc;
    } else {
      for (size_t i = threadIdx.x; i < rows; i += kCopyThreads) scales_to[i] = __ldg(scales + i);
    }
    if (!wide) copy_any(rope_to, rope, rope_bytes);
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ PagedState p) {
  pdl_wait();
  copy_jobs(p, blockIdx.x, gridDim.x);
}

// After compact_kernel: the tables in the first blocks, the rows in the others.
__global__ void __launch_bounds__(kCopyThreads) move_kernel(const __grid_constant__ PagedState p,
                                                            int* __restrict__ table_out,
                                                            int table_blocks) {
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= table_blocks) {
    copy_jobs(p, blockIdx.x - table_blocks, gridDim.x - table_blocks);
    return;
  }
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  const int live = w.head[1];
  const int n = p.n_seqs * p.max_pages;
  for (long long i = blockIdx.x * static_cast<long long>(kCopyThreads) + threadIdx.x; i < n;
       i += static_cast<long long>(table_blocks) * kCopyThreads) {
    const int q = p.table[i];
    table_out[i] = q >= live && q < p.n_pages ? w.map[q] : q;
  }
}

// Blocks that keep the memory busy: eight an SM hold what one of them waits for
// (275 MB moved: 112 us with the tables, 141 with two an SM; 41 MB forked: 28
// and 31).
int copy_blocks(long long most) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long all = 8ll * sms;
  return static_cast<int>(most < 1 ? 1 : most < all ? most : all);
}

}  // namespace

size_t paged_workspace_bytes(int n_pages, int n_seqs) {
  return 256 + sizeof(PageJob) * static_cast<size_t>(max_jobs(n_pages, n_seqs)) + 16 +
         sizeof(long long) * (static_cast<size_t>(n_seqs) + 1) +
         sizeof(int) * static_cast<size_t>(n_pages);
}

cudaError_t paged_fork(const PagedState& p, const int* dst, const int* src, int n,
                       cudaStream_t st) {
  if (n <= 0) return cudaSuccess;
  const size_t smem = sizeof(int) * (static_cast<size_t>(p.n_seqs) + 2 * static_cast<size_t>(n));
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(fork_kernel),
                                       sizeof(int) * 3 * kPagedMaxSeqs);
  if (e != cudaSuccess) return e;
  fork_kernel<<<1, kMetaThreads, smem, st>>>(p, dst, src, n);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_pdl(copy_kernel, dim3(copy_blocks(static_cast<long long>(n) * p.layers)),
                    dim3(kCopyThreads), 0, st, p);
}

cudaError_t paged_append(const PagedState& p, const int* slots, const int* counts, int n,
                         long long* rows, long long n_rows, cudaStream_t st) {
  if (n <= 0)
    return rows && n_rows > 0 ? cudaMemsetAsync(rows, 0xFF, sizeof(long long) * n_rows, st)
                              : cudaSuccess;
  const size_t smem = sizeof(int) * (static_cast<size_t>(p.n_seqs) + static_cast<size_t>(n));
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(append_kernel),
                                       sizeof(int) * 2 * kPagedMaxSeqs);
  if (e != cudaSuccess) return e;
  append_kernel<<<1, kMetaThreads, smem, st>>>(p, slots, counts, n, rows, n_rows);
  e = cudaGetLastError();
  if (e != cudaSuccess || !rows || n_rows <= 0) return e;
  return launch_pdl(rows_kernel, dim3(copy_blocks((n_rows + 255) / 256)), dim3(256),
                    sizeof(long long) * (static_cast<size_t>(n) + 1), st, p, slots, n, rows, n_rows);
}

cudaError_t paged_compact(const PagedState& p, int* table_out, int* refs_out, cudaStream_t st) {
  compact_kernel<<<1, kMetaThreads, 0, st>>>(p, refs_out);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int table_blocks =
      copy_blocks((static_cast<long long>(p.n_seqs) * p.max_pages + 1023) / 1024);
  return launch_pdl(move_kernel,
                    dim3(table_blocks + copy_blocks(static_cast<long long>(p.n_pages / 2) * p.layers)),
                    dim3(kCopyThreads), 0, st, p, table_out, table_blocks);
}

}  // namespace dsv4
