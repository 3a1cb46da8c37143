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
  int* map;       // [n_pages]
};

__host__ __device__ inline int max_jobs(int n_pages, int n_seqs) {
  return n_pages > n_seqs ? n_pages : n_seqs;
}

__host__ __device__ inline Ws carve(void* ws, int n_pages, int n_seqs) {
  Ws w;
  w.head = static_cast<int*>(ws);
  w.jobs = reinterpret_cast<PageJob*>(w.head + 64);
  w.map = reinterpret_cast<int*>(w.jobs + max_jobs(n_pages, n_seqs));
  return w;
}

// Exclusive prefix sum over the block's threads; *total = the block's sum.
__device__ int block_scan(int v, int* total) {
  __shared__ int part[32];
  __shared__ int sum;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();  // the previous call's reads of part and sum
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int w = lane < nw ? part[lane] : 0;
    int wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, wi, o);
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

// The lowest `want` free pages, ascending, into page[]; returns how many
// there are. Whole block.
__device__ int take_free(const PagedState& p, int want, int* page) {
  int have = 0;
  for (int base = 0; base < p.n_pages && have < want; base += blockDim.x) {
    const int q = base + threadIdx.x;
    const int is_free = q < p.n_pages && p.refs[q] == 0;
    int total;
    const int r = have + block_scan(is_free, &total);
    if (is_free && r < want) page[r] = q;
    have += total;
  }
  __syncthreads();
  return have < want ? have : want;
}

// ops' first claims on a slot: owner[s] = the lowest op that names it.
__device__ void claim(const PagedState& p, const int* slots, int n, int* owner) {
  for (int s = threadIdx.x; s < p.n_seqs; s += blockDim.x) owner[s] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (in_range(slots[i], p.n_seqs)) atomicMin(&owner[slots[i]], i);
  __syncthreads();
}

__global__ void __launch_bounds__(kMetaThreads) fork_kernel(const __grid_constant__ PagedState p,
                                                            const int* __restrict__ dst,
                                                            const int* __restrict__ src, int n) {
  extern __shared__ int sm[];
  int* owner = sm;                 // [n_seqs]
  int* rank = owner + p.n_seqs;    // [n] place among the ops that need a page; -1 none, -2 no op
  int* page = rank + n;            // [n] the pages taken
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  claim(p, dst, n, owner);
  // Which ops are done, and which of them need a page of their own: the
  // source's last page where it is not full.
  int needs = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0, state = -2;
    if (i < n) {
      const int d = dst[i], s = src[i];
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
    for (int j = lane; j < p.max_pages; j += 32) {
      const int q = row[j];
      if (in_range(q, p.n_pages)) atomicSub(&p.refs[q], 1);
      row[j] = -1;
    }
  }
  __syncthreads();
  const int got = take_free(p, needs, page);
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  if (threadIdx.x == 0) w.head[0] = got;
  for (int i = warp; i < n; i += nw) {
    const int r = rank[i];
    if (r == -2) continue;
    const int d = dst[i], s = src[i];
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
    for (int j = lane; j < f; j += 32) {
      const int q = from[j];
      if (in_range(q, p.n_pages)) {
        atomicAdd(&p.refs[q], 1);
        row[j] = q;
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
  claim(p, slots, n, owner);
  int needs = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0;
    bool ok = false;
    if (i < n) {
      const int s = slots[i], c = counts[i];
      ok = in_range(s, p.n_seqs) && c >= 0 && owner[s] == i;
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
  long long out = 0;  // tokens of the ops before
  for (int base = 0; base < n; base += nw) {
    // this round's ops: where their tokens' rows go
    long long mine = out;
    for (int k = 0; k < nw && base + k < n; ++k) {
      const int c = max(counts[base + k], 0);
      if (k < warp) mine += c;
      out += c;
    }
    const int i = base + warp;
    if (i >= n) continue;
    const int s = slots[i], c = max(counts[i], 0), r = start[i];
    bool done = r >= 0;
    int len = 0;
    if (done) {
      len = p.length[s];
      const int have = (len + p.page - 1) / p.page, want = (len + c + p.page - 1) / p.page;
      if (want > have && r + want - have > got) {
        done = false;
        if (lane == 0) raise(p, kPagedExhausted);
      } else {
        int* row = p.table + static_cast<size_t>(s) * p.max_pages;
        for (int j = lane; j < want - have; j += 32) {
          row[have + j] = page[r + j];
          p.refs[page[r + j]] = 1;
        }
        __syncwarp();
      }
    }
    if (rows) {
      const int* row = done ? p.table + static_cast<size_t>(s) * p.max_pages : nullptr;
      for (int t = lane; t < c && mine + t < n_rows; t += 32) {
        const int pos = len + t;
        rows[mine + t] =
            done ? static_cast<long long>(row[pos / p.page]) * p.page + pos % p.page : -1;
      }
      if (mine + c > n_rows && lane == 0) raise(p, kPagedBadOp);
    }
    __syncwarp();
    if (done && lane == 0) p.length[s] = len + c;
  }
}

// The i-th page in use beyond the live count moves to the i-th hole below
// it: no page is both, so all moves can run at once, and their number is
// the smallest that makes the pool dense.
__global__ void __launch_bounds__(kMetaThreads) compact_kernel(
    const __grid_constant__ PagedState p, int* __restrict__ refs_out) {
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  int live = 0;
  for (int base = 0; base < p.n_pages; base += blockDim.x) {
    const int q = base + threadIdx.x;
    int total;
    block_scan(q < p.n_pages && p.refs[q] > 0, &total);
    live += total;
  }
  int holes = 0, moves = 0;
  for (int base = 0; base < p.n_pages; base += blockDim.x) {
    const int q = base + threadIdx.x;
    const bool used = q < p.n_pages && p.refs[q] > 0;
    const bool hole = q < live && !used, move = q >= live && used;
    int th, tm;
    const int h = holes + block_scan(hole, &th);
    const int m = moves + block_scan(move, &tm);
    if (hole) w.jobs[h].dst = q;
    if (move) {
      w.jobs[m].src = q;
      w.jobs[m].rows = p.page;
      w.map[q] = m;
    }
    holes += th;
    moves += tm;
  }
  __syncthreads();
  // refs_out may be refs: a move's two pages are read and written by one thread
  for (int q = threadIdx.x; q < p.n_pages; q += blockDim.x) {
    if (q >= live && p.refs[q] > 0) {
      const int to = w.jobs[w.map[q]].dst, r = p.refs[q];
      refs_out[to] = r;
      refs_out[q] = 0;
      w.map[q] = to;
    } else if (q >= live) {
      refs_out[q] = p.refs[q];
      w.map[q] = -1;  // free: no table names it
    } else if (p.refs[q] > 0) {
      refs_out[q] = p.refs[q];
    }
  }
  if (threadIdx.x == 0) {
    w.head[0] = moves;
    w.head[1] = live;
  }
}

__global__ void remap_kernel(const __grid_constant__ PagedState p, int* __restrict__ table_out) {
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  const int live = w.head[1];
  const size_t n = static_cast<size_t>(p.n_seqs) * p.max_pages;
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<size_t>(gridDim.x) * blockDim.x) {
    const int q = p.table[i];
    table_out[i] = q >= live && q < p.n_pages ? w.map[q] : q;
  }
}

__device__ void copy_bytes(uint8_t* dst, const uint8_t* src, size_t bytes) {
  for (size_t i = threadIdx.x; i < bytes; i += blockDim.x) dst[i] = src[i];
}

// One block per (job, layer), jobs striding over the grid.
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ PagedState p) {
  const Ws w = carve(p.ws, p.n_pages, p.n_seqs);
  const long long n = static_cast<long long>(w.head[0]) * p.layers;
  for (long long b = blockIdx.x; b < n; b += gridDim.x) {
    const PageJob j = w.jobs[b / p.layers];
    const int l = static_cast<int>(b % p.layers);
    const size_t from = static_cast<size_t>(j.src) * p.page, to = static_cast<size_t>(j.dst) * p.page;
    copy_bytes(p.codes[l] + to * p.nope, p.codes[l] + from * p.nope,
               static_cast<size_t>(j.rows) * p.nope);
    copy_bytes(p.scales[l] + to * 8, p.scales[l] + from * 8, static_cast<size_t>(j.rows) * 8);
    copy_bytes(reinterpret_cast<uint8_t*>(p.rope[l] + to * p.rope_dim),
               reinterpret_cast<const uint8_t*>(p.rope[l] + from * p.rope_dim),
               static_cast<size_t>(j.rows) * p.rope_dim * 2);
  }
}

cudaError_t smem_limit(const void* fn, size_t bytes) {
  return bytes <= 48 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(bytes));
}

}  // namespace

size_t paged_workspace_bytes(int n_pages, int n_seqs) {
  return 256 + sizeof(PageJob) * static_cast<size_t>(max_jobs(n_pages, n_seqs)) +
         sizeof(int) * static_cast<size_t>(n_pages);
}

cudaError_t paged_fork(const PagedState& p, const int* dst, const int* src, int n,
                       cudaStream_t st) {
  if (n <= 0) return cudaSuccess;
  const size_t smem = sizeof(int) * (static_cast<size_t>(p.n_seqs) + 2 * static_cast<size_t>(n));
  cudaError_t e = smem_limit(reinterpret_cast<const void*>(fork_kernel), smem);
  if (e != cudaSuccess) return e;
  fork_kernel<<<1, kMetaThreads, smem, st>>>(p, dst, src, n);
  copy_kernel<<<148 * 8, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t paged_append(const PagedState& p, const int* slots, const int* counts, int n,
                         long long* rows, long long n_rows, cudaStream_t st) {
  if (n <= 0) return cudaSuccess;
  const size_t smem = sizeof(int) * (static_cast<size_t>(p.n_seqs) + static_cast<size_t>(n));
  cudaError_t e = smem_limit(reinterpret_cast<const void*>(append_kernel), smem);
  if (e != cudaSuccess) return e;
  append_kernel<<<1, kMetaThreads, smem, st>>>(p, slots, counts, n, rows, n_rows);
  return cudaGetLastError();
}

cudaError_t paged_compact(const PagedState& p, int* table_out, int* refs_out, cudaStream_t st) {
  compact_kernel<<<1, kMetaThreads, 0, st>>>(p, refs_out);
  remap_kernel<<<148, 256, 0, st>>>(p, table_out);
  copy_kernel<<<148 * 8, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dsv4
