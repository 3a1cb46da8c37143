// grouped.cu - products of many rows grouped by expert, on the block-scaled
// tensor cores, and the routed experts of a MoE layer built from them.
//
//   out[r, i] = sum_k x[r, k] W_e[i, k]          for the rows r of group e
//
// x is E4M3 with a power of two per 128 columns, W E2M1 with one per 32 (or
// E4M3 with one per 128 x 128): exactly what tcgen05.mma's mxf8f6f4 kind
// multiplies, scales included, into fp32 sums. The weights are the A operand
// (128 outputs are the M of an instruction) and a group's rows its N, so that
// a group of a few rows wastes columns of a small N instead of rows of a
// large M: a decode step's experts are read at the same cost as a GEMV's.
//
// One block per SM takes an equal share of all (tile, 128-column chunk) units
// laid end to end; a tile is 256 outputs (or 128 gate and 128 up outputs) of
// up to 192 rows. A tile that a share's end cuts is written as fp32 parts,
// and whoever brings its last part adds them in the order of the columns, so
// that results do not depend on timing.
//
// Roles: warps 0-7 epilogue, 8-11 scales (to TMEM, each warp the copy of its
// lane quarter), 12-15 rows of x that are gathered, 16 copies by TMA (weights, and
// rows that lie in their order), 17-18 MMAs (a tile of 128 outputs each).
//
// What bounds it: with few rows a group HBM (32 tokens of 8 routes over 256
// experts of 7168 x 2048: 641 us, 5.98 TB/s of the 6.45 of a copy), as long as six
// stages are under way. With more the TMA engine, which brings a row of 128 bytes
// of shared memory in some 2.7 clocks, whatever its bytes in memory, so that 256
// weights' rows of a chunk take 690 clocks; and the shared memory's own
// bandwidth, 64 KB a chunk for writing and reading expanded E2M1 tiles and 384
// bytes a row (256 experts of 4096 x 2048: 2,000 tokens 877 us, 8,192 tokens 2.2
// ms, 1.1 PFLOP/s at the power cap). With one token launches, the plan and the
// first bytes' way (36.7 us).
#include "grouped.cuh"

#include <cuda_bf16.h>

#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

constexpr int kChunk = 128;              // columns of a stage: one row of swizzled shared memory
constexpr int kTileRows = 128;           // M of an instruction
constexpr int kATile = kTileRows * kChunk;
constexpr int kTiles = 2;                // of 128 outputs, on the same rows of x: gate and up, or 256 outputs
constexpr int kEpiWarps = 8, kScaleWarps = 4, kRowWarps = 4;
constexpr int kWarpRows = kEpiWarps + kScaleWarps, kWarpCopy = kWarpRows + kRowWarps;
constexpr int kWarpMma = kWarpCopy + 1;  // and the next, for a second tile
constexpr int kThreads = 32 * (kWarpMma + 2);
constexpr int kBlockCols = 16;           // rows of a group that an epilogue step takes
constexpr int kMaxN = 192, kHalfN = 96;  // rows of a tile; up to kHalfN two tiles' sums fit in TMEM
constexpr int kMaxStages = 6;
// TMEM columns: two buffers of scales (four chunks: 2 x 4 columns of weights'
// and 8 of rows' scales each), then the sums.
constexpr int kScaleCols = 64, kSumCol = 2 * kScaleCols, kTmemCols = 512;
constexpr int kMaxShares = 160;          // blocks
constexpr size_t kMaxSmem = 227 * 1024;

struct Args {
  GroupedProblem p;
  bool early;         // offsets are of a kernel that the one before this has waited for
  int shares;         // blocks
  int n_max, ring;    // rows of a tile at most; bytes of the ring of stages
  bool wide;          // out is BF16 and takes four outputs of a row at once
  int* counters;      // [kMaxShares] chunks whose parts are there
  float* parts;       // [shares][2][2][n_max][128]
};

struct alignas(16) Control {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t scale_full[2], scale_empty[2];
  uint64_t sum_full[2], sum_empty[2];
  uint64_t fin;
  uint32_t tmem;
  int abort_flag;
  int plan[3][kThreads / 32];  // of the warps
  long long costs[kThreads / 32];
  int last;      // the block brought a tile's last part
  alignas(16) float top[2][2][4][kBlockCols];  // largest |h| of a warp's 32 outputs
  alignas(16) float factor[2][4][kBlockCols];  // rows' weights over their blocks' scales
  alignas(16) uint8_t codes[2][kBlockCols][kTileRows];
};

// The ring of scales: an entry holds four chunks' of 256 outputs and n_max rows.
// Behind it the rows of x of two pieces.
__host__ __device__ constexpr int row_table_ints(int n_max) { return n_max + 16; }
constexpr int kScaleEntries = 3, kScaleBytes = 2 * kTileRows * 16;
__host__ __device__ constexpr int scale_entry_bytes(int n_max) { return kScaleBytes + n_max * 4; }
__host__ __device__ constexpr int scale_ring_bytes(int n_max) {
  return kScaleEntries * scale_entry_bytes(n_max) + 2 * row_table_ints(n_max) * 4;
}

__host__ __device__ constexpr int stage_bytes(int n_max) { return kTiles * kATile + n_max * kChunk; }
// Shared memory behind the ring of stages.
__host__ __device__ inline size_t rest_bytes(int n_max, int experts) {
  return scale_ring_bytes(n_max) + sizeof(Control) + (kMaxShares + 1) * sizeof(long long) +
         (experts + 1) * (sizeof(long long) + sizeof(int));
}

// Suspended waits: the epilogue needs the issue slots.
__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;"
      " selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity), "r"(20000u)  // at most 20 us at a time
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                         unsigned* err) {
  if (try_wait_long(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!try_wait_long(bar, parity)) {
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      if (err) atomicOr(err, kErrWait);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

// D (+)= A B with block scales: A and B types in idesc, one E8M0 per 32
// columns. a and b: shared memory in 16 bytes, of tiles with the 128-byte
// swizzle whose groups of eight rows lie one behind the other.
__device__ __forceinline__ void mma_scaled(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           uint32_t scale_a, uint32_t scale_b, bool accumulate) {
  constexpr uint32_t kHigh = (1024 >> 4) | (1u << 14) | (2u << 29);  // as umma_desc has it
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %6, 0;\n"
      " mov.b64 x, {%1, %7};\n mov.b64 y, {%2, %7};\n"
      " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X"
      " [%0], x, y, %3, [%4], [%5], p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate ? 1u : 0u), "r"(kHigh)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e; }" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_addr(bar))
      : "memory");
}
// 16 consecutive TMEM columns of this thread's lane, of two tiles.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait16(float (&r)[16], float (&s)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]),
                 "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]),
                 "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(s[0]), "+f"(s[1]),
                 "+f"(s[2]), "+f"(s[3]), "+f"(s[4]), "+f"(s[5]), "+f"(s[6]), "+f"(s[7]),
                 "+f"(s[8]), "+f"(s[9]), "+f"(s[10]), "+f"(s[11]), "+f"(s[12]), "+f"(s[13]),
                 "+f"(s[14]), "+f"(s[15])::"memory");
}
// The smaller or larger of two, NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
// The largest magnitude of a warp's, NaN if one is.
__device__ __forceinline__ float warp_top(float a) {
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(a));
  return r;
}
// 8 consecutive TMEM columns of this thread's lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(taddr));
}
// The wait names the registers so that no use is scheduled before it.
__device__ __forceinline__ void tmem_ld_wait8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7])::"memory");
}

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
// Zeros where there is nothing to be read.
__device__ __forceinline__ void cp_async16_or_0(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0)
               : "memory");
}
// This thread's arrival once all its copies so far are there.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// ------------------------------------------------------------------ plan --

// How a group of n rows is cut: tiles of the same number of rows, a multiple
// of 16, and what a chunk of one costs in clocks (as measured: 740 for 16 rows, 830
// for 48, 930 for 80, where two tiles' sums fit in TMEM; beyond that the epilogue
// is not overlapped). With every chunk counted alike the slowest block took 558 us
// where the mean was 455 (2,000 tokens of 4096 x 2048, gate and up).
struct Cut {
  int tiles, rows, cost;
};
constexpr int kSnapTiles = 8;  // shares of so many tiles on average are not cut
// What a tile's parts take to meet, in such clocks (one group of 8 rows: 64 tiles
// of 56 chunks 22.9 us cut and 25.1 whole, 96 tiles of 32 chunks 21.5 and 18.4).
constexpr int kJoin = 20000;
// (flat: shares are single tiles, and a chunk counts 1)
__device__ __forceinline__ Cut cut_group(int n, int n_max, int chunks, bool flat) {
  Cut c;
  const int sixteens = (n + 15) >> 4, most = n_max >> 4;
  c.tiles = n > 0;
  int each = max(sixteens, 1);
  if (sixteens > most) {  // (three divisions: 500 clocks that most groups need not wait for)
    c.tiles = (sixteens + most - 1) / most;
    each = (sixteens + c.tiles - 1) / c.tiles;
    c.tiles = (sixteens + each - 1) / each;
  }
  c.rows = each * 16;
  c.cost = flat ? 1 : 690 + 3 * c.rows + (c.rows > kHalfN ? 67 * c.rows / chunks : 0);
  return c;
}

// A share's part of one tile.
struct Piece {
  int e, row_tile;     // matrix, 256 (gated: 128) outputs
  int row0, rows, n;   // first row of the tile, rows there are, columns of the MMAs
  int lo, hi;          // chunks
};

// d / by, quotients of a few million at most off by a handful at first: a
// fraction of what a division of 64 bits takes.
__device__ __forceinline__ int quotient(long long d, long long by) {
  int q = static_cast<int>(static_cast<float>(d) * __frcp_rn(static_cast<float>(by)));
  long long rest = d - q * by;
  while (rest < 0) rest += by, --q;
  while (rest >= by) rest -= by, ++q;
  return q;
}

// The chunk of a tile of `cost` a chunk in which position d behind its start lies.
__device__ __forceinline__ int chunk_at(long long d, int chunks, int cost) {
  return d <= 0 ? 0
                : d >= static_cast<long long>(chunks) * cost
                      ? chunks
                      : static_cast<int>(static_cast<unsigned>(d) / static_cast<unsigned>(cost));
}

// The last group that does not start behind position b; prefix [experts + 1].
__device__ __forceinline__ int group_at(const long long* prefix, int experts, long long b) {
  int low = 0, high = experts;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (prefix[mid] <= b) low = mid; else high = mid;
  }
  return low;
}

// Each role walks its share's pieces by itself. All of it stays in registers:
// there is no L1 to speak of beside 227 KB of shared memory, so a stack costs
// an L2 access each time.
struct Walk {
  const int* offsets;       // [experts + 1]
  int experts, row_tiles, chunks, n_max;
  Cut cut;                  // of group e
  int e, row_tile, t, lo;   // the next piece
  long long left;           // from its tile's start to the share's end, in cost

  __device__ __forceinline__ void recut(bool flat) {
    cut = cut_group(offsets[e + 1] - offsets[e], n_max, chunks, flat);
  }
  // prefix [experts + 1]: cost before each group; the share is b0 .. b1.
  __device__ __forceinline__ void begin(const long long* prefix, long long b0, long long b1, bool flat) {
    left = 0;
    if (b0 >= b1) return;
    e = group_at(prefix, experts, b0);
    recut(flat);
    const long long tile = static_cast<long long>(chunks) * cut.cost, d = b0 - prefix[e];
    const int item = quotient(d, tile);
    row_tile = cut.tiles == 1 ? item : item / cut.tiles;
    t = item - row_tile * cut.tiles;
    const long long start = prefix[e] + item * tile;
    lo = chunk_at(b0 - start, chunks, cut.cost);
    left = b1 - start;
  }
  __device__ __forceinline__ bool next(Piece* p) {
    if (left <= 0) return false;
    p->lo = lo;
    p->hi = chunk_at(left, chunks, cut.cost);
    if (p->lo >= p->hi) {
      left = 0;
      return false;
    }
    p->e = e;
    p->row_tile = row_tile;
    p->row0 = offsets[e] + t * cut.rows;
    p->rows = min(offsets[e + 1] - p->row0, cut.rows);
    p->n = cut.rows;
    lo = 0;
    left -= static_cast<long long>(chunks) * cut.cost;
    // the tiles of the same weights follow one another: the second reads them
    // from L2
    if (++t == cut.tiles) {
      t = 0;
      if (++row_tile == row_tiles && left > 0) {
        row_tile = 0;
        do ++e; while (e + 1 < experts && offsets[e + 1] == offsets[e]);
        recut(false);  // (a flat share is one tile)
        if (cut.tiles == 0) left = 0;
      }
    }
    return true;
  }
};

// -------------------------------------------------------------- products --

template <bool kFp8, bool kGated>
__global__ void __launch_bounds__(kThreads, 1) grouped_kernel(
    const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1,
    const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const GroupedProblem& p = a.p;
  uint8_t* scale_ring = smem + a.ring;
  int* row_table = reinterpret_cast<int*>(scale_ring + kScaleEntries * scale_entry_bytes(a.n_max));
  Control* ctl = reinterpret_cast<Control*>(scale_ring + scale_ring_bytes(a.n_max));
  long long* bounds = reinterpret_cast<long long*>(ctl + 1);  // [shares + 1] in cost
  long long* prefix = bounds + kMaxShares + 1;                // [experts + 1] cost before each group
  int* offsets = reinterpret_cast<int*>(prefix + p.experts + 1);
  volatile int* abort_flag = &ctl->abort_flag;
  unsigned* err = p.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = p.width / kChunk;
  constexpr int kOuts = kGated ? kTileRows : kTiles * kTileRows;  // of a tile
  const int row_tiles = (p.outs + kOuts - 1) / kOuts;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(&ctl->full[i], 1 + (p.src ? 32 * kRowWarps : 0));  // copies by TMA, row threads
      mbar_init(&ctl->empty[i], kTiles);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->scale_full[i], 32 * kScaleWarps);
      mbar_init(&ctl->scale_empty[i], kTiles);
      mbar_init(&ctl->sum_full[i], kTiles);
      mbar_init(&ctl->sum_empty[i], 32 * kEpiWarps);
    }
    mbar_init(&ctl->fin, kTiles);
    ctl->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kWarpCopy && lane == 0) {
    tma_prefetch_desc(&map0);
    if (kGated) tma_prefetch_desc(&map1);
    tma_prefetch_desc(&xmap);
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&ctl->tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  const int me = blockIdx.x;
  Walk walk;
  walk.offsets = offsets;
  walk.experts = p.experts;
  walk.row_tiles = row_tiles;
  walk.chunks = chunks;
  walk.n_max = a.n_max;
  // The plan. (Its 3 us are mostly code that a block runs once, from beyond the
  // instruction caches; a rehearsal while the kernel before runs only delayed the
  // blocks that start late.)
  if (!a.early) pdl_wait();  // offsets, rows and counters of the kernels before
  // offsets that are out of order or beyond `rows` leave groups empty
  for (int e = threadIdx.x; e <= p.experts; e += kThreads)
    offsets[e] = min(max(__ldcg(p.offsets + e), 0), p.rows);
  __syncthreads();
  // A thread an expert: offsets in ascending order, and how many tiles there are.
  // (One warp took some 4 us for 256 experts.)
  int tiles = 0, widest = 0, tallest = 16;
  for (int e0 = 0, at = 0; e0 <= p.experts; e0 += kThreads) {
    const int e = e0 + threadIdx.x;
    int o = e <= p.experts ? offsets[e] : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, o, s);
      if (lane >= s) o = max(o, u);
    }
    if (lane == 31) ctl->plan[0][warp] = o;
    __syncthreads();
    const int other = lane < kThreads / 32 ? ctl->plan[0][lane] : 0;
    o = max(max(o, at), __reduce_max_sync(0xffffffffu, lane < warp ? other : 0));
    at = max(at, __reduce_max_sync(0xffffffffu, other));
    if (e <= p.experts) offsets[e] = o;
    __syncthreads();
  }
  constexpr int kEach = (kGroupedMaxExperts + 1 + kThreads - 1) / kThreads;
  Cut cuts[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = i * kThreads + threadIdx.x;
    cuts[i] = cut_group(e < p.experts ? offsets[e + 1] - offsets[e] : 0, a.n_max, chunks, false);
    tiles += cuts[i].tiles;
    if (cuts[i].tiles) widest = max(widest, cuts[i].cost);
    tallest = max(tallest, cuts[i].rows);
  }
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  widest = __reduce_max_sync(0xffffffffu, widest);
  tallest = __reduce_max_sync(0xffffffffu, tallest);
  if (lane == 0) {
    ctl->plan[0][warp] = tiles;
    ctl->plan[1][warp] = widest;
    ctl->plan[2][warp] = tallest;
  }
  __syncthreads();
  tiles = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? ctl->plan[0][lane] : 0);
  widest = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? ctl->plan[1][lane] : 0);
  tallest = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? ctl->plan[2][lane] : 0);
  // The ring in stages for the rows that the largest tile has.
  const int stage = stage_bytes(tallest);
  int stages = 2;
  while (stages < kMaxStages && (stages + 1) * stage <= a.ring) ++stages;
  // No more tiles than blocks: a block each, without cuts, where the largest
  // takes no longer than an equal share and the parts' meeting.
  const long long all_tiles = static_cast<long long>(tiles) * row_tiles;
  const bool flat = all_tiles <= a.shares &&
                    widest * chunks * (a.shares - all_tiles) <= static_cast<long long>(kJoin) * a.shares;
  // Cost before each group.
  long long run = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (i * kThreads > p.experts) break;
    const int e = i * kThreads + threadIdx.x;
    const long long mine =
        static_cast<long long>(cuts[i].tiles) * row_tiles * (chunks * (flat ? 1 : cuts[i].cost));
    long long incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += u;
    }
    if (lane == 31) ctl->costs[warp] = incl;
    __syncthreads();
    // (sums of the warps by 26 and by 38 bits)
    const long long other = lane < kThreads / 32 ? ctl->costs[lane] : 0;
    const unsigned low = other & 0x3FFFFFF, high = static_cast<unsigned>(other >> 26);
    auto sum = [&](bool in) {
      return __reduce_add_sync(0xffffffffu, in ? low : 0u) +
             (static_cast<long long>(__reduce_add_sync(0xffffffffu, in ? high : 0u)) << 26);
    };
    const long long before = run + sum(lane < warp);
    run += sum(true);
    if (e <= p.experts) prefix[e] = before + incl - mine;
    __syncthreads();
  }
  // Otherwise shares of a few chunks at least: a cut costs two fp32 parts, their
  // writing, meeting and reading.
  constexpr int kMinChunks = 4;
  const long long most = flat ? all_tiles : run / (kMinChunks * 738);
  const int shares = most < 1 ? 1 : most < a.shares ? static_cast<int>(most) : a.shares;
  const bool snap = all_tiles >= static_cast<long long>(kSnapTiles) * shares;
  __syncthreads();
  // Where each share begins. Shares of many tiles take whole ones.
  for (int c = threadIdx.x; c <= shares; c += kThreads) {
    const long long total = prefix[p.experts];
    long long b = total * c / shares;
    if (snap && c > 0 && c < shares) {
      const int e = group_at(prefix, p.experts, b);
      const Cut g = cut_group(offsets[e + 1] - offsets[e], a.n_max, chunks, flat);
      const long long tile = chunks * g.cost;
      b = prefix[e] + (b - prefix[e] + tile / 2) / tile * tile;
    }
    bounds[c] = b;
  }
  __syncthreads();
  const long long share_end = me < shares ? bounds[me + 1] : 0;
  walk.begin(prefix, me < shares ? bounds[me] : 0, share_end, flat);
  if (a.early) pdl_wait();
  pdl_trigger();
  auto bound = [&](int c) { return bounds[c]; };
  Piece piece;
  auto two_tiles = [&](const Piece& q) {
    return kGated || q.row_tile * kOuts + kTileRows < p.outs;
  };

  if (warp < kEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int side = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int at = quarter * 32 + lane;  // output of a tile
    unsigned uses[2] = {0, 0};           // of each half of the sums' columns
    int half = 0, flip = 0;
    while (true) {
      // where its tile starts and what a chunk of it costs
      const long long start = share_end - walk.left;
      const int cost = walk.cut.cost;
      if (!walk.next(&piece)) break;
      const bool big = piece.n > kHalfN;
      const int blocks = piece.n / kBlockCols;
      // this lane's row of a block: its weight, or its row of out
      auto lane_row = [&](int b) {
        const int r = b * kBlockCols + (lane & 15);
        const bool in = b < blocks && r < piece.rows;
        if (kGated) return in && p.weight ? __float_as_int(p.weight[piece.row0 + r]) : 0x3F800000;
        const int d = !in ? -1 : p.dst ? p.dst[piece.row0 + r] : piece.row0 + r;
        return d < p.out_rows ? d : -1;
      };
      int row_next = lane_row(side);
      const int h = big ? 0 : half;
      const uint32_t sums = tmem + lanes + kSumCol + (big ? 0 : h * (kMaxN));
      const uint32_t sums1 = sums + (big ? kMaxN : kHalfN);
      if (big) {
        wait_bar(&ctl->sum_full[0], uses[0]++ & 1, abort_flag, err);
        wait_bar(&ctl->sum_full[1], uses[1]++ & 1, abort_flag, err);
      } else {
        wait_bar(&ctl->sum_full[h], uses[h]++ & 1, abort_flag, err);
        half ^= 1;
      }
      tc_fence_after();
      auto release = [&] {
        tc_fence_before();
        if (big) {
          mbar_arrive(&ctl->sum_empty[0]);
          mbar_arrive(&ctl->sum_empty[1]);
        } else {
          mbar_arrive(&ctl->sum_empty[h]);
        }
      };
      const bool cut = piece.lo > 0 || piece.hi < chunks;
      const bool second = two_tiles(piece);
      const size_t tile_floats = static_cast<size_t>(a.n_max) * kTileRows;
      auto part_of = [&](int c) {  // share c's part of this tile
        const int slot = bound(c) >= start ? 0 : 1;
        return a.parts + (static_cast<size_t>(c) * 2 + slot) * 2 * tile_floats + at;
      };
      int c0 = me, c1 = me;
      if (cut) {
        float* mine = part_of(me);
#pragma unroll 1
        for (int r = side * 8; r < piece.rows; r += 16) {
          uint32_t r0[8], r1[8];
          tmem_ld8(sums + r, r0);
          tmem_ld8(sums1 + r, r1);  // (not used where there is no second tile)
          tmem_ld_wait8(r0);
          tmem_ld_wait8(r1);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (r + i >= piece.rows) break;
            float* q = mine + static_cast<size_t>(r + i) * kTileRows;
            __stcg(q, __uint_as_float(r0[i]));
            if (second) __stcg(q + tile_floats, __uint_as_float(r1[i]));
          }
        }
        release();
        while (chunk_at(bound(c0) - start, chunks, cost) > 0) --c0;
        while (chunk_at(bound(c1 + 1) - start, chunks, cost) < chunks) ++c1;
        __threadfence();
        bar_sync(1, 32 * kEpiWarps);
        if (threadIdx.x == 0) {
          const int n = piece.hi - piece.lo;
          ctl->last = atomicAdd(a.counters + c0, n) + n == chunks;
          __threadfence();
        }
        bar_sync(1, 32 * kEpiWarps);
        const bool last = *static_cast<volatile int*>(&ctl->last) != 0;
        bar_sync(1, 32 * kEpiWarps);  // read by all before it is written again
        if (!last) continue;
        __threadfence();
      }
      // the sums of 16 rows from r on, this lane's output(s)
      auto take = [&](int r, float (&v0)[16], float (&v1)[16]) {
        if (!cut) {
          tmem_ld16(sums + r, v0);
          tmem_ld16(sums1 + r, v1);
          tmem_ld_wait16(v0, v1);
          return;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) v0[i] = v1[i] = 0.f;
        // the parts added in their order, all of one asked for at once
#pragma unroll 1
        for (int c = c0; c <= c1; ++c) {
          if (chunk_at(bound(c) - start, chunks, cost) >= chunk_at(bound(c + 1) - start, chunks, cost))
            continue;
          const float* q = part_of(c) + static_cast<size_t>(r) * kTileRows;
          float x[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[i] = __ldcg(q + i * kTileRows);  // (what is behind the tile's rows is not used)
            x[16 + i] = second ? __ldcg(q + tile_floats + i * kTileRows) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v0[i] += x[i];
            v1[i] += x[16 + i];
          }
        }
      };
      // (not unrolled, nor in the parts above and below: what a piece runs once has
      // to come from the instruction caches; six blocks' code in a row took 8,000
      // clocks a block)
#pragma unroll 1
      for (int b = side; b < blocks; b += 2) {
        const int row_data = row_next;
        row_next = lane_row(b + 2);
        float v0[16], v1[16];
        take(b * kBlockCols, v0, v1);
        if (kGated) {
          // A row's weight w is the same for all of its outputs, and rounding keeps an
          // order: the block's largest |h| is the largest |silu u| times |w|, and w over
          // the scale, a power of two, is one factor. So an output costs a limit, an
          // exponential, a reciprocal, two products and a maximum. (The hardware's
          // exponential and reciprocal: |h| errs by (10 + 2 |g|) 2^-24 of itself, beside
          // the half step of 2^-4 that follows.)
          const int n = min(kBlockCols, piece.rows - b * kBlockCols);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float g = min_nan(v0[j], p.limit), u = min_nan(max_nan(v1[j], -p.limit), p.limit);
            v0[j] = g * rcp_approx(1.f + ex2_approx(-g * kLog2e)) * u;
            v1[j] = warp_top(v0[j]);
          }
          if (lane == 0) {
            float4* top = reinterpret_cast<float4*>(ctl->top[side][flip][quarter]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              top[j] = make_float4(v1[4 * j], v1[4 * j + 1], v1[4 * j + 2], v1[4 * j + 3]);
          }
          bar_sync(2 + side, 128);
          // lane l of each warp: block's scale of row l
          const float(*tops)[kBlockCols] = ctl->top[side][flip];
          const int l = lane & 15;
          const float w = __int_as_float(row_data);
          const float m = max_nan(max_nan(tops[0][l], tops[1][l]), max_nan(tops[2][l], tops[3][l])) * fabsf(w);
          uint32_t e8 = 255;  // an infinity or NaN makes the block NaN
          float factor = NAN;
          bool huge = false;
          if (m < INFINITY) {
            e8 = __float_as_uint(pow2_scale_448(m)) >> 23;
            const float inv = __uint_as_float((254u - e8) << 23);
            factor = w * inv;
            // w over the scale may pass the largest float where h does not (weights
            // from 8e31 on): the other part then goes to the row's outputs
            huge = fabsf(factor) == INFINITY;
            if (huge) factor = w * 0x1p-64f * inv;
          }
          if (__any_sync(0xffffffffu, huge)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v0[j] *= __shfl_sync(0xffffffffu, huge ? 0x1p64f : 1.f, j);
          }
          if (lane < 16) ctl->factor[side][quarter][l] = factor;
          if (quarter == 0 && lane < n)
            p.hs[static_cast<size_t>(piece.row0 + b * kBlockCols + lane) * (p.outs / kTileRows) +
                 piece.row_tile] = static_cast<uint8_t>(e8);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(&ctl->factor[side][quarter][j]);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              unsigned short t;
              asm("{ .reg .b16 h; cvt.rn.satfinite.e4m3x2.f32 h, %2, %1; mov.b16 %0, h; }"
                  : "=h"(t)
                  : "f"(v0[j + i] * (i ? f.z : f.x)), "f"(v0[j + i + 1] * (i ? f.w : f.y)));
              ctl->codes[side][j + i][at] = static_cast<uint8_t>(t);
              ctl->codes[side][j + i + 1][at] = static_cast<uint8_t>(t >> 8);
            }
          }
          bar_sync(2 + side, 128);
          const int t = (threadIdx.x & 127) >> 3, v = threadIdx.x & 7;
          if (t < n)
            *reinterpret_cast<uint4*>(
                p.hq + static_cast<size_t>(piece.row0 + b * kBlockCols + t) * p.outs +
                piece.row_tile * kTileRows + v * 16) =
                *reinterpret_cast<const uint4*>(&ctl->codes[side][t][v * 16]);
          flip ^= 1;
        } else {
          const int o0 = piece.row_tile * kOuts + at, o1 = o0 + kTileRows;
          const bool in0 = o0 < p.outs, in1 = o1 < p.outs;
          {
            if (a.wide) {
              // BF16, four outputs of a row a lane: pairs of rows as a word, and
              // two exchanges turn rows into outputs (half the time of stores
              // of two bytes a lane)
              const int k = lane & 3;
#pragma unroll
              for (int t = 0; t < kTiles; ++t) {
                const float* v = t ? v1 : v0;
                const int o = (t ? o1 : o0) - k;
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  uint32_t w0 = pack_bf16x2(v[j], v[j + 1]), w1 = pack_bf16x2(v[j + 2], v[j + 3]);
                  // lane 2i: rows j and j + 2 of outputs 2i, 2i + 1; lane 2i + 1: the others
                  const uint32_t x0 = __shfl_xor_sync(0xffffffffu, w0, 1);
                  const uint32_t x1 = __shfl_xor_sync(0xffffffffu, w1, 1);
                  const uint32_t pick = (k & 1) ? 0x3276u : 0x5410u;
                  w0 = __byte_perm(w0, x0, pick);
                  w1 = __byte_perm(w1, x1, pick);
                  // lane 4i + k: row j + (k & 1) + (k & 2) of outputs 4i .. 4i + 3
                  const uint32_t y = __shfl_xor_sync(0xffffffffu, (k & 2) ? w0 : w1, 2);
                  const uint2 word = (k & 2) ? make_uint2(y, w1) : make_uint2(w0, y);
                  const int d = __shfl_sync(0xffffffffu, row_data, j + k);
                  if (d >= 0 && o < p.outs)
                    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + d * p.out_stride + o) = word;
                }
              }
            } else {
              auto put = [&](auto* o, int d, auto x0, auto x1) {
                o += d * p.out_stride;
                if (in0 && d >= 0) o[o0] = x0;
                if (in1 && d >= 0) o[o1] = x1;
              };
              if (p.bf16) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  put(static_cast<__nv_bfloat16*>(p.out), __shfl_sync(0xffffffffu, row_data, j),
                      __float2bfloat16_rn(v0[j]), __float2bfloat16_rn(v1[j]));
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  put(static_cast<float*>(p.out), __shfl_sync(0xffffffffu, row_data, j), v0[j], v1[j]);
              }
            }
          }
        }
      }
      if (!cut) release();
    }
  } else if (warp < kWarpRows) {
    // -------------------------------------------------------------- scales
    // Lane l of each quarter holds outputs (rows) l, 32 + l, ... in
    // consecutive columns; a column's four bytes are a chunk's four groups.
    // They come through a ring in shared memory, four chunks an entry, some
    // ten chunks ahead of their use.
    const int st = threadIdx.x - 32 * kEpiWarps;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool whole = chunks % 4 == 0;
    const uintptr_t off = reinterpret_cast<uintptr_t>(p.ws[0]) |
                          (kGated ? reinterpret_cast<uintptr_t>(p.ws[1]) : 0);
    const bool wide = whole && (off & (kFp8 ? 3 : 15)) == 0;
    const bool x_words = whole && (reinterpret_cast<uintptr_t>(p.xs) & 3) == 0;
    const int entry_bytes = scale_entry_bytes(a.n_max);
    // entries are filled piece after piece, its chunks by fours
    bool more = walk.next(&piece);
    int q = piece.lo / 4;
    unsigned filled = 0;
    int xrow[2];  // rows of x whose scales this thread fetches, -1: none
    auto find_rows = [&] {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = st + i * 32 * kScaleWarps;
        int v = -1;
        if (r < piece.rows) v = p.src ? p.src[piece.row0 + r] : piece.row0 + r;
        xrow[i] = v >= 0 && v < p.x_rows ? v : -1;
      }
    };
    const int blocks128 = (p.outs + kTileRows - 1) / kTileRows;
    auto fetch = [&] {
      if (more) {
        uint8_t* entry = scale_ring + (filled % kScaleEntries) * entry_bytes;
        const int left = min(chunks - 4 * q, 4);  // chunks there are
        if (kFp8) {
          // one block of 128 outputs: the same in every lane
          if (st < kTiles) {
            const int rb = min(piece.row_tile * kTiles + st, blocks128 - 1);
            const uint8_t* from =
                p.ws[0] + (static_cast<size_t>(piece.e) * blocks128 + rb) * chunks + 4 * q;
            if (wide) {
              cp_async4(smem_addr(entry + 4 * st), from);
            } else {
#pragma unroll 1
              for (int c = 0; c < left; ++c) entry[4 * st + c] = from[c];
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const int row = piece.row_tile * kOuts + (kGated ? 0 : t * kTileRows) + st;
            const uint8_t* from =
                p.ws[kGated ? t : 0] +
                (static_cast<size_t>(piece.e) * p.outs + min(row, p.outs - 1)) * (p.width / 32) + 16 * q;
            const uint32_t to = smem_addr(entry + (t * kTileRows + st) * 16);
            if (wide) {
              cp_async16(to, from);
            } else {
#pragma unroll 1
              for (int c = 0; c < left; ++c) cp_async4(to + 4 * c, from + 4 * c);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = st + i * 32 * kScaleWarps;
          if (r >= piece.n) continue;
          uint8_t* to = entry + kScaleBytes + r * 4;
          const uint8_t* from = p.xs + static_cast<size_t>(max(xrow[i], 0)) * chunks + 4 * q;
          if (xrow[i] < 0) {
            *reinterpret_cast<uint32_t*>(to) = 0x7F7F7F7Fu;
          } else if (x_words) {
            cp_async4(smem_addr(to), from);
          } else {
#pragma unroll 1
            for (int c = 0; c < left; ++c) to[c] = from[c];
          }
        }
        ++filled;
        if (++q > (piece.hi - 1) / 4) {
          more = walk.next(&piece);
          q = piece.lo / 4;
          if (more) find_rows();
        }
      }
      cp_async_commit();
    };
    if (more) find_rows();
#pragma unroll 1
    for (int i = 0; i < kScaleEntries - 1; ++i) fetch();
    for (unsigned n = 0; n < filled; ++n) {
      cp_async_wait<kScaleEntries - 2>();
      bar_sync(4, 32 * kScaleWarps);  // all have this entry's copies, and have read the one before
      const uint8_t* entry = scale_ring + (n % kScaleEntries) * entry_bytes;
      const int buf = n & 1;
      // (no break after an abort: the others wait at the barrier above)
      wait_bar(&ctl->scale_empty[buf], ((n >> 1) & 1) ^ 1, abort_flag, err);
      tc_fence_after();
      // (what lies behind a tile's rows or chunks is not used)
      uint32_t v[32] = {};
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (kFp8) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(entry + 4 * t);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[c * 8 + t * 4 + j] = ((u >> (8 * c)) & 0xFFu) * 0x01010101u;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 u = *reinterpret_cast<const uint4*>(entry + (t * kTileRows + j * 32 + lane) * 16);
            v[t * 4 + j] = u.x;
            v[8 + t * 4 + j] = u.y;
            v[16 + t * 4 + j] = u.z;
            v[24 + t * 4 + j] = u.w;
          }
        }
      }
      tmem_st32(tmem + lanes + buf * kScaleCols, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t w = 0;
        if (j * 32 < a.n_max)
          w = *reinterpret_cast<const uint32_t*>(entry + kScaleBytes + (j * 32 + lane) * 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c * 8 + j] = ((w >> (8 * c)) & 0xFFu) * 0x01010101u;
      }
      tmem_st32(tmem + lanes + buf * kScaleCols + 32, v);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&ctl->scale_full[buf]);
      fetch();  // (into the entry before; behind the store, since the first MMA waits for that)
    }
    cp_async_wait<0>();
  } else if (warp < kWarpCopy) {
    // ---------------------------------------------------------------- rows
    // Rows that are not in their order: 16 bytes a thread, eight threads a row,
    // swizzled. (Gathers by TMA take 48 clocks for four rows; bringing the rows into
    // their order first and copying them by TMA, beside the weights, 930 clocks a
    // chunk of 48 rows where this takes 800.) The loop is short and asks for a row's
    // number one copy ahead: with the numbers in registers and the loop unrolled it
    // ran from the second-level instruction cache and took 800 clocks for 16 rows as
    // for 192.
    const int st = threadIdx.x - 32 * kWarpRows;
    const uint8_t* x_from = p.xq + (st & 7) * 16;
    const uint32_t x_to = kTiles * kATile + (st >> 3) * kChunk + (((st & 7) ^ ((st >> 3) & 7)) << 4);
    Piece next;
    int found[2];  // of the next piece, asked for while this one's are copied; -1: zeros
    auto find_rows = [&] {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = st + i * 32 * kRowWarps;
        int v = -1;
        if (r < next.rows) v = p.src[next.row0 + r];
        found[i] = v >= 0 && v < p.x_rows ? v : -1;
      }
    };
    int s = 0, turn = 0;
    uint32_t phase = 1;
    bool good = true, more = p.src && walk.next(&next);
    if (more) find_rows();
    while (more) {
      int* table = row_table + turn * row_table_ints(a.n_max);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (st + i * 32 * kRowWarps < a.n_max) table[st + i * 32 * kRowWarps] = found[i];
      bar_sync(5, 32 * kRowWarps);  // (two tables: nobody is two pieces behind)
      piece = next;
      more = walk.next(&next);
      if (more) find_rows();
      table += st >> 3;
      const uint8_t* from = x_from + piece.lo * kChunk;
#pragma unroll 1
      for (int c = piece.lo; c < piece.hi; ++c) {
        good = good && wait_bar(&ctl->empty[s], phase, abort_flag, err);
        if (good) {
          uint32_t to = smem_addr(smem + s * stage) + x_to;
          int ahead = table[0];
#pragma unroll 1
          for (int r = 16; r <= piece.n; r += 16) {
            const int row = ahead;
            ahead = table[r];  // (one entry of 16 behind the tile's last row)
            cp_async16_or_0(to, from + static_cast<size_t>(max(row, 0)) * p.width, row >= 0);
            to += 16 * kChunk;
          }
          cp_async_arrive(&ctl->full[s]);
        }
        from += kChunk;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
      turn ^= 1;
    }
    cp_async_wait<0>();
  } else if (warp == kWarpCopy) {
    // -------------------------------------------------------------- copies
    if (lane == 0) {
      unsigned n = 0;
      bool good = true;
      int s = 0;
      uint32_t phase = 1;
      while (good && walk.next(&piece)) {
        const bool second = two_tiles(piece);
        // (a tile of E2M1 takes a byte an element in shared memory, but counts
        // with what is read)
        constexpr int kTileTx = kFp8 ? kATile : kATile / 2;
        const int row = piece.row_tile * kOuts;
        const int x_rows = p.src ? 0 : piece.n;
        for (int c = piece.lo; c < piece.hi; ++c) {
          good = wait_bar(&ctl->empty[s], phase, abort_flag, err);
          if (!good) break;
          uint8_t* st = smem + s * stage;
          mbar_arrive_expect_tx(&ctl->full[s], (second ? 2 : 1) * kTileTx + x_rows * kChunk);
          tma_load_3d(st, &map0, c * kChunk, row, piece.e, &ctl->full[s]);
          if (second)
            tma_load_3d(st + kATile, kGated ? &map1 : &map0, c * kChunk,
                        kGated ? row : row + kTileRows, piece.e, &ctl->full[s]);
          for (int r = 0; r < x_rows; r += 16)
            tma_load_2d(st + (kTiles * kTileRows + r) * kChunk, &xmap, c * kChunk, piece.row0 + r,
                        &ctl->full[s]);
          ++n;
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // after an abort: no copy may be under way when the block ends
      if (!good)
        for (unsigned i = n < static_cast<unsigned>(stages) ? 0 : n - stages; i < n; ++i)
          mbar_wait(&ctl->full[i % stages], (i / stages) & 1, err);
    }
    __syncwarp();
  } else if (warp < kWarpMma + kTiles) {
    // ---------------------------------------------------------------- MMAs
    // A thread a tile: what a chunk's waits, operands and commit take of one
    // thread is more than the tensor pipe takes for small tiles.
    if (elect_one()) {
      const int tile = warp - kWarpMma;
      const uint32_t idesc0 = ((kFp8 ? 0u : 5u) << 7) | (1u << 23) | (8u << 24);
      const uint32_t stage_step = stage >> 4;
      const uint32_t base0 = smem_addr(smem) >> 4;
      uint32_t base = base0;  // of the stage, in 16 bytes
      unsigned uses[2] = {0, 0}, scales = 0;
      int half = 0, s = 0;
      uint32_t phase = 0;
      bool good = true;
      while (good && walk.next(&piece)) {
        const bool big = piece.n > kHalfN, mine = tile == 0 || two_tiles(piece);
        const int h = big ? 0 : half;
        if (big) {
          good = wait_bar(&ctl->sum_empty[0], (uses[0]++ & 1) ^ 1, abort_flag, err) &&
                 wait_bar(&ctl->sum_empty[1], (uses[1]++ & 1) ^ 1, abort_flag, err);
        } else {
          good = wait_bar(&ctl->sum_empty[h], (uses[h]++ & 1) ^ 1, abort_flag, err);
          half ^= 1;
        }
        const uint32_t d = tmem + kSumCol + (big ? 0 : h * kMaxN) + tile * (big ? kMaxN : kHalfN);
        const uint32_t idesc = idesc0 | (static_cast<uint32_t>(piece.n >> 3) << 17);
        uint32_t sa = 0;
        for (int c = piece.lo; good && c < piece.hi; ++c) {
          const int buf = scales & 1;
          if (c == piece.lo || (c & 3) == 0) {
            good = mbar_try_wait(&ctl->scale_full[buf], (scales >> 1) & 1) ||
                   wait_bar(&ctl->scale_full[buf], (scales >> 1) & 1, abort_flag, err);
            tc_fence_after();
            sa = tmem + buf * kScaleCols + (c & 3) * 8;
          }
          if (!mbar_try_wait(&ctl->full[s], phase))
            good = good && wait_bar(&ctl->full[s], phase, abort_flag, err);
          if (!good) break;
          fence_async_smem();  // the rows' copies are ordinary writes
          if (mine) {
            const uint32_t at = base + tile * (kATile >> 4), bt = base + kTiles * (kATile >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_scaled(d, at + 2 * k, bt + 2 * k,
                         idesc | (static_cast<uint32_t>(k) << 4) | (static_cast<uint32_t>(k) << 29),
                         sa + tile * 4, sa + 32, k > 0 || c > piece.lo);
          }
          mma_commit(&ctl->empty[s]);
          sa += 8;
          if ((c & 3) == 3 || c + 1 == piece.hi) {
            mma_commit(&ctl->scale_empty[buf]);
            ++scales;
          }
          base += stage_step;
          if (++s == stages) {
            s = 0;
            base = base0;
            phase ^= 1;
          }
        }
        if (!good) break;
        mma_commit(&ctl->sum_full[h]);
        if (big) mma_commit(&ctl->sum_full[1]);
      }
      mma_commit(&ctl->fin);
      mbar_wait(&ctl->fin, 0, err);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
}

__global__ void grouped_reset_kernel(int* counters) {
  pdl_wait();
  pdl_trigger();
  counters[threadIdx.x] = 0;
}

// --------------------------------------------------- routes, tokens' sums --

constexpr int kGroupThreads = 256, kGroupWarps = kGroupThreads / 32;
constexpr int kGroupFew = 64, kGroupAhead = 4, kGroupSlots = 1024, kGroupBlocks = 16;

struct GroupArgs {
  const int* idx;    // [slots]
  const float* wt;   // [slots]
  int slots, topk, lo, experts;
  int* offsets;      // [experts + 1]
  int* slot;         // [slots] sorted by expert, in slot order within one
  int* token;        // [slots] their tokens
  float* weight;     // [slots] their weights
  int* counters;     // two products' [kMaxShares]
};

// A stable counting sort by a cluster of blocks: each warp counts, then places,
// its own stretch of the slots; blocks read one another's counts. (One block
// took 126 us for 49,152 slots.)
__global__ void __launch_bounds__(kGroupThreads) group_kernel(const GroupArgs a) {
  extern __shared__ int count[];  // [kGroupWarps][experts], [experts] of the block
  __shared__ int total[kGroupWarps], before;
  const int rank = blockIdx.x, blocks = gridDim.x;  // one cluster
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* sums = count + kGroupWarps * a.experts;
  for (int i = rank * kGroupThreads + threadIdx.x; i < 2 * kMaxShares; i += blocks * kGroupThreads)
    a.counters[i] = 0;
  if (a.slots <= kGroupFew) {
    // Few slots (one block): each counts those that come before it, and each
    // expert those of the experts before it. (Six slots of 256 experts: 4 us, 6.5
    // by the way below.)
    int e = a.experts;
    if (threadIdx.x < kGroupFew) {
      if (threadIdx.x < a.slots) {
        e = a.idx[threadIdx.x] - a.lo;
        if (e >= a.experts || e < 0) e = a.experts;
      }
      count[threadIdx.x] = e;
    }
    __syncthreads();
    if (e < a.experts) {
      int at = 0;
      for (int j = 0; j < a.slots; ++j) at += count[j] < e || (count[j] == e && j < threadIdx.x);
      a.slot[at] = threadIdx.x;
      a.token[at] = threadIdx.x / a.topk;
      a.weight[at] = a.wt[threadIdx.x];
    }
    for (int x = threadIdx.x; x <= a.experts; x += kGroupThreads) {
      int first = 0;
      for (int j = 0; j < a.slots; ++j) first += count[j] < x;
      a.offsets[x] = first;
    }
    return;
  }
  for (int i = threadIdx.x; i < kGroupWarps * a.experts; i += kGroupThreads) count[i] = 0;
  __syncthreads();
  int* mine = count + warp * a.experts;
  const int warps = blocks * kGroupWarps;
  const int each = (a.slots / 32 + warps) / warps * 32;  // slots of a warp
  const int s0 = min((rank * kGroupWarps + warp) * each, a.slots), s1 = min(s0 + each, a.slots);
  auto walk = [&](auto&& f) {
    for (int base = s0; base < s1; base += 32 * kGroupAhead) {
      int e[kGroupAhead];
#pragma unroll
      for (int i = 0; i < kGroupAhead; ++i) {
        const int s = base + i * 32 + lane;
        e[i] = s < s1 ? a.idx[s] - a.lo : a.experts;
        if (e[i] >= a.experts || e[i] < 0) e[i] = a.experts;  // none of these
      }
#pragma unroll 1
      for (int i = 0; i < kGroupAhead && base + i * 32 < s1; ++i) {
        const int x = i == 0 ? e[0] : i == 1 ? e[1] : i == 2 ? e[2] : e[3];
        // the lanes with this lane's expert
        unsigned same = 0xffffffffu;
        for (int b = 1; b <= a.experts; b <<= 1) {
          const unsigned set = __ballot_sync(0xffffffffu, x & b);
          same &= (x & b) ? set : ~set;
        }
        const int first = __ffs(same) - 1;
        int at = 0;
        if (lane == first && x < a.experts) {
          at = mine[x];
          mine[x] = at + __popc(same);
        }
        at = __shfl_sync(0xffffffffu, at, first) + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (x < a.experts) f(base + i * 32 + lane, at);
      }
    }
  };
  walk([](int, int) {});
  __syncthreads();
  // this block's counts, and its warps' places in them
  for (int e = threadIdx.x; e < a.experts; e += kGroupThreads) {
    int sum = 0;
    for (int w = 0; w < kGroupWarps; ++w) {
      const int c = count[w * a.experts + e];
      count[w * a.experts + e] = sum;
      sum += c;
    }
    sums[e] = sum;
  }
  if (threadIdx.x == 0) before = 0;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // first places: over the experts, and the blocks before this one
  for (int e0 = 0; e0 < a.experts; e0 += kGroupThreads) {
    const int e = e0 + threadIdx.x;
    int all = 0, earlier = 0;
    if (e < a.experts)
      for (int r = 0; r < blocks; ++r) {
        uint32_t from;
        int c;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(smem_addr(sums + e)), "r"(r));
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(from) : "memory");
        if (r < rank) earlier += c;
        all += c;
      }
    int incl = all;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += u;
    }
    if (lane == 31) total[warp] = incl;
    __syncthreads();
    int first = before + incl - all;
    for (int w = 0; w < warp; ++w) first += total[w];
    __syncthreads();
    if (threadIdx.x == kGroupThreads - 1) before = first + all;
    if (e < a.experts) {
      if (rank == 0) {
        a.offsets[e] = first;
        if (e == a.experts - 1) a.offsets[a.experts] = first + all;
      }
      for (int w = 0; w < kGroupWarps; ++w) count[w * a.experts + e] += first + earlier;
    }
    __syncthreads();
  }
  walk([&](int s, int at) {
    a.slot[at] = s;
    a.token[at] = s / a.topk;
    a.weight[at] = a.wt[s];
  });
  // until then the others read this block's counts
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// out[t] = the sum of the token's slots in route order; slots of experts that
// are not here were not written. The slots are BF16, which is what a GEMV of
// the layer hands on; their sum is fp32 and rounded once. Bound by their reading:
// 8,192 tokens of six 93 us, 5.0 TB/s.
__global__ void __launch_bounds__(256) experts_combine_kernel(const uint16_t* __restrict__ y,
                                                              const int* __restrict__ idx, int n, int topk,
                                                              int hidden, int lo, int experts,
                                                              uint16_t* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  const int vecs = hidden / 8;
  const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  if (i >= static_cast<long long>(n) * vecs) return;
  const int t = static_cast<int>(i / vecs), v = static_cast<int>(i % vecs);
  float sum[8] = {};
  for (int k0 = 0; k0 < topk; k0 += 8) {
    uint4 r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[k] = make_uint4(0, 0, 0, 0);
      if (k0 + k < topk)  // (before it is known whether it was written)
        r[k] = __ldcs(
            reinterpret_cast<const uint4*>(y + (static_cast<size_t>(t) * topk + k0 + k) * hidden) + v);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = k0 + k < topk ? idx[t * topk + k0 + k] - lo : -1;
      if (e < 0 || e >= experts) r[k] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[2 * j] += __uint_as_float(w[j] << 16);
        sum[2 * j + 1] += __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
  reinterpret_cast<uint4*>(out + static_cast<size_t>(t) * hidden)[v] =
      make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]),
                 pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
}

// ------------------------------------------------------------------ host --

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms < kMaxShares ? sms : kMaxShares;
}

int tile_rows(const GroupedProblem& p) {
  const long long rows = p.rows, each = p.experts;  // rows <= k each: k of a group on average
  const int outs = p.w[1] ? kTileRows : kTiles * kTileRows;
  // Rows of a tile. Small ones leave more of the parts' memory unused and more of
  // the ring to stages (256 experts of 4096 x 2048: 100 tokens 515 us with 16, 522
  // with 32; 500 tokens 578 with 32, 601 with 96). Beyond 96 the sums fill TMEM and
  // the epilogue is not overlapped, which long sums of large groups make up for
  // (8,192 tokens 2162 us with 192, 2216 with 96; 2,000 tokens, uneven, 913 and 929),
  // others not (1,500 tokens 741, 693 with 96; 2048 rows of 1024 columns 135, 127
  // with 96).
  int n_max = rows <= 8 * each ? 16 : rows <= 24 * each ? 32 : kHalfN;
  if (rows > 40 * each && p.width >= 24 * kChunk) n_max = kMaxN;
  // Fewer where there would be too few tiles: to cut one along its columns costs
  // more (777 rows of 24 groups, 1003 outputs: 17.4 us with 32, 19.9 with 96)
  const long long row_tiles = (p.outs + outs - 1) / outs;
  while (n_max > 32 && row_tiles * ((rows + n_max - 1) / n_max) < 2ll * sm_count())
    n_max = n_max > kHalfN ? kHalfN : 32;
  return n_max;
}

size_t parts_bytes(const GroupedProblem& p) {
  return static_cast<size_t>(sm_count()) * 4 * tile_rows(p) * kTileRows * sizeof(float);
}

constexpr size_t kCounterBytes = kMaxShares * sizeof(int);

bool weight_map(CUtensorMap* m, const GroupedProblem& p, const uint8_t* w) {
  if (p.fp8)
    return make_tma_map_u8_3d(m, w, p.width, p.outs, p.width, p.experts,
                              static_cast<uint64_t>(p.outs) * p.width, kChunk, kTileRows, 1);
  return make_tma_map_u4_3d(m, w, p.width, p.outs, p.experts, kTileRows);
}

cudaError_t launch(const GroupedProblem& p, bool early, int* counters, float* parts, cudaStream_t st) {
  const bool gated = p.w[1] != nullptr;
  CUtensorMap map0, map1, xmap;
  if (!weight_map(&map0, p, p.w[0]) || !weight_map(&map1, p, gated ? p.w[1] : p.w[0]) ||
      !make_tma_map_u8(&xmap, p.xq, p.width, p.x_rows, kChunk, 16, true, false))
    return cudaErrorInvalidValue;
  Args a;
  a.p = p;
  a.early = early;
  a.shares = sm_count();
  a.n_max = tile_rows(p);
  a.ring = static_cast<int>((kMaxSmem - rest_bytes(a.n_max, p.experts)) & ~static_cast<size_t>(1023));
  a.wide = p.bf16 && p.outs % 4 == 0 && p.out_stride % 4 == 0 &&
           reinterpret_cast<uintptr_t>(p.out) % 8 == 0;
  a.counters = counters;
  a.parts = parts;
  if (a.shares < 1) return cudaErrorInvalidDevice;
  if (gated && p.fp8) return cudaErrorInvalidValue;
  auto kernel = gated ? grouped_kernel<false, true>
                      : p.fp8 ? grouped_kernel<true, false> : grouped_kernel<false, false>;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), static_cast<int>(kMaxSmem));
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(a.shares), dim3(kThreads),
                    a.ring + rest_bytes(a.n_max, p.experts), st, map0, map1, xmap, a);
}

// Pieces of a buffer, 256-byte aligned.
struct Carver {
  char* at;
  size_t used = 0;
  template <class T>
  T* take(size_t n) {
    T* p = reinterpret_cast<T*>(at + used);
    used += (n * sizeof(T) + 255) & ~static_cast<size_t>(255);
    return p;
  }
};

struct ExpertsWork {
  int *counters, *offsets, *slot, *token;
  float *weight, *parts;
  uint8_t *hq, *hs;
  uint16_t* y;
  size_t bytes;
};

GroupedProblem gate_up(const ExpertsProblem& p, const ExpertsWork& w) {
  GroupedProblem g;
  g.experts = p.experts;
  g.rows = p.n * p.topk;
  g.outs = p.inter;
  g.width = p.hidden;
  g.w[0] = p.w1; g.ws[0] = p.s1;
  g.w[1] = p.w3; g.ws[1] = p.s3;
  g.xq = p.xq;
  g.xs = p.xs;
  g.x_rows = p.n;
  g.offsets = w.offsets;
  g.src = w.token;
  g.limit = p.limit;
  g.weight = w.weight;
  g.hq = w.hq;
  g.hs = w.hs;
  g.err = p.err;
  return g;
}

GroupedProblem down(const ExpertsProblem& p, const ExpertsWork& w) {
  GroupedProblem d;
  d.experts = p.experts;
  d.rows = p.n * p.topk;
  d.outs = p.hidden;
  d.width = p.inter;
  d.w[0] = p.w2;
  d.ws[0] = p.s2;
  d.xq = w.hq;
  d.xs = w.hs;
  d.x_rows = d.rows;
  d.offsets = w.offsets;
  d.dst = w.slot;
  d.out_rows = d.rows;
  d.out = w.y;
  d.out_stride = p.hidden;
  d.err = p.err;
  return d;
}

ExpertsWork experts_work(const ExpertsProblem& p, void* base) {
  Carver c{static_cast<char*>(base)};
  const size_t slots = static_cast<size_t>(p.n) * p.topk;
  ExpertsWork w;
  w.counters = c.take<int>(2 * kMaxShares);
  w.offsets = c.take<int>(p.experts + 1);
  w.slot = c.take<int>(slots);
  w.token = c.take<int>(slots);
  w.weight = c.take<float>(slots);
  w.hq = c.take<uint8_t>(slots * p.inter);
  w.hs = c.take<uint8_t>(slots * (p.inter / 128));
  w.y = c.take<uint16_t>(slots * p.hidden);
  // (either product may have the larger tiles)
  const size_t parts[2] = {parts_bytes(gate_up(p, w)), parts_bytes(down(p, w))};
  w.parts = c.take<float>((parts[0] > parts[1] ? parts[0] : parts[1]) / sizeof(float));
  w.bytes = c.used;
  return w;
}

}  // namespace

size_t grouped_workspace_bytes(const GroupedProblem& p) {
  return kCounterBytes + parts_bytes(p);
}

cudaError_t grouped_reset(void* ws, cudaStream_t st) {
  return launch_pdl(grouped_reset_kernel, dim3(1), dim3(kMaxShares), 0, st, static_cast<int*>(ws));
}

cudaError_t grouped_forward(const GroupedProblem& p, void* ws, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  return launch(p, false, static_cast<int*>(ws),
                reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes), st);
}

size_t experts_workspace_bytes(const ExpertsProblem& p) { return experts_work(p, nullptr).bytes; }

cudaError_t experts_forward(const ExpertsProblem& p, void* ws, cudaStream_t st) {
  if (p.n <= 0) return cudaSuccess;
  const ExpertsWork w = experts_work(p, ws);
  GroupArgs a;
  a.idx = p.idx;
  a.wt = p.wt;
  a.slots = p.n * p.topk;
  a.topk = p.topk;
  a.lo = p.lo;
  a.experts = p.experts;
  a.offsets = w.offsets;
  a.slot = w.slot;
  a.token = w.token;
  a.weight = w.weight;
  a.counters = w.counters;
  const void* group = reinterpret_cast<const void*>(group_kernel);
  cudaError_t e = set_max_dynamic_smem(
      group, static_cast<int>(sizeof(int)) * (kGroupWarps + 1) * kGroupedMaxExperts);
  int blocks = 1;
  while (blocks < kGroupBlocks && a.slots > blocks * kGroupSlots) blocks *= 2;
  if (e == cudaSuccess && blocks > 8)  // more than every device has to take
    e = cudaFuncSetAttribute(group, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  prefer_max_shared(group);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kGroupThreads);
  cfg.dynamicSmemBytes = sizeof(int) * (kGroupWarps + 1) * (p.experts > kGroupFew ? p.experts : kGroupFew);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(blocks), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, group_kernel, a);
  if (e != cudaSuccess) return e;
  e = launch(gate_up(p, w), false, w.counters, w.parts, st);
  if (e != cudaSuccess) return e;
  e = launch(down(p, w), true, w.counters + kMaxShares, w.parts, st);
  if (e != cudaSuccess) return e;
  const long long vecs = static_cast<long long>(p.n) * (p.hidden / 8);
  return launch_pdl(experts_combine_kernel, dim3(static_cast<unsigned>((vecs + 255) / 256)), dim3(256),
                    0, st, static_cast<const uint16_t*>(w.y), p.idx, p.n, p.topk, p.hidden, p.lo,
                    p.experts, p.out);
}

}  // namespace dsv4
