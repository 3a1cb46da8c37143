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
#include <type_traits>
#include <cuda_bf16.h>

#include "attn.cuh"
#include "bulk.cuh"
#include "dsv4_common.cuh"
#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

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

// The first position that a token at `pos` sees. (No difference is formed that
// could leave the range of an int, whatever the window.)
__device__ __forceinline__ int seen_from(int window, int pos) {
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}

// Positions of a slot; what is not a length counts as none.
__device__ __forceinline__ int slot_length(const PagedLayer& c, int s) { return max(c.length[s], 0); }

__device__ __forceinline__ float load_q(const PagedAttnProblem& p, long long at) {
  return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[at])
                : bf16_round(static_cast<const float*>(p.q)[at]);
}
__device__ __forceinline__ void store_out(const PagedAttnProblem& p, long long at, float v) {
  if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(p.out)[at] = __bfloat162float(__float2bfloat16_rn(v));
}

// ========================================================== general path ==
//
// For shapes that the tensor-core kernel does not take: a block per token, 8
// or 16 heads and a piece of the keys, in fp32. 32 keys at a time are decoded
// to BF16 (what the cache's values round to) in shared memory, once for all
// heads of the block; then a lane has a key for the scores and two neighbouring
// dims of each 64 for the sums, a warp one head or two. The pieces are a
// cluster's blocks, which merge through one another's shared memory, each
// some of the heads. Shared-memory reads and FMAs of few warps bound it: 64
// heads of 576 dims on 2048 keys take 100 us for one token (1.7 ms with a
// block per head that decodes its own keys), 1.29 ms for 64 (21.7 ms).
constexpr int kMaxDim = 1024;
constexpr int kGenWarps = 8;
constexpr int kGenThreads = 32 * kGenWarps;
constexpr int kGenKeys = 32;       // of a step
constexpr int kGenParts = 8;       // at most, of a token's keys

// Words of a decoded key: odd, so that lanes on 32 keys meet 32 banks.
__host__ __device__ inline int gen_pitch(int d) { return (d / 2) | 1; }

__device__ __forceinline__ uint32_t in_part(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_part(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_part2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void all_parts() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" :::
                   "memory");
}

// One of two BF16 values is a NaN or an infinity.
__device__ __forceinline__ bool special2(uint32_t w) {
  return (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) != 0;
}

// kHeads: of a warp; kWords: pairs of dims of a lane, dim <= 64 kWords.
template <int kHeads, int kWords>
__global__ void __launch_bounds__(kGenThreads) paged_attn_general_kernel(
    const __grid_constant__ PagedAttnProblem p, int parts) {
  constexpr int kBlockHeads = kGenWarps * kHeads;
  extern __shared__ __align__(16) float sm_q[];  // [kBlockHeads][d]: q, at the end the sums
  __shared__ float sm_m[kBlockHeads], sm_den[kBlockHeads];
  __shared__ int sm_row[kGenKeys];
  __shared__ unsigned sm_there, sm_broken;
  __shared__ float sm_bad;
  const PagedLayer& c = p.pages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / parts, part = blockIdx.x % parts, head0 = blockIdx.y * kBlockHeads;
  const int d = c.nope + c.rope_dim, words = d / 2, pitch = gen_pitch(d);
  uint32_t* sm_k = reinterpret_cast<uint32_t*>(sm_q + kBlockHeads * d);
  const int s = slot_of(p.q_start, c.n_seqs, row);
  if (s < 0) return;  // (the whole cluster)
  const int len = slot_length(c, s), end = p.q_start[s + 1];
  const bool beyond = end - p.q_start[s] > p.max_new || len > p.max_len;
  if (beyond && tid == 0 && c.status) atomicOr(c.status, kPagedBounds);
  const int self = len - end + row;  // the token's position
  const int first = seen_from(p.window, self);
  const int last = min(self, c.max_pages * c.page - 1);
  const int steps = beyond || last < first ? 0 : (last - first) / kGenKeys + 1;
  const int step0 = static_cast<int>(static_cast<long long>(steps) * part / parts);
  const int step1 = static_cast<int>(static_cast<long long>(steps) * (part + 1) / parts);
  for (int hl = warp * kHeads; hl < (warp + 1) * kHeads; ++hl)  // read by this warp alone
    for (int i = lane; i < d; i += 32)
      sm_q[hl * d + i] = head0 + hl < p.H
                             ? load_q(p, row * p.q_stride + static_cast<long long>(head0 + hl) * d + i)
                             : 0.f;
  const int* table = c.table + static_cast<size_t>(s) * c.max_pages;
  const int units = c.nope / 16, pairs = c.rope_dim / 2;  // of a key
  const bool idle = head0 + warp * kHeads >= p.H;
  bool bad = beyond;
  float m[kHeads], den[kHeads], o[kHeads][2 * kWords];  // den: this lane's keys
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    m[i] = -INFINITY;
    den[i] = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * kWords; ++u) o[i][u] = 0.f;
  }
  // the cache row of this lane's key of a step, -1: none
  auto find_row = [&](int step) {
    const unsigned t = static_cast<unsigned>(first) + step * kGenKeys + lane;
    if (step >= step1 || t > static_cast<unsigned>(last)) return -1;
    const int page = table[static_cast<int>(t) / c.page];
    return page >= 0 && page < c.n_pages ? page * c.page + static_cast<int>(t) % c.page : -1;
  };
  int next_row = warp == 0 ? find_row(step0) : -1;
  constexpr int kAhead = 4;  // loads of a thread on their way together
  for (int step = step0; step < step1; ++step) {
    __syncthreads();  // the keys before have been used
    if (warp == 0) {
      sm_row[lane] = next_row;
      const unsigned there = __ballot_sync(0xffffffffu, next_row >= 0);
      if (lane == 0) {
        sm_there = there;
        sm_broken = 0;
      }
    }
    __syncthreads();
    if (warp == 0) next_row = find_row(step + 1);
    // 16 codes at a time
    for (int i0 = tid; i0 < kGenKeys * units; i0 += kAhead * kGenThreads) {
      uint4 v[kAhead];
      uint32_t scale[kAhead];
      int at[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * kGenThreads, k = i / units, u = i - k * units;
        const int r = i < kGenKeys * units ? sm_row[k] : -1;
        at[x] = i < kGenKeys * units ? (k << 16) | u : -1;
        v[x] = make_uint4(0, 0, 0, 0);
        scale[x] = 127;
        if (r >= 0) {
          v[x] = __ldg(reinterpret_cast<const uint4*>(c.codes + static_cast<size_t>(r) * c.nope) + u);
          scale[x] = __ldg(c.scales + static_cast<size_t>(r) * kKvScaleSlots + u / 4);
        }
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        if (at[x] < 0) continue;
        const int k = at[x] >> 16, u = at[x] & 0xFFFF;
        const float f = e8m0_decode(scale[x]);
        const uint2 w[4] = {e4m3x4_to_bf16(v[x].x, f), e4m3x4_to_bf16(v[x].y, f),
                            e4m3x4_to_bf16(v[x].z, f), e4m3x4_to_bf16(v[x].w, f)};
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          odd = odd || special2(w[j].x) || special2(w[j].y);
          sm_k[k * pitch + 8 * u + 2 * j] = w[j].x;
          sm_k[k * pitch + 8 * u + 2 * j + 1] = w[j].y;
        }
        if (odd) atomicOr(&sm_broken, 1u << k);
      }
    }
    for (int i0 = tid; i0 < kGenKeys * pairs; i0 += kAhead * kGenThreads) {
      uint32_t v[kAhead];
      int at[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * kGenThreads, k = i / pairs, j = i - k * pairs;
        const int r = i < kGenKeys * pairs ? sm_row[k] : -1;
        at[x] = i < kGenKeys * pairs ? (k << 16) | j : -1;
        v[x] = r < 0 ? 0u
                     : __ldg(reinterpret_cast<const uint32_t*>(
                                 c.rope + static_cast<size_t>(r) * c.rope_dim) + j);
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        if (at[x] < 0) continue;
        const int k = at[x] >> 16;
        sm_k[k * pitch + c.nope / 2 + (at[x] & 0xFFFF)] = v[x];
        if (special2(v[x])) atomicOr(&sm_broken, 1u << k);
      }
    }
    __syncthreads();
    if (sm_broken) bad = true;  // every key of these is visible
    const unsigned use = sm_there & ~sm_broken;
    if (use == 0 || idle) continue;
    float w[kHeads];
    {
      float acc[kHeads][2] = {};
      const uint32_t* kr = sm_k + lane * pitch;
      const float2* q = reinterpret_cast<const float2*>(sm_q + warp * kHeads * d);
#pragma unroll 8
      for (int j = 0; j < words; ++j) {
        const uint32_t kw = kr[j];
        const float x = __uint_as_float(kw << 16), y = __uint_as_float(kw & 0xFFFF0000u);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const float2 qv = q[i * words + j];
          acc[i][0] = fmaf(qv.x, x, acc[i][0]);
          acc[i][1] = fmaf(qv.y, y, acc[i][1]);
        }
      }
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const float x = (use >> lane) & 1u ? (acc[i][0] + acc[i][1]) * p.scale : -INFINITY;
        const float mx = fmaxf(m[i], warp_max(x));
        const float a = m[i] == -INFINITY ? 0.f : expf(m[i] - mx);
        w[i] = x == -INFINITY ? 0.f : expf(x - mx);
        den[i] = den[i] * a + w[i];
        if (a != 1.f) {
#pragma unroll
          for (int u = 0; u < 2 * kWords; ++u) o[i][u] *= a;
        }
        m[i] = mx;
      }
    }
#pragma unroll 2
    for (int k = 0; k < kGenKeys; ++k) {
      float wk[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) wk[i] = __shfl_sync(0xffffffffu, w[i], k);
      if (!((use >> k) & 1u)) continue;  // (may hold a NaN)
      const uint32_t* kr = sm_k + k * pitch;
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
        const int j = lane + 32 * u;
        const uint32_t kw = j < words ? kr[j] : 0u;
        const float x = __uint_as_float(kw << 16), y = __uint_as_float(kw & 0xFFFF0000u);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          o[i][2 * u] = fmaf(wk[i], x, o[i][2 * u]);
          o[i][2 * u + 1] = fmaf(wk[i], y, o[i][2 * u + 1]);
        }
      }
    }
  }
  // each part's sums where its q was
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int hl = warp * kHeads + i;
    float sum = den[i];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) {
      sm_m[hl] = m[i];
      sm_den[hl] = sum;
    }
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const int j = lane + 32 * u;
      if (j < words)
        reinterpret_cast<float2*>(sm_q + hl * d)[j] = make_float2(o[i][2 * u], o[i][2 * u + 1]);
    }
  }
  if (tid == 0) sm_bad = bad ? 1.f : 0.f;
  all_parts();
  const int r0 = d - p.rope_out;
  for (int hl = part + parts * warp; hl < kBlockHeads; hl += parts * kGenWarps) {
    const int h = head0 + hl;
    if (h >= p.H) break;
    float pm = -INFINITY, pden = 0.f, pbad = 0.f;  // lane: part
    if (lane < parts) {
      pm = ld_part(in_part(&sm_m[hl], lane));
      pden = ld_part(in_part(&sm_den[hl], lane));
      pbad = ld_part(in_part(&sm_bad, lane));
    }
    const float sink = p.sink ? p.sink[h] : -INFINITY;
    const float M = fmaxf(warp_max(pm), sink);
    const float f = pm == -INFINITY ? 0.f : expf(pm - M);
    float total = pden * f;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    if (sink != -INFINITY) total += expf(sink - M);
    const bool nan = __any_sync(0xffffffffu, pbad != 0.f);
    const float inv = nan ? NAN : total == 0.f ? 0.f : 1.f / total;
    for (int j = lane; j < ((words + 31) & ~31); j += 32) {
      float x0 = 0.f, x1 = 0.f;
      for (int q = 0; q < parts; ++q) {
        const float fq = __shfl_sync(0xffffffffu, f, q);
        if (j < words) {
          const float2 v = ld_part2(in_part(sm_q + hl * d + 2 * j, q));
          x0 = fmaf(v.x, fq, x0);
          x1 = fmaf(v.y, fq, x1);
        }
      }
      if (j >= words) continue;
      x0 *= inv;
      x1 *= inv;
      if (p.rope_cos && 2 * j >= r0) {
        const long long at = static_cast<long long>(row) * (p.rope_out / 2) + (2 * j - r0) / 2;
        const float cs = p.rope_cos[at], sn = p.rope_sin[at];
        const float y0 = x0 * cs + x1 * sn, y1 = x1 * cs - x0 * sn;
        x0 = y0;
        x1 = y1;
      }
      const long long at = row * p.out_stride + static_cast<long long>(h) * d + 2 * j;
      store_out(p, at, x0);
      store_out(p, at + 1, x1);
    }
    if (p.lse && lane == 0)
      p.lse[static_cast<size_t>(row) * p.H + h] = nan ? NAN : total == 0.f ? -INFINITY : M + logf(total);
  }
  all_parts();  // nobody leaves while its sums are read
}

// ===================================================== tensor-core path ==
//
// Three launches. (1) The latents that any new token sees are decoded once
// into BF16 rows, sequence after sequence, each padded to whole blocks of 64
// keys (a prompt's chunk reads them hundreds of times; pages, freed pages
// and broken rows are dealt with here alone), and one block lists the tiles:
// 128 (token, head) rows of one sequence, with the key blocks they see.
// (2) The (tile, key block) pairs, laid end to end, are cut into equal
// shares, one per pair of CTAs, whatever the lengths of the sequences; the
// two CTAs of a pair accumulate 256 output dims each, because 128 rows of 512
// fp32 sums fill all of TMEM. A tile inside one share is finished there.
// (3) Tiles cut by a share's end are merged from their fp32 parts.

constexpr int kD = 512, kNope = 448, kRope = 64;
constexpr int kRows = 128;        // (token, head) rows of a tile: M of both products
constexpr int kKeys = 64;         // keys of a block: N of Q K^T, K of P V
constexpr int kHalf = 256;        // output dims of a CTA: N of P V
// What a tile costs besides its blocks (Q in, O out), in blocks: shares are
// cut by the sum, so that many short tiles weigh as much as a long one (2000
// tiles of three blocks: 189 us, 251 where a tile costs nothing, 186 at 8; 8
// sequences of 3 tiles of 32 to 63 blocks: 47.7, 50.1 and 49.4).
constexpr int kTileCost = 4;
// A smaller share costs more to merge than it saves (one tile of 32 blocks:
// 20.7 us, 22.8 with shares from one unit on, 22.0 from four).
constexpr int kMinShare = 2;
// The weights of P V are BF16, each off by up to 2^-8 of itself. Their sum as
// P V takes them is kept next to the exact one, and O is multiplied by the
// ratio: then what is left of the roundings is sum p_t d_t (v_t - o), |d_t| <=
// 2^-8, which is nothing where one key has the row, whatever its weight (up
// to 2^8: the running maximum lags), and averages out where many keys share
// it. lse takes the exact sum. (A sum more in the softmax: 2048 tokens on 11987
// keys 3684 us, 3640 with the weights off by their rounding.) Where a row sees
// few keys that is not enough: a tile of at most this many blocks carries its
// weights in two BF16 terms. Twice the MMAs of P V there do not show (2000 tiles
// of three blocks in the kernel that has both: 199 us with one term or two).
constexpr int kTwoTermBlocks = 4;
constexpr float kLazyMargin = 8.0f;  // log2 units: the running max moves only past this

struct Tile {
  long long start;  // units of the tiles before: kTileCost and the blocks of each
  int blocks;       // blocks that its tokens see
  int block0;       // first of them among the decoded blocks
  int key0;         // position of that block's first key
  int row0;         // first row of q
  int tokens;       // <= 128 / H
  int pos0;         // position of its first token
  int bad;          // beyond the caller's bounds: NaN
  int pad[3];
};
static_assert(sizeof(Tile) == 48, "one warp reads a tile's description in one go");

struct PlanHead {
  long long total;  // units of all tiles
  long long share;  // units per pair of CTAs
  int tiles;
};

struct TcWs {
  PlanHead* head;
  Tile* tiles;
  Tile* first_tile;       // [pairs] the tile that a share starts in
  uint8_t* valid;         // [blocks][8] a bit per key
  uint8_t* broken;        // [blocks][8] keys with a NaN or infinity (decoded as zeros)
  float* part_m;          // [pairs][2][2 halves][128] log2 units
  float* part_den;
  float* part_back;       // what the part's O is multiplied by
  float* part_o;          // [pairs][2][128][512]
  __nv_bfloat16* stage;   // [blocks * 64][512]
};

struct TcShape {
  int tile_cap, tokens_per_tile, pairs;
  long long block_cap;
};

struct TcCall {
  PagedAttnProblem p;
  TcShape s;
  TcWs w;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b > 0); }

// One slot's new tokens and the positions they see.
struct Slot {
  int row0, tokens, len, first, klo, blocks, tiles;
  bool bad;
};

__device__ __forceinline__ Slot slot_geometry(const PagedAttnProblem& p, int tokens_per_tile,
                                              int s) {
  Slot g;
  g.row0 = p.q_start[s];
  const int end = p.q_start[s + 1];
  g.len = slot_length(p.pages, s);
  const bool rows_ok = g.row0 >= 0 && end >= g.row0 && end <= p.total;
  g.tokens = rows_ok ? end - g.row0 : 0;
  g.bad = g.tokens > 0 && (g.tokens > p.max_new || g.len > p.max_len);
  if (!rows_ok || g.bad) {
    if (p.pages.status) atomicOr(p.pages.status, kPagedBounds);
  }
  g.first = g.len - g.tokens;
  g.klo = seen_from(p.window, g.first);
  g.tiles = ceil_div(g.tokens, tokens_per_tile);
  g.blocks = g.tokens == 0 ? 0 : g.bad ? 1 : max(1, ceil_div(max(0, g.len - g.klo), kKeys));
  return g;
}

constexpr int kStageThreads = 256;
constexpr int kStageBlocks = 3;     // of an SM: their loads are what keeps the memory busy
constexpr int kUnit = 8;            // rows that a warp decodes together

// Exclusive prefix sum over the block; *total = the sum.
__device__ int stage_scan(int v, int* total) {
  __shared__ int part[kStageThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kStageThreads / 32; ++w) {
    if (w < warp) before += part[w];
    sum += part[w];
  }
  *total = sum;
  return before + incl - v;
}

// Whole block: the tiles of all slots.
__device__ void list_tiles(const TcCall& c, const int* block_start, const int* tile_start) {
  const PagedAttnProblem& p = c.p;
  const int n_seqs = p.pages.n_seqs, per = c.s.tokens_per_tile;
  const int tiles = min(tile_start[n_seqs], c.s.tile_cap);
  if (tile_start[n_seqs] > c.s.tile_cap && threadIdx.x == 0 && p.pages.status)
    atomicOr(p.pages.status, kPagedBounds);
  long long done = 0;
  for (int base = 0; base < tiles; base += kStageThreads) {
    const int t = base + threadIdx.x;
    Tile tile = {};
    if (t < tiles) {
      int lo = 0, hi = n_seqs;  // the last slot with tile_start <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      // slots without tokens share their start with the next one
      const Slot g = slot_geometry(p, per, lo);
      const int i0 = (t - tile_start[lo]) * per;
      tile.tokens = min(per, g.tokens - i0);
      tile.row0 = g.row0 + i0;
      tile.pos0 = g.first + i0;
      tile.bad = g.bad || block_start[lo] + g.blocks > c.s.block_cap;
      if (tile.bad) {
        tile.blocks = 1;
        if (p.pages.status) atomicOr(p.pages.status, kPagedBounds);
      } else {
        const int from = seen_from(p.window, tile.pos0);
        const int b0 = min(max(0, from - g.klo) / kKeys, g.blocks - 1);
        const int b1 = min(max(ceil_div(max(0, tile.pos0 + tile.tokens - g.klo), kKeys), b0 + 1),
                           g.blocks);
        tile.blocks = b1 - b0;
        tile.block0 = block_start[lo] + b0;
        tile.key0 = g.klo + b0 * kKeys;
      }
    }
    int total;
    tile.start = done + stage_scan(t < tiles ? tile.blocks + kTileCost : 0, &total);
    if (t < tiles) c.w.tiles[t] = tile;
    done += total;
  }
  if (threadIdx.x == 0) {
    const long long pairs = c.s.pairs;
    long long share = (done + pairs - 1) / pairs;
    if (share < kMinShare) share = kMinShare;
    *c.w.head = {done, share, tiles};
  }
}

__device__ __forceinline__ void st_global_32(void* p, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x),
               "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// Latents to BF16 rows: a warp per 8 rows, no barriers. Lane l has the dims
// 16 l .. 16 l + 15 of each: 16 codes, or (lanes 28-31) the first 8 of 16 RoPE
// values, whose other 8 are lane 4 r + (l - 28)'s for row r. All loads of the
// 8 rows are on their way before the first is used; a row's codes leave as
// whole sectors.
// Memory bounds it: 147k rows (86 MB read, 151 MB written) in 42 us, 5.6 TB/s
// where a copy reaches 6.5; 53 us with blocks in two waves and a unit's rows
// looked up when it is due, 45 without the prefetch of the next unit's.
// Rows decoded inside the attention kernel would spare the 151 MB, but the
// conversions then share the issue slots with the softmax: 153 to 202 us for
// that call, where decoding ahead took 150 at the time.
__global__ void __launch_bounds__(kStageThreads, kStageBlocks) stage_kernel(const __grid_constant__ TcCall c) {
  extern __shared__ int sm[];
  const PagedAttnProblem& p = c.p;
  const PagedLayer& g = p.pages;
  int* block_start = sm;                  // [n_seqs + 1]
  int* tile_start = sm + g.n_seqs + 1;
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  int blocks = 0, tiles = 0;
  for (int base = 0; base < g.n_seqs; base += kStageThreads) {
    const int s = base + tid;
    int nb = 0, nt = 0;
    if (s < g.n_seqs) {
      const Slot slot = slot_geometry(p, c.s.tokens_per_tile, s);
      nb = slot.blocks;
      nt = slot.tiles;
    }
    int tb, tt;
    const int b = blocks + stage_scan(nb, &tb), t = tiles + stage_scan(nt, &tt);
    if (s < g.n_seqs) {
      block_start[s] = b;
      tile_start[s] = t;
    }
    blocks += tb;
    tiles += tt;
  }
  if (tid == 0) {
    block_start[g.n_seqs] = blocks;
    tile_start[g.n_seqs] = tiles;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    list_tiles(c, block_start, tile_start);
    return;
  }
  const long long units = min(static_cast<long long>(blocks), c.s.block_cap) * (kKeys / kUnit);
  const int lane = tid & 31, warps = kStageThreads / 32;
  const bool is_code = lane < 28;
  const uint8_t* lane_src = is_code ? g.codes + 16 * lane
                                    : reinterpret_cast<const uint8_t*>(g.rope) + 32 * (lane - 28);
  const size_t pitch = is_code ? kNope : 2 * kRope;
  // Non-zero where one of this lane's values is not finite: the E4M3 NaN has
  // all magnitude bits set, a BF16 NaN or infinity all exponent bits, and
  // adding one to the field carries into the bit above it.
  const uint32_t field = is_code ? 0x7F7F7F7Fu : 0x7F807F80u;
  const uint32_t one = is_code ? 0x01010101u : 0x00800080u;
  const uint32_t above = is_code ? 0x80808080u : 0x80008000u;
  auto special4 = [](const uint4& v, uint32_t f, uint32_t o, uint32_t a) {
    return (((v.x & f) + o) | ((v.y & f) + o) | ((v.z & f) + o) | ((v.w & f) + o)) & a;
  };
  auto special_bf16 = [&](const uint4& v) {
    return special4(v, 0x7F807F80u, 0x00800080u, 0x80008000u);
  };
  // The cache row of key lane & 7 of unit u, -1: none. Found while the unit
  // before is decoded, so that a unit waits for its rows alone.
  auto find_row = [&](long long u) {
    const int block = static_cast<int>(u / (kKeys / kUnit));
    int lo = 0, hi = g.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (block_start[mid] <= block) lo = mid;
      else hi = mid;
    }
    const int len = slot_length(g, lo), first = len - (p.q_start[lo + 1] - p.q_start[lo]);
    const unsigned at = static_cast<unsigned>(seen_from(p.window, first)) +
                        (block - block_start[lo]) * kKeys +
                        static_cast<int>(u % (kKeys / kUnit)) * kUnit + (lane & 7);
    const int t = static_cast<int>(at);
    int row = -1;
    if (at < static_cast<unsigned>(len) && t / g.page < g.max_pages) {
      const int page = g.table[static_cast<size_t>(lo) * g.max_pages + t / g.page];
      if (page >= 0 && page < g.n_pages) row = page * g.page + t % g.page;
    }
    return row;
  };
  const long long step = (gridDim.x - 1ll) * warps;
  long long u = (blockIdx.x - 1ll) * warps + (tid >> 5);
  int next_row = u < units ? find_row(u) : -1;
  for (; u < units; u += step) {
    const int row = next_row;
    const unsigned there = __ballot_sync(0xffffffffu, row >= 0) & 0xFFu;
    const int rc = max(row, 0);  // (an absent key's lanes load row 0 and do not use it)
    uint4 raw[kUnit];
    // 4 scale codes: of key lane & 7, groups 0-3 or (lanes 16-31) 4-7
    const uint32_t sc = __ldg(reinterpret_cast<const uint32_t*>(
        g.scales + static_cast<size_t>(__shfl_sync(0xffffffffu, rc, lane & 7)) * kKvScaleSlots +
        4 * (lane >> 4)));
#pragma unroll
    for (int r = 0; r < kUnit; ++r)
      raw[r] = __ldg(reinterpret_cast<const uint4*>(
          lane_src + static_cast<size_t>(__shfl_sync(0xffffffffu, rc, r)) * pitch));
    const uint4 more = __ldg(reinterpret_cast<const uint4*>(
        reinterpret_cast<const uint8_t*>(g.rope) +
        static_cast<size_t>(__shfl_sync(0xffffffffu, rc, lane >> 2)) * (2 * kRope) +
        32 * (lane & 3) + 16));
    if (u + step < units) next_row = find_row(u + step);
    uint32_t code[kUnit];  // the scale code of this lane's dims
    bool in_range = true;
    unsigned bad = special_bf16(more) ? 1u << (lane >> 2) : 0u;
#pragma unroll
    for (int r = 0; r < kUnit; ++r) {
      code[r] = (__shfl_sync(0xffffffffu, sc, r + (lane & 16)) >> (8 * ((lane >> 2) & 3))) & 0xFFu;
      in_range = in_range && code[r] - 10u <= 124u;
      bad |= (special4(raw[r], field, one, above) ? 1u : 0u) << r;
    }
    const bool fast = __all_sync(0xffffffffu, in_range || !is_code);
    if (!fast && is_code) {  // a large scale may take a finite code beyond BF16's range
#pragma unroll
      for (int r = 0; r < kUnit; ++r) {
        const float f = e8m0_decode(code[r]);
        const uint2 a = e4m3x4_to_bf16(raw[r].x, f), b = e4m3x4_to_bf16(raw[r].y, f);
        const uint2 d = e4m3x4_to_bf16(raw[r].z, f), e = e4m3x4_to_bf16(raw[r].w, f);
        if (special_bf16(make_uint4(a.x, a.y, b.x, b.y)) | special_bf16(make_uint4(d.x, d.y, e.x, e.y)))
          bad |= 1u << r;
      }
    }
    bad = __reduce_or_sync(0xffffffffu, bad) & there;
    const unsigned keep = there & ~bad;  // the others are zeros: they take part in no sum
    if (next_row >= 0) {  // the next unit's rows to L2: lane's key, a line of its codes each
      const uint8_t* at = g.codes + static_cast<size_t>(next_row) * kNope + 128 * (lane >> 3);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      if (lane < kUnit)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(g.rope + static_cast<size_t>(next_row) * kRope));
    }
    uint8_t* dst = reinterpret_cast<uint8_t*>(c.w.stage + u * kUnit * kD) + 32 * lane;
#pragma unroll
    for (int r = 0; r < kUnit; ++r) {
      uint4 x = make_uint4(0, 0, 0, 0), y = x;
      if ((keep >> r) & 1u) {
        if (fast) {
          const uint32_t k2 = (code[r] + 120) * 0x00800080u;
          const uint2 a = e4m3x4_to_bf16_mul(raw[r].x, k2), b = e4m3x4_to_bf16_mul(raw[r].y, k2);
          const uint2 d = e4m3x4_to_bf16_mul(raw[r].z, k2), e = e4m3x4_to_bf16_mul(raw[r].w, k2);
          x = make_uint4(a.x, a.y, b.x, b.y);
          y = make_uint4(d.x, d.y, e.x, e.y);
        } else {
          const float f = e8m0_decode(code[r]);
          const uint2 a = e4m3x4_to_bf16(raw[r].x, f), b = e4m3x4_to_bf16(raw[r].y, f);
          const uint2 d = e4m3x4_to_bf16(raw[r].z, f), e = e4m3x4_to_bf16(raw[r].w, f);
          x = make_uint4(a.x, a.y, b.x, b.y);
          y = make_uint4(d.x, d.y, e.x, e.y);
        }
        if (!is_code) x = raw[r];
      }
      if (is_code) st_global_32(dst + r * (2 * kD), x, y);
      else *reinterpret_cast<uint4*>(dst + r * (2 * kD)) = x;
    }
    // row lane / 4, second halves of its RoPE quarters
    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c.w.stage + (u * kUnit + (lane >> 2)) * kD) +
                              2 * kNope + 32 * (lane & 3) + 16) =
        (keep >> (lane >> 2)) & 1u ? more : make_uint4(0, 0, 0, 0);
    if (lane == 0) {
      c.w.valid[u] = static_cast<uint8_t>(there);
      c.w.broken[u] = static_cast<uint8_t>(bad);
    }
  }
  // the attention kernel reads the rows through the async proxy
  asm volatile("fence.proxy.async.global;" ::: "memory");
}

constexpr int kOwnStages = 3;    // 32 KB: a block's dims of this CTA's half, also the V of P V
constexpr int kOtherStages = 4;  // 16 KB: half of its other dims
constexpr uint32_t kBlk = kKeys * 128;       // 64 keys x 64 dims, one swizzled box (8 KB)
constexpr uint32_t kQBlk = kRows * 128;      // 128 rows x 64 dims (16 KB)
constexpr uint32_t kSmQ = 0;                 // Q dims 256-511 (64 KB)
constexpr uint32_t kSmOwn = 4 * kQBlk;
constexpr uint32_t kSmOther = kSmOwn + kOwnStages * 4 * kBlk;
constexpr uint32_t kSmBar = kSmOther + kOtherStages * 2 * kBlk;
constexpr uint32_t kSmMax = kSmBar + 256;    // [2 blocks][2 key halves][128] row maxima
constexpr uint32_t kSmScale = kSmMax + 2 * 2 * kRows * 4;  // [128] what O is multiplied by
constexpr uint32_t kTcBytes = kSmScale + kRows * 4;
static_assert(kTcBytes <= 232448, "beyond the shared memory of a CTA");
// TMEM: O 0-255, S, P and what its rounding left (two values a column), Q dims 0-255
constexpr uint32_t kColS = 256, kColP = 320, kColQ = 384, kCols = 512;

constexpr int kSoftmaxWarps = 8, kLoadWarps = 4;
constexpr int kWarpTma = kSoftmaxWarps + kLoadWarps, kWarpMma = kWarpTma + 1;
constexpr int kTcThreads = 32 * (kWarpMma + 1);

struct Bars {
  uint64_t full_own[kOwnStages], empty_own[kOwnStages];
  uint64_t full_other[kOtherStages], empty_other[kOtherStages];
  uint64_t s_full, s_free, p_full, pv_done, q_full, q_free, o_ready, o_free, fin, pair[4];
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(Bars) <= 256, "barriers exceed their room");

// The tile that holds unit F (whole warp; F < total): 32 probes a step.
__device__ __forceinline__ int find_tile(const Tile* tiles, int n, long long F) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // tiles[lo].start <= F
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool ok = at < hi && tiles[at].start <= F;
    const int k = __popc(__ballot_sync(0xffffffffu, ok)) - 1;
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// A piece of a tile that one share holds.
struct Segment {
  Tile t;
  int j0, j1;     // its blocks
};

// Walks a share's segments: every role runs the same walk. Block j of a tile
// is its unit kTileCost + j and belongs to the share that has it.
struct Walk {
  const Tile* tiles;
  long long F, end;
  int t;
  __device__ bool next(Segment& s) {
    if (F >= end) return false;
    s.t = tiles[t++];
    const long long first = s.t.start + kTileCost;
    s.j0 = F > first ? static_cast<int>(F - first) : 0;
    const long long to = end - first;
    if (to <= 0) {  // the share ends before the tile's first block
      F = end;
      return false;
    }
    s.j1 = to < s.t.blocks ? static_cast<int>(to) : s.t.blocks;
    F = first + s.j1;
    return true;
  }
};

__device__ __forceinline__ uint4 load_q8(const PagedAttnProblem& p, long long at) {
  if (p.bf16)
    return __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at));
  const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at);
  const float4 a = __ldg(s), b = __ldg(s + 1);
  return make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                    pack_bf16x2(b.z, b.w));
}

__device__ __forceinline__ int part_slot(const Tile& t, long long share0) {
  return t.start + kTileCost < share0 ? 0 : 1;  // 0: the tile began in an earlier share
}

// 16 output dims of a row (16-byte aligned; whole sectors where 32 fit).
__device__ __forceinline__ void store_o16(const PagedAttnProblem& p, long long at, const float* v) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (p.bf16) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.out) + at;
    const uint4 a = make_uint4(w[0], w[1], w[2], w[3]), b = make_uint4(w[4], w[5], w[6], w[7]);
    if (p.out_32) {
      st_global_32(d, a, b);
    } else {
      reinterpret_cast<uint4*>(d)[0] = a;
      reinterpret_cast<uint4*>(d)[1] = b;
    }
  } else {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = make_float4(__uint_as_float(w[2 * i] << 16), __uint_as_float(w[2 * i] & 0xFFFF0000u),
                         __uint_as_float(w[2 * i + 1] << 16),
                         __uint_as_float(w[2 * i + 1] & 0xFFFF0000u));
  }
}

// Inverse RoPE of 32 dims from d0 on, the pairs from r0 on; the row's factors
// are loaded together, in whole vectors where they are whole.
__device__ __forceinline__ void rope_dims(const PagedAttnProblem& p, long long row, int d0, int r0,
                                          float (&v)[32]) {
  const long long ra = row * (p.rope_out / 2);
  float cs[16], sn[16];
  if (p.rope_vec) {  // all 32 dims, 16-byte aligned
    const float4* c4 = reinterpret_cast<const float4*>(p.rope_cos + ra + (d0 - r0) / 2);
    const float4* s4 = reinterpret_cast<const float4*>(p.rope_sin + ra + (d0 - r0) / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = __ldg(c4 + i), b = __ldg(s4 + i);
      cs[4 * i] = a.x, cs[4 * i + 1] = a.y, cs[4 * i + 2] = a.z, cs[4 * i + 3] = a.w;
      sn[4 * i] = b.x, sn[4 * i + 1] = b.y, sn[4 * i + 2] = b.z, sn[4 * i + 3] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool in = d0 + 2 * i >= r0;
      const long long at = ra + (in ? (d0 + 2 * i - r0) / 2 : 0);
      cs[i] = __ldg(p.rope_cos + at);
      sn[i] = __ldg(p.rope_sin + at);
      if (!in) {
        cs[i] = 1.f;
        sn[i] = 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x0 = v[2 * i], x1 = v[2 * i + 1];
    v[2 * i] = x0 * cs[i] + x1 * sn[i];
    v[2 * i + 1] = x1 * cs[i] - x0 * sn[i];
  }
}

// Denominator with the sink and what the sums are divided by, from the
// running max m, the sum den of the scores and the sink s2, in log2 units.
struct Norm {
  float scale;  // of the value sums
  float lse;
};
__device__ __forceinline__ Norm finish(float m, float den, float s2) {
  const float mx = fmaxf(m, s2);
  if (den != den) return {NAN, NAN};
  if (mx == -INFINITY) return {0.f, -INFINITY};  // nothing seen, no sink
  const float f = m == -INFINITY ? 0.f : exp2f(m - mx);
  const float total = den * f + exp2f(s2 - mx);
  return {f / total, (mx + log2f(total)) * 0.69314718055994531f};
}

// Waits suspended in hardware rather than spinning: the softmax warps need
// the issue slots.
__device__ __forceinline__ bool long_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned* err) {
  auto wait = [&] {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;"
        " selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity), "r"(20000u)  // at most 20 us at a time
        : "memory");
    return ok != 0;
  };
  if (wait()) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!wait()) {
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      if (err) atomicOr(err, kErrWait);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

// MMA issue by one thread of a role that only this thread runs: no election
// per instruction, and no vote or fence at waits that order nothing but
// copies, so that the issue stays ahead of the tensor pipe.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e; }" : "=r"(p));
  return p != 0;
}

// The two warps of 32 rows meet (a barrier in shared memory, because a named
// one could not give up).
struct PairSync {
  uint64_t* bar;
  unsigned done;
  volatile int* abort_flag;
  unsigned* err;
  __device__ __forceinline__ bool operator()() {
    mbar_arrive(bar);
    return long_wait(bar, done++ & 1, abort_flag, err);
  }
};

// 32 scores of a row (this thread's half of the block's keys) to weights in
// TMEM, in one BF16 term or two. P V of the block before, which reads them there, is waited for when the new ones are
// ready. `rescale`: O (and what was summed before) is to be
// multiplied by alpha.
struct RowState {
  float m, den;
  float held;  // the sum of the weights as P V takes them
};
template <bool kMasked, bool kTwoTerms, class WaitPv>
__device__ __forceinline__ bool softmax_block(uint32_t s_col, uint32_t mask, float sc2,
                                              float* max_mine, const float* max_other,
                                              PairSync& meet, bool& good, RowState& st,
                                              float& alpha, uint32_t p_col, uint64_t* s_free,
                                              WaitPv wait_pv) {
  uint32_t r[32];
  tmem_ld32(s_col, r);
  tc_fence_before();
  mbar_arrive(s_free);  // the next block's scores may come
  float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (kMasked && !((mask >> i) & 1u)) r[i] = 0xFF800000u;
    tm[i & 3] = fmaxf(tm[i & 3], __uint_as_float(r[i]));
  }
  const float mine = fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]));
  *max_mine = mine;
  good = meet() && good;
  const float tmax = fmaxf(mine, *max_other) * sc2;  // scale > 0
  // the running max moves only when a score exceeds it by the margin:
  // weights stay <= 2^8 and O is rarely rescaled
  bool rescale = false;
  alpha = 1.f;
  if (tmax != -INFINITY) {
    if (st.m == -INFINITY) {
      st.m = tmax;
    } else if (tmax > st.m + kLazyMargin) {
      alpha = ex2_approx(st.m - tmax);
      st.m = tmax;
      rescale = true;
    }
  }
  const float neg = st.m == -INFINITY ? 0.f : -st.m;
  float part[4] = {0.f, 0.f, 0.f, 0.f}, held[2] = {0.f, 0.f};
  uint32_t less[16];  // what the rounding left
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float e0 = ex2_approx(fmaf(__uint_as_float(r[i]), sc2, neg));
    const float e1 = ex2_approx(fmaf(__uint_as_float(r[i + 1]), sc2, neg));
    part[(i >> 1) & 3] += e0 + e1;
    const uint32_t h = pack_bf16x2(e0, e1);
    const float h0 = __uint_as_float(h << 16), h1 = __uint_as_float(h & 0xFFFF0000u);
    if (kTwoTerms) less[i / 2] = pack_bf16x2(e0 - h0, e1 - h1);
    else held[(i >> 1) & 1] += h0 + h1;
    r[i / 2] = h;
  }
  good = wait_pv() && good;
  __syncwarp();
  tc_fence_after();
  tmem_st16(p_col, r);
  if (kTwoTerms) tmem_st16(p_col + kKeys / 2, less);
  tmem_st_wait();
  const float sum = (part[0] + part[1]) + (part[2] + part[3]);
  st.den = st.den * alpha + sum;
  if (!kTwoTerms) st.held = st.held * alpha + (held[0] + held[1]);
  return rescale;
}

// One share of (tile, block) pairs and one half of the output dims. Roles:
//   warps 0-7  softmax: row = TMEM lane, two threads a row, one for each half of
//              a block's keys
//   warps 8-11 dims 0-255 of the next segment's Q to TMEM, once this one's last
//              Q K^T is done, then this one's O out, while the others go on
//   warp 12    key blocks and Q by TMA (one lane)
//   warp 13    TMEM allocation and MMA issue
// Per block: S = Q K^T (32 MMAs of 128 x 64 x 16, the other half's dims first
// so that their slots are free early), P = 2^(S - m) in BF16 back to TMEM,
// O += P V (4 MMAs of 128 x 256 x 16, P the A operand in TMEM, the own half
// read MN-major). Q K^T of a block is issued once the scores of the one before
// are in registers, P V of that one after it, so the tensor pipe works while
// the softmax does. P in TMEM leaves 32 KB to the ring of the other dims, two
// blocks ahead instead of one: where the rows come from DRAM that is what
// counts (32 sequences of 4.6k keys: 55 us of 64; keys that L2 holds: 2% more
// than with P in shared memory and two buffers of S).
// kShort: no tile has more than kTwoTermBlocks blocks.
template <bool kShort>
__global__ void __launch_bounds__(kTcThreads, 1) paged_attn_tc_kernel(
    const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap qmap,
    const __grid_constant__ TcCall c) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_addr(smem);
  Bars* bars = reinterpret_cast<Bars*>(smem + kSmBar);
  volatile int* abort_flag = &bars->abort_flag;
  const PagedAttnProblem& p = c.p;
  unsigned* err = p.err;
  const int half = blockIdx.x & 1, pair = blockIdx.x >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kOwnStages; ++i) {
      mbar_init(&bars->full_own[i], 1);
      mbar_init(&bars->empty_own[i], 1);
    }
    for (int i = 0; i < kOtherStages; ++i) {
      mbar_init(&bars->full_other[i], 1);
      mbar_init(&bars->empty_other[i], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->s_free, 32 * kSoftmaxWarps);
    mbar_init(&bars->p_full, 32 * kSoftmaxWarps);
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->q_full, 32 * kLoadWarps + 1);  // and the TMA warp's
    mbar_init(&bars->q_free, 1);
    mbar_init(&bars->o_ready, 32 * kSoftmaxWarps);
    mbar_init(&bars->o_free, 32 * kLoadWarps);
    mbar_init(&bars->fin, 1);
    for (int i = 0; i < 4; ++i) mbar_init(&bars->pair[i], 64);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kWarpTma && lane == 0) {
    tma_prefetch_desc(&map);
    tma_prefetch_desc(&qmap);
  }
  pdl_wait();  // the plan and the decoded rows
  pdl_trigger();
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&bars->tmem)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  const PlanHead head = *c.w.head;
  Walk walk;
  walk.tiles = c.w.tiles;
  walk.F = static_cast<long long>(pair) * head.share;
  walk.end = min(head.total, walk.F + head.share);
  walk.t = walk.F < walk.end ? find_tile(c.w.tiles, head.tiles, walk.F) : 0;
  Segment seg;

  if (warp < kSoftmaxWarps) {
    // ----------------------------------------------------- softmax, epilogue
    if (half == 0 && threadIdx.x == 0 && walk.F < walk.end) c.w.first_tile[pair] = c.w.tiles[walk.t];
    const int side = warp >> 2, w4 = warp & 3;
    const int row = w4 * 32 + lane;
    const int tok = row / p.H, h = row - tok * p.H;
    const uint32_t lanes = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t o_cols = tmem + lanes + side * (kHalf / 2);
    const uint32_t s_col = tmem + lanes + kColS + side * 32, p_col = tmem + lanes + kColP + side * 16;
    float* maxima = reinterpret_cast<float*>(smem + kSmMax);
    float* max_mine = maxima + side * kRows + row;
    const float* max_other = maxima + (1 - side) * kRows + row;
    const float sc2 = p.scale * kLog2e;
    const float sink2 = p.sink && h < p.H && tok < kRows / p.H ? p.sink[h] * kLog2e : -INFINITY;
    const long long share0 = walk.F;
    PairSync meet = {&bars->pair[w4], 0, abort_flag, err};
    unsigned n = 0, segs = 0;  // blocks and segments done by this CTA
    bool ok = true;
    while (ok && walk.next(seg)) {
      const Tile& t = seg.t;
      const bool mine = tok < t.tokens;
      const int last = mine ? t.pos0 + tok : -1;  // the position of this row's token
      const int from = seen_from(p.window, last);
      const bool two_terms = kShort || t.blocks <= kTwoTermBlocks;
      RowState st = {-INFINITY, 0.f, 0.f};
      bool bad = t.bad != 0;
      const unsigned long long* valid =
          reinterpret_cast<const unsigned long long*>(c.w.valid) + t.block0;
      const unsigned long long* brk =
          reinterpret_cast<const unsigned long long*>(c.w.broken) + t.block0;
      unsigned long long mask_next = valid[seg.j0], broken_next = brk[seg.j0];
      for (int j = seg.j0; j < seg.j1; ++j, ++n) {
        const int key0 = t.key0 + j * kKeys;
        unsigned long long mask = mask_next;
        const unsigned long long broken = broken_next;
        if (j + 1 < seg.j1) {
          mask_next = valid[j + 1];
          broken_next = brk[j + 1];
        }
        // a block that every row sees whole needs no mask
        const int hi_key = last - key0, lo_key = from - key0;
        const bool whole = hi_key >= kKeys - 1 && lo_key <= 0 && mask == ~0ull && broken == 0;
        const bool masked = two_terms || !__all_sync(0xffffffffu, whole);
        uint32_t mask32 = ~0u;
        if (masked) {
          // bits 0 .. last - key0, and from the window's first on
          mask &= hi_key < 0 ? 0ull : hi_key >= 63 ? ~0ull : (2ull << hi_key) - 1;
          if (lo_key > 0) mask &= lo_key > 63 ? 0ull : ~0ull << lo_key;
          if (broken & mask) bad = true;
          mask &= ~broken;
          mask32 = static_cast<uint32_t>(mask >> (32 * side));
        }
        // A wait that gives up ends the loop at the block's vote; what is
        // computed until then is not used.
        bool good = long_wait(&bars->s_full, n & 1, abort_flag, err);
        __syncwarp();
        tc_fence_after();
        const int buf = static_cast<int>(n & 1) * 2 * kRows;
        float alpha;
        // P V of the block before has read P, and O holds all blocks before
        auto wait_pv = [&] {
          return n == 0 || long_wait(&bars->pv_done, (n - 1) & 1, abort_flag, err);
        };
        auto softmax = [&](auto m, auto two) {
          return softmax_block<m.value, two.value>(s_col, mask32, sc2, max_mine + buf,
                                                   max_other + buf, meet, good, st, alpha, p_col,
                                                   &bars->s_free, wait_pv);
        };
        bool rescale;
        if constexpr (kShort)
          rescale = softmax(std::true_type(), std::true_type());
        else
          rescale = !masked     ? softmax(std::false_type(), std::false_type())
                    : two_terms ? softmax(std::true_type(), std::true_type())
                                : softmax(std::true_type(), std::false_type());
        if (!__all_sync(0xffffffffu, good)) {
          ok = false;
          break;
        }
        if (__any_sync(0xffffffffu, rescale)) {
          tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < kHalf / 2; cb += 32) {
            uint32_t o[32];
            tmem_ld32(o_cols + cb, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_cols + cb, o);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&bars->p_full);
      }
      if (!ok) break;
      // the row's denominators: both threads' sums (the buffer of the block
      // before the last one is free, the last one's once both have been here)
      const int buf = (n & 1) * 2 * kRows, buf_held = 2 * kRows - buf;
      max_mine[buf] = st.den;
      bool good = meet();
      float den = st.den + max_other[buf];
      if (!two_terms) max_mine[buf_held] = st.held;
      good = meet() && good;  // read before the next segment writes it
      // O has the weights as P V took them: times this, they sum to den
      float back = 1.f;
      if (!two_terms) {
        const float held = st.held + max_other[buf_held];
        if (held > 0.f) back = den / held;
      }
      // the segment before is out, so its factors may be overwritten
      if (segs > 0) good = long_wait(&bars->o_free, (segs - 1) & 1, abort_flag, err) && good;
      ++segs;
      if (!__all_sync(0xffffffffu, good)) {
        ok = false;
        break;
      }
      if (bad) den = NAN;
      if (seg.j0 == 0 && seg.j1 == t.blocks) {
        const Norm norm = finish(st.m, den, sink2);
        if (side == 0) {
          reinterpret_cast<float*>(smem + kSmScale)[row] = norm.scale * back;
          if (mine && half == 0 && p.lse)
            p.lse[static_cast<long long>(t.row0 + tok) * p.H + h] = norm.lse;
        }
      } else if (mine && side == 0) {
        const long long at = pair * 2 + part_slot(t, share0);
        c.w.part_m[(at * 2 + half) * kRows + row] = st.m;
        c.w.part_den[(at * 2 + half) * kRows + row] = den;
        c.w.part_back[(at * 2 + half) * kRows + row] = back;
      }
      mbar_arrive(&bars->o_ready);
    }
  } else if (warp < kWarpTma) {
    // ------------------------------------------------------- Q in, O out
    const int w4 = warp & 3, row = w4 * 32 + lane;
    const int tok = row / p.H, h = row - tok * p.H;
    const uint32_t lanes = static_cast<uint32_t>(w4 * 32) << 16;
    const long long share0 = walk.F;
    unsigned it = 0, slot = 0, phase = 0;  // slot and phase of the own ring
    unsigned n = 0;                        // blocks of the segments before
    auto to_tmem = [&](const uint4 (&a)[16], int k) {  // dims 128 k ..
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t r[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          r[4 * i] = a[8 * q + i].x;
          r[4 * i + 1] = a[8 * q + i].y;
          r[4 * i + 2] = a[8 * q + i].z;
          r[4 * i + 3] = a[8 * q + i].w;
        }
        tmem_st32(tmem + lanes + kColQ + 64 * k + 32 * q, r);
      }
    };
    auto load_q = [&](const Segment& sg) {
      const Tile& t = sg.t;
      bool good = true;
      uint4 a[16];
      // (also before the own ring is looked at: only now is the slot's phase
      // the one before Q's)
      if (it > 0) good = long_wait(&bars->q_free, (it - 1) & 1, abort_flag, err);
      __syncwarp();
      tc_fence_after();
      if (p.bf16) {
        // dims 0-255 come through two slots of the own ring, ahead of the
        // segment's first block
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          good = long_wait(&bars->full_own[slot], phase, abort_flag, err) && good;
          const uint8_t* src = smem + kSmOwn + slot * 4 * kBlk + row * 128;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            a[i] = *reinterpret_cast<const uint4*>(src + (i >> 3) * kQBlk +
                                                   (((i & 7) ^ (row & 7)) << 4));
          to_tmem(a, k);
          if (++slot == kOwnStages) { slot = 0; phase ^= 1; }
        }
        slot += static_cast<unsigned>(sg.j1 - sg.j0);
        phase ^= (slot / kOwnStages) & 1;
        slot %= kOwnStages;
      } else {
        // fp32 rows are converted on their way
        const long long at = tok < t.tokens ? static_cast<long long>(t.row0 + tok) * p.q_stride +
                                                  static_cast<long long>(h) * kD
                                            : -1ll;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            a[i] = at >= 0 ? load_q8(p, at + 128 * k + 8 * i) : make_uint4(0, 0, 0, 0);
          to_tmem(a, k);
        }
#pragma unroll 1
        for (int i0 = 0; i0 < 32; i0 += 16) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const long long b = __shfl_sync(0xffffffffu, at, i0 + i);
            a[i] = b >= 0 ? load_q8(p, b + kHalf + 8 * lane) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            st_shared_v4(base + kSmQ + sw128_off(w4 * 32 + i0 + i, lane, kRows), a[i]);
        }
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->q_full);
      return __all_sync(0xffffffffu, good);
    };
    // O of segment number i, whose last block is block number nb
    auto store_o = [&](const Segment& sg, unsigned i, unsigned nb) {
      const Tile& t = sg.t;
      const bool mine = tok < t.tokens;
      bool good = long_wait(&bars->o_ready, i & 1, abort_flag, err);
      good = long_wait(&bars->pv_done, nb & 1, abort_flag, err) && good;
      if (!__all_sync(0xffffffffu, good)) return false;
      tc_fence_after();
      if (sg.j0 == 0 && sg.j1 == t.blocks) {
        const float scale = reinterpret_cast<const volatile float*>(smem + kSmScale)[row];
        const long long at = static_cast<long long>(t.row0 + tok);
        const long long o_at = at * p.out_stride + static_cast<long long>(h) * kD + half * kHalf;
        const int r0 = kD - p.rope_out;
#pragma unroll 1
        for (int cb = 0; cb < kHalf; cb += 32) {
          uint32_t o[32];
          tmem_ld32(tmem + lanes + cb, o);
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o[k]) * scale;
          const int d0 = half * kHalf + cb;
          if (mine) {
            if (p.rope_cos && d0 + 32 > r0) rope_dims(p, at, d0, r0, v);
#pragma unroll
            for (int k = 0; k < 32; k += 16) store_o16(p, o_at + cb + k, v + k);
          }
        }
      } else {
        float* part = c.w.part_o +
                      ((pair * 2 + part_slot(t, share0)) * static_cast<long long>(kRows) + row) * kD +
                      half * kHalf;
#pragma unroll 1
        for (int cb = 0; cb < kHalf; cb += 32) {
          uint32_t o[32];
          tmem_ld32(tmem + lanes + cb, o);
          if (mine) {
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              st_global_32(part + cb + k, make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]),
                           make_uint4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]));
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&bars->o_free);  // the next segment's P V may overwrite it
      return true;
    };
    // The next segment's Q goes in as soon as this one's last Q K^T is done,
    // before this one's O comes out.
    Segment before;
    bool ok = true;
    while (ok && walk.next(seg)) {
      ok = load_q(seg);
      if (ok && it > 0) {
        n += before.j1 - before.j0;
        ok = store_o(before, it - 1, n - 1);
      }
      before = seg;
      ++it;
    }
    if (ok && it > 0) store_o(before, it - 1, n + (before.j1 - before.j0) - 1);
  } else if (warp == kWarpTma) {
    // ------------------------------------------------------------ key blocks
    if (lane == 0) {
      asm volatile("fence.proxy.async.global;" ::: "memory");
      unsigned no = 0, nw = 0, it = 0;  // other / own slots and Q tiles filled so far
      bool ok = true;
      const uint32_t q_rows = (kRows / p.H) * p.H;
      auto load_q = [&](const Tile& t) {  // dims 256-511
        if (it > 0 && !long_wait(&bars->q_free, (it - 1) & 1, abort_flag, err)) return false;
        ++it;
        if (!p.bf16) {
          mbar_arrive(&bars->q_full);
          return true;
        }
        mbar_arrive_expect_tx(&bars->q_full, 4 * 128 * q_rows);
        for (int b = 0; b < 4; ++b)
          tma_load_3d(smem + kSmQ + b * kQBlk, &qmap, 512 + b * 128, 0, t.row0, &bars->q_full);
        return true;
      };
      auto load_own = [&](const CUtensorMap* m, int x, int y, bool q) {
        const unsigned s = nw % kOwnStages;
        if (!long_wait(&bars->empty_own[s], ((nw / kOwnStages) & 1) ^ 1, abort_flag, err))
          return false;
        mbar_arrive_expect_tx(&bars->full_own[s], q ? 2 * 128 * q_rows : 4 * kBlk);
        if (q) {
          for (int b = 0; b < 2; ++b)
            tma_load_3d(smem + kSmOwn + s * 4 * kBlk + b * kQBlk, m, x + b * 128, 0, y,
                        &bars->full_own[s]);
        } else {
          for (int b = 0; b < 4; b += 2)
            tma_load_3d(smem + kSmOwn + (s * 4 + b) * kBlk, m, 0, y, x + b, &bars->full_own[s]);
        }
        ++nw;
        return true;
      };
      while (ok && walk.next(seg)) {
        // Q and the first key blocks are on their way before Q's room is free (2000
        // tiles take 4% longer with Q's second part behind them)
        if (p.bf16) {
          for (int k = 0; k < 2 && ok; ++k) ok = load_own(&qmap, 256 * k, seg.t.row0, true);
        }
        bool q_due = true;
        for (int j = seg.j0; j < seg.j1 && ok; ++j) {
          const int y = (seg.t.block0 + j) * kKeys;
          for (int q = 0; q < 2; ++q, ++no) {
            const unsigned s = no % kOtherStages;
            if (!long_wait(&bars->empty_other[s], ((no / kOtherStages) & 1) ^ 1, abort_flag, err)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&bars->full_other[s], 2 * kBlk);
            tma_load_3d(smem + kSmOther + s * 2 * kBlk, &map, 0, y, (1 - half) * 4 + q * 2,
                        &bars->full_other[s]);
          }
          if (!ok) break;
          if (q_due) {
            q_due = false;
            if (!load_q(seg.t)) { ok = false; break; }
          }
          ok = load_own(&map, half * 4, y, false);
        }
      }
      // no copy may be in flight when the CTA ends: the last one of each slot
      for (unsigned i = no > kOtherStages ? no - kOtherStages : 0; i < no; ++i)
        mbar_wait(&bars->full_other[i % kOtherStages], (i / kOtherStages) & 1, err);
      for (unsigned i = nw > kOwnStages ? nw - kOwnStages : 0; i < nw; ++i)
        mbar_wait(&bars->full_own[i % kOwnStages], (i / kOwnStages) & 1, err);
      if (it > 0) mbar_wait(&bars->q_full, (it - 1) & 1, err);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- MMA issue
    if (elect_one()) {
      constexpr uint32_t idesc_qk = umma_idesc_bf16(kRows, kKeys, false);
      constexpr uint32_t idesc_pv = umma_idesc_bf16(kRows, kHalf, true);
      const uint64_t q_desc = umma_desc(base + kSmQ, 16, 1024);
      const uint64_t own_desc = umma_desc(base + kSmOwn, 16, 1024);
      const uint64_t other_desc = umma_desc(base + kSmOther, 16, 1024);
      const uint64_t v_desc = umma_desc(base + kSmOwn, kBlk, 1024);
      // A barrier is looked at before the MMAs that come first are issued, so
      // that its answer is there when they are.
      auto peek = [&](uint64_t* bar, unsigned parity) { return mbar_try_wait(bar, parity & 1); };
      auto waits = [&](bool ready, uint64_t* bar, unsigned parity) {
        return ready || long_wait(bar, parity & 1, abort_flag, err);
      };
      // Q K^T over 128 dims at column blocks cb, cb + 1 of a 256-dim half
      auto qk = [&](uint32_t s_col, uint64_t k_desc, int q_half, int cb, bool first) {
        if (q_half == 0) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_ts(s_col, tmem + kColQ + cb * 32 + kk * 8,
                   k_desc + ((kk >> 2) * kBlk + (kk & 3) * 32) / 16, idesc_qk,
                   !(first && kk == 0));
        } else {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_ss(s_col, q_desc + ((cb + (kk >> 2)) * kQBlk + (kk & 3) * 32) / 16,
                   k_desc + ((kk >> 2) * kBlk + (kk & 3) * 32) / 16, idesc_qk,
                   !(first && kk == 0));
        }
      };
      unsigned n = 0, it = 0;
      unsigned so = 0, po = 0, sw = 0, pw = 0;  // slot and phase of the other / own ring
      unsigned sv = 0;                          // the own slot that P V reads next
      // O += P V of block number nb of this CTA
      auto pv = [&](bool ready, unsigned nb, bool first, bool two_terms) {
        if (!waits(ready, &bars->p_full, nb)) return false;
        if (first && it > 1 && !waits(false, &bars->o_free, it - 2)) return false;
        tc_fence_after();  // the softmax's reads of S and writes of O, the reads of O
        const uint64_t v = v_desc + sv * (4 * kBlk / 16);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts(tmem, tmem + kColP + kk * 8, v + kk * 128, idesc_pv, !(first && kk == 0));
        if (two_terms) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_ts(tmem, tmem + kColP + kKeys / 2 + kk * 8, v + kk * 128, idesc_pv, true);
        }
        mma_commit(&bars->pv_done);
        mma_commit(&bars->empty_own[sv]);
        if (++sv == kOwnStages) sv = 0;
        return true;
      };
      bool ok = true;
      while (ok && walk.next(seg)) {
        if (!waits(false, &bars->q_full, it)) break;
        tc_fence_after();  // the loaders' writes of Q
        ++it;
        if (p.bf16) {  // its two slots of the own ring have been read
          for (int k = 0; k < 2; ++k) {
            mbar_arrive(&bars->empty_own[sw]);
            if (++sw == kOwnStages) { sw = 0; pw ^= 1; }
            if (++sv == kOwnStages) sv = 0;
          }
        }
        const bool two_terms = kShort || seg.t.blocks <= kTwoTermBlocks;
        bool ready = false;
        for (int j = seg.j0; j < seg.j1; ++j, ++n) {
          // the softmax has read the scores of the block before
          if (n > 0) {
            if (!(ok = waits(false, &bars->s_free, n - 1))) break;
            tc_fence_after();
          }
          const uint32_t s_col = tmem + kColS;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (!(ok = waits(ready, &bars->full_other[so], po))) break;
            const unsigned s = so;
            if (++so == kOtherStages) { so = 0; po ^= 1; }
            ready = q == 0 ? peek(&bars->full_other[so], po) : peek(&bars->full_own[sw], pw);
            qk(s_col, other_desc + s * (2 * kBlk / 16), 1 - half, 2 * q, q == 0);
            mma_commit(&bars->empty_other[s]);
          }
          if (!ok || !(ok = waits(ready, &bars->full_own[sw], pw))) break;
          const uint64_t k_desc = own_desc + sw * (4 * kBlk / 16);
          const bool pv_due = j > seg.j0;
          ready = pv_due && peek(&bars->p_full, n - 1);
          qk(s_col, k_desc, half, 0, false);
          qk(s_col, k_desc + 2 * kBlk / 16, half, 2, false);
          if (++sw == kOwnStages) { sw = 0; pw ^= 1; }
          mma_commit(&bars->s_full);
          if (j + 1 == seg.j1) mma_commit(&bars->q_free);
          const bool p_ready = ready;
          ready = peek(&bars->full_other[so], po);
          if (pv_due && !(ok = pv(p_ready, n - 1, j - 1 == seg.j0, two_terms))) break;
        }
        ok = ok && pv(false, n - 1, seg.j1 - seg.j0 == 1, two_terms);
      }
      mma_commit(&bars->fin);
      mbar_wait(&bars->fin, 0, err);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols)
                 : "memory");
}

// Tiles that a share's end cuts: a warp per (cut, row, half of the dims), 8
// dims a lane. Everything it reads is asked for as early as its address is
// known: the plan and the cut's tile, then maxima, sums and the first parts;
// that chain bounds it, and how many of the blocks, most of which have nothing
// to merge, run at once (73 cuts, 32 tiles of 64 rows: 7.4 us with four blocks
// an SM and four parts asked for together, 9.6 with two and eight; one tile in
// 19 parts: 5.7 and 5.5).
constexpr int kMergeWarps = 8, kMergeBlocks = 4;  // blocks of an SM
__global__ void __launch_bounds__(32 * kMergeWarps, kMergeBlocks) paged_attn_merge_kernel(
    const __grid_constant__ TcCall c) {
  pdl_wait();
  pdl_trigger();
  const PagedAttnProblem& p = c.p;
  const int cut = blockIdx.y + 1, lane = threadIdx.x & 31;
  const int wid = blockIdx.x * kMergeWarps + (threadIdx.x >> 5), row = wid >> 1, half = wid & 1;
  const PlanHead head = *c.w.head;
  const Tile t = c.w.first_tile[cut];  // (holds anything where the share is empty)
  const long long F = cut * head.share;
  if (F >= head.total) return;
  // the first cut inside a tile merges it
  const long long first = t.start + kTileCost;  // its first block's unit
  if (first >= F || first < F - head.share) return;
  const int tok = row / p.H, h = row - tok * p.H;
  if (tok >= t.tokens) return;
  const int n = static_cast<int>((first + t.blocks - 1) / head.share) - (cut - 1) + 1;
  auto part = [&](int i) { return static_cast<long long>(cut - 1 + i) * 2 + (i == 0 ? 1 : 0); };
  // dims 4 lane + 128 q of the half: a warp's loads are whole lines
  const float* src = c.w.part_o + half * kHalf + 4 * lane;
  constexpr int kBatch = 4;
  float4 v[kBatch][2];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i0 + k < n) {
        const float* at = src + (part(i0 + k) * kRows + row) * kD;
        v[k][0] = __ldcg(reinterpret_cast<const float4*>(at));
        v[k][1] = __ldcg(reinterpret_cast<const float4*>(at + 128));
      }
  };
  load(0);
  constexpr int kPer = 3;  // a lane's parts: lane, lane + 32, lane + 64 of at most 96
  float wt[kPer], m[kPer], d[kPer], back[kPer], M = -INFINITY;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = lane + 32 * k;
    const long long at = (part(i) * 2 + half) * kRows + row;
    m[k] = i < n ? __ldcg(c.w.part_m + at) : -INFINITY;
    d[k] = i < n ? __ldcg(c.w.part_den + at) : 0.f;
    back[k] = i < n ? __ldcg(c.w.part_back + at) : 0.f;
    M = fmaxf(M, m[k]);
  }
  M = warp_max(M);
  float den = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    wt[k] = m[k] == -INFINITY ? 0.f : exp2f(m[k] - M);
    den += d[k] * wt[k];
    // a part that saw a broken latent and nothing else has no maximum
    if (d[k] != d[k]) den = NAN;
    wt[k] *= back[k];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  const Norm norm = finish(M, den, p.sink ? p.sink[h] * kLog2e : -INFINITY);
  float acc[2][4] = {};
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k, r = i >> 5;
      const float f = __shfl_sync(0xffffffffu, r == 0 ? wt[0] : r == 1 ? wt[1] : wt[2], i & 31);
      if (i < n) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          acc[q][0] = fmaf(v[k][q].x, f, acc[q][0]);
          acc[q][1] = fmaf(v[k][q].y, f, acc[q][1]);
          acc[q][2] = fmaf(v[k][q].z, f, acc[q][2]);
          acc[q][3] = fmaf(v[k][q].w, f, acc[q][3]);
        }
      }
    }
  }
  const long long at = static_cast<long long>(t.row0 + tok);
  const int r0 = kD - p.rope_out;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int d0 = half * kHalf + 128 * q + 4 * lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[q][i] *= norm.scale;
    if (p.rope_cos) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        if (d0 + i >= r0) {
          const long long ra = at * (p.rope_out / 2) + (d0 + i - r0) / 2;
          const float cs = p.rope_cos[ra], sn = p.rope_sin[ra];
          const float y0 = acc[q][i] * cs + acc[q][i + 1] * sn;
          const float y1 = acc[q][i + 1] * cs - acc[q][i] * sn;
          acc[q][i] = y0;
          acc[q][i + 1] = y1;
        }
      }
    }
    const long long to = at * p.out_stride + static_cast<long long>(h) * kD + d0;
    const uint2 w = make_uint2(pack_bf16x2(acc[q][0], acc[q][1]), pack_bf16x2(acc[q][2], acc[q][3]));
    if (p.bf16)
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + to) = w;
    else
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + to) =
          make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u),
                      __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
  }
  if (p.lse && half == 0 && lane == 0) p.lse[at * p.H + h] = norm.lse;
}

// ------------------------------------------------------------------- host --

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2)
    return 148;
  return n;
}

bool tc_shape_ok(const PagedAttnProblem& p) {
  return p.pages.nope == kNope && p.pages.rope_dim == kRope && p.H <= kRows &&
         p.q_stride % 8 == 0 && p.out_stride % 8 == 0 && p.rope_out % 2 == 0;
}

TcShape tc_shape(const PagedAttnProblem& p) {
  TcShape s;
  s.tokens_per_tile = kRows / p.H;
  const long long active = p.pages.n_seqs < p.total ? p.pages.n_seqs : p.total;
  const long long tiles = p.total / s.tokens_per_tile + active;
  s.tile_cap = static_cast<int>(tiles < p.total ? tiles : p.total);
  // positions that one slot's tokens see
  long long one = p.max_len;
  if (p.window > 0 && static_cast<long long>(p.max_new) + p.window - 1 < one)
    one = static_cast<long long>(p.max_new) + p.window - 1;
  long long keys = active * one;
  if (p.max_keys > 0 && p.max_keys < keys) keys = p.max_keys;
  s.block_cap = keys / kKeys + active;  // each slot rounds up to a whole block
  const long long per_tile = one / kKeys + 2 + kTileCost;
  const long long most = (s.tile_cap * per_tile + kMinShare - 1) / kMinShare;
  const int pairs = sm_count() / 2 < 96 ? sm_count() / 2 : 96;
  s.pairs = static_cast<int>(most < pairs ? (most < 1 ? 1 : most) : pairs);
  return s;
}

// No tile sees more than kTwoTermBlocks blocks: n positions from any on touch
// at most (n + 62) / 64 + 1. They take a kernel of their own, without the code
// of one-term weights: 2000 tiles of three blocks 189 us, 199 in the kernel that
// has both.
bool short_tiles(const PagedAttnProblem& p, const TcShape& s) {
  long long n = p.max_len;
  if (p.window > 0) {
    const long long most =
        p.window - 1ll + (s.tokens_per_tile < p.max_new ? s.tokens_per_tile : p.max_new);
    if (most < n) n = most;
  }
  return (n + kKeys - 2) / kKeys + 1 <= kTwoTermBlocks;
}

size_t up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

size_t tc_carve(const TcShape& s, char* base, TcWs* w) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* at = base + off;
    off += up(bytes);
    return at;
  };
  const size_t pairs = s.pairs, blocks = static_cast<size_t>(s.block_cap);
  w->head = reinterpret_cast<PlanHead*>(take(sizeof(PlanHead)));
  w->tiles = reinterpret_cast<Tile*>(take(sizeof(Tile) * s.tile_cap));
  w->first_tile = reinterpret_cast<Tile*>(take(sizeof(Tile) * pairs));
  w->valid = reinterpret_cast<uint8_t*>(take(8 * blocks));
  w->broken = reinterpret_cast<uint8_t*>(take(8 * blocks));
  w->part_m = reinterpret_cast<float*>(take(sizeof(float) * pairs * 4 * kRows));
  w->part_den = reinterpret_cast<float*>(take(sizeof(float) * pairs * 4 * kRows));
  w->part_back = reinterpret_cast<float*>(take(sizeof(float) * pairs * 4 * kRows));
  w->part_o = reinterpret_cast<float*>(take(sizeof(float) * pairs * 2 * kRows * kD));
  w->stage = reinterpret_cast<__nv_bfloat16*>(take(2 * blocks * kKeys * kD));
  return off;
}

cudaError_t tc_forward(const PagedAttnProblem& p, void* ws, cudaStream_t st) {
  TcCall c;
  c.p = p;
  auto aligned = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n == 0; };
  c.p.out_32 = aligned(p.out, 32) && p.out_stride % 16 == 0;
  c.p.rope_vec = p.rope_cos && p.rope_out % 32 == 0 && aligned(p.rope_cos, 16) &&
                 aligned(p.rope_sin, 16);
  c.s = tc_shape(p);
  tc_carve(c.s, static_cast<char*>(ws), &c.w);
  if (c.s.block_cap * kKeys > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  CUtensorMap map;
  // 64 keys x 128 dims a copy: two column blocks of 128 bytes as planes (2000
  // tiles of three blocks take 2% longer with a copy a column block)
  if (!make_tma_map_u8_3d(&map, c.w.stage, 128, static_cast<uint64_t>(c.s.block_cap) * kKeys, kD * 2,
                          kD / 64, 128, 128, kKeys, 2))
    return cudaErrorInvalidValue;
  CUtensorMap qmap = map;  // not read for fp32 rows
  if (p.bf16 && !make_tma_map_u8_3d(&qmap, p.q, kD * 2, p.H, kD * 2, p.total, p.q_stride * 2, 128, p.H,
                                    kRows / p.H))
    return cudaErrorInvalidValue;
  const size_t smem = sizeof(int) * 2 * (static_cast<size_t>(p.pages.n_seqs) + 1);
  const long long units =
      (c.s.block_cap * (kKeys / kUnit) + kStageThreads / 32 - 1) / (kStageThreads / 32);
  const int most = sm_count() * kStageBlocks - 1;
  cudaError_t e = launch_pdl(stage_kernel, dim3(1 + static_cast<unsigned>(units < most ? units : most)),
                             dim3(kStageThreads), smem, st, c);
  if (e != cudaSuccess) return e;
  auto attn = short_tiles(p, c.s) ? paged_attn_tc_kernel<true> : paged_attn_tc_kernel<false>;
  e = set_max_dynamic_smem(reinterpret_cast<const void*>(attn), kTcBytes);
  if (e != cudaSuccess) return e;
  e = launch_pdl(attn, dim3(2 * c.s.pairs), dim3(kTcThreads), kTcBytes, st, map, qmap,
                 c);
  const int rows = p.H * (c.s.tokens_per_tile < p.max_new ? c.s.tokens_per_tile : p.max_new);
  if (e != cudaSuccess || c.s.pairs == 1 || rows <= 0) return e;
  return launch_pdl(paged_attn_merge_kernel,
                    dim3((2 * rows + kMergeWarps - 1) / kMergeWarps, c.s.pairs - 1),
                    dim3(32 * kMergeWarps), 0, st, c);
}

// Two heads a warp share a key's reads (8 tokens of 64 heads on 2048 keys: 184
// us, 268 with one head); one where there are no more heads than warps, or so
// few tokens that more blocks are worth more (1 token: 100 us, 182 with two
// before the loads were put ahead). The keys are cut until every SM has a
// block, not below 64 a piece (1 token: 8 pieces, 666 us uncut; cut on to two
// blocks an SM, 16 tokens take 363 us instead of 341).
template <int kWords>
cudaError_t general_launch(const PagedAttnProblem& p, cudaStream_t st) {
  const int d = p.pages.nope + p.pages.rope_dim, sms = sm_count();
  const bool one = p.H <= kGenWarps ||
                   static_cast<long long>(p.total) * ((p.H + 15) / 16) * kGenParts <= sms;
  auto kernel = one ? paged_attn_general_kernel<1, kWords> : paged_attn_general_kernel<2, kWords>;
  const int heads = kGenWarps * (one ? 1 : 2), groups = (p.H + heads - 1) / heads;
  const int keys = p.window > 0 && p.window < p.max_len ? p.window : p.max_len;
  int parts = 1;
  while (parts < kGenParts && static_cast<long long>(p.total) * groups * parts < sms &&
         keys > 2 * kGenKeys * parts)
    parts *= 2;
  if (static_cast<long long>(p.total) * parts > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  auto bytes = [&](int dim) {
    return sizeof(float) * static_cast<size_t>(heads) * dim + 4 * static_cast<size_t>(kGenKeys) * gen_pitch(dim);
  };
  const void* fn = reinterpret_cast<const void*>(kernel);
  cudaError_t e = set_max_dynamic_smem(fn, static_cast<int>(bytes(64 * kWords)));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.total * parts, groups);
  cfg.blockDim = dim3(kGenThreads);
  cfg.dynamicSmemBytes = bytes(d);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, parts);
}

// The sums of a lane stay in registers: as many as the dims need, so that small
// rows do not pay for large ones.
cudaError_t general_forward(const PagedAttnProblem& p, cudaStream_t st) {
  const int d = p.pages.nope + p.pages.rope_dim;
  if (d <= 256) return general_launch<4>(p, st);
  if (d <= 640) return general_launch<10>(p, st);
  return d <= kMaxDim ? general_launch<kMaxDim / 64>(p, st) : cudaErrorInvalidValue;
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnProblem& p) {
  if (!tc_shape_ok(p) || p.total <= 0) return 0;
  TcWs w;
  return tc_carve(tc_shape(p), nullptr, &w);
}

cudaError_t paged_attn_forward(const PagedAttnProblem& p, void* ws, cudaStream_t st) {
  if (p.total <= 0) return cudaSuccess;
  if (tc_shape_ok(p)) return tc_forward(p, ws, st);
  return general_forward(p, st);
}

}  // namespace dsv4
