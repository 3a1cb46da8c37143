// norm.cu - RMS norm of rows with the residual's addition and an 8-bit
// output, and the write of new latents into their pages.
//
//   v = x + residual,  y = v / sqrt(mean v^2 + eps) * gain
//   per 128 columns: 2^e the smallest power of two with max |y| <= 448 2^e,
//   codes = E4M3(y / 2^e)
//
// One read and one write: a row stays with its threads, eight consecutive values a
// vector, so that 16 lanes hold a block of 128 and its maximum is four shuffles. Sum and square are fp32 from the inputs' sum on;
// each output is rounded once, from fp32.
#include "norm.cuh"

#include <cmath>
#include <type_traits>
#include <cuda_bf16.h>

#include "launch.cuh"
#include "umma.cuh"

namespace dsv4 {
namespace {

constexpr int kVec = 8;  // values of a vector

// Eight values as they lie in memory, so that several can be asked for before
// the first is turned into floats.
template <bool kBf16>
struct Raw {
  uint4 w[kBf16 ? 1 : 2];
  // Rows that are not whole aligned vectors are read and written value by value (4096
  // BF16 rows of 7167: 131 us, 50 where they are 7168 wide).
  __device__ __forceinline__ void load(const void* row, int i, int n, bool wide) {
    const char* p = static_cast<const char*>(row) + static_cast<size_t>(i) * (kBf16 ? 2 : 4);
    if (wide && n >= kVec) {
#pragma unroll
      for (int k = 0; k < (kBf16 ? 1 : 2); ++k) w[k] = reinterpret_cast<const uint4*>(p)[k];
      return;
    }
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      v[k] = k >= n  ? 0u
             : kBf16 ? reinterpret_cast<const uint16_t*>(p)[k]
                     : reinterpret_cast<const uint32_t*>(p)[k];
    if (kBf16) {
      w[0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    } else {
      w[0] = make_uint4(v[0], v[1], v[2], v[3]);
      w[kBf16 ? 0 : 1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
  __device__ __forceinline__ float get(int k) const {
    const uint4& u = w[kBf16 ? 0 : k / 4];
    const int i = kBf16 ? k / 2 : k % 4;
    const uint32_t x = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
    if (!kBf16) return __uint_as_float(x);
    return __uint_as_float((k & 1) ? x & 0xFFFF0000u : x << 16);
  }
};

template <bool kBf16>
__device__ __forceinline__ void store8(void* row, int i, int n, bool wide, const float (&v)[kVec]) {
  if (kBf16) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(row) + i;
    if (wide) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      return;
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (k < n) p[k] = __float2bfloat16_rn(v[k]);
  } else {
    float* p = static_cast<float*>(row) + i;
    if (wide) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
      return;
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (k < n) p[k] = v[k];
  }
}

// Eight E4M3 codes of v * inv, low byte first; an exact zero of either sign is +0,
// as the cache's other writers have it.
__device__ __forceinline__ uint2 codes8(const float (&v)[kVec], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    unsigned short t;
    asm("{ .reg .b16 h; cvt.rn.satfinite.e4m3x2.f32 h, %2, %1; mov.b16 %0, h; }"
        : "=h"(t) : "f"(fmaf(v[2 * k], inv, 0.f)), "f"(fmaf(v[2 * k + 1], inv, 0.f)));
    h[k] = t;
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// The magnitude bits order like the magnitudes, infinities and NaN above all.
__device__ __forceinline__ uint32_t top8(const float (&v)[kVec]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int k = 1; k + 1 < kVec; k += 2)
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[k])), "f"(fabsf(v[k + 1])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[kVec - 1])));
  return __float_as_uint(m);
}

// Whether a row's mean of squares and eps add up to more than fp32 holds (values
// from 1.8e19 on; NaN) or to so little that squares have lost bits. Its values are
// then squared again, times square_scale (2^-76 or 2^76), eps times its square.
__device__ __forceinline__ bool square_odd(float sum) {
  constexpr uint32_t kLow = 0x0DA24260u, kHigh = 0x7F61B1E6u;  // 1e-30, 3e38
  return __float_as_uint(sum) - kLow > kHigh - kLow;
}
__device__ __forceinline__ float square_scale(float sum) {
  return sum < 1.f ? 7.555786372591432e22f : 1.3234889800848443e-23f;
}

struct NormArgs {
  NormProblem p;
  int threads;                       // of a row
  bool wide_x, wide_r, wide_s, wide_o, wide_g, wide_c;  // whole aligned vectors
};

// The row that its threads hold in v: sum, norm, output. Whole block.
//
// 4096 BF16 rows of 7168 with residual, sum, normed rows and codes: 56.7 us, 4.66
// TB/s of the 6.45 that a copy reaches: a block's reads, meeting and writes follow
// one another, and the registers hold four rows an SM, not quite: above 4,096
// columns a thread's 64 spill some 140 bytes (fp32 rows 290; three blocks an SM,
// which spill nothing, took 58.6 us). fp32 rows with residual, sum and codes 86 us,
// 4.4 TB/s (BF16 50). Rows streamed through shared memory by blocks that stay took
// 67 us.
template <bool kBf16, int kVecs>
__device__ __forceinline__ void finish_row(const NormArgs& a, long long row, bool live, int tid,
                                           float (&v)[kVecs][kVec], float* part) {
  const NormProblem& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kSize = kBf16 ? 2 : 4;
  auto at = [&](const void* base, long long stride) {
    return static_cast<const char*>(base) + row * stride * kSize;
  };
  float squares = 0.f;
  if (p.sum && live) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int i = (tid + j * a.threads) * kVec, n = min(kVec, p.width - i);
      if (n > 0) store8<kBf16>(const_cast<char*>(at(p.sum, p.sum_stride)), i, n, a.wide_s, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
#pragma unroll
    for (int k = 0; k < kVec; ++k) squares = fmaf(v[j][k], v[j][k], squares);
  // the gain is on its way meanwhile
  Raw<true> gain[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int i = (tid + j * a.threads) * kVec, n = min(kVec, p.width - i);
    gain[j] = Raw<true>{make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u)};  // ones
    if (p.gain && n > 0) gain[j].load(p.gain, i, n, a.wide_g);
  }
  // over the row's warps
  const int warps = a.threads >> 5, first = warp - (tid >> 5);
  auto row_sum = [&](float s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (warps > 1) {
      if (lane == 0) part[warp] = s;
      __syncthreads();
      s = lane < warps ? part[first + lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    return s;
  };
  float mean = row_sum(squares) / p.width, eps = p.eps;
  // All rows of a block take the step together.
  const bool odd = square_odd(mean + eps);
  if (__syncthreads_or(odd)) {
    const float scale = square_scale(mean + eps);
    squares = 0.f;
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const float d = v[j][k] * scale;
        squares = fmaf(d, d, squares);
      }
    const float m = row_sum(squares) / p.width;
    if (odd) {
      mean = m;
      eps = eps * scale * scale;
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int k = 0; k < kVec; ++k) v[j][k] *= scale;
    }
  }
  const float rs = rsqrtf(mean + eps);
  const int blocks = (p.width + 127) / 128;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int i = (tid + j * a.threads) * kVec, n = min(kVec, p.width - i);
    const bool in = live && n > 0;
#pragma unroll
    for (int k = 0; k < kVec; ++k)  // (0 behind the row's end, but in rows that are NaN)
      v[j][k] = v[j][k] * rs * gain[j].get(k);
    if (p.out && in) store8<kBf16>(const_cast<char*>(at(p.out, p.out_stride)), i, n, a.wide_o, v[j]);
    uint32_t top = top8(v[j]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    uint2 c = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);  // an infinity or NaN makes the block NaN
    uint32_t e8 = 255;
    if (top < 0x7F800000u) {
      // the exponent of top / 448, rounded up
      e8 = (__float_as_uint(fmaxf(__uint_as_float(top), 1e-4f) * (1.0f / 448.0f)) + 0x7FFFFFu) >> 23;
      c = codes8(v[j], __uint_as_float((254u - e8) << 23));
    }
    if (!in) continue;
    uint8_t* to = p.codes + row * p.width + i;
    if (a.wide_c) {
      *reinterpret_cast<uint2*>(to) = c;
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        if (k < n) to[k] = static_cast<uint8_t>((k < 4 ? c.x : c.y) >> (8 * (k & 3)));
    }
    if ((tid & 15) == 0) p.scales[row * blocks + i / 128] = static_cast<uint8_t>(e8);
  }
}

// kVecs vectors a thread; blockDim.x / threads rows a block.
template <bool kBf16, int kVecs, int kMost>
__global__ void __launch_bounds__(kMost, 1024 / kMost) norm_quant_kernel(const NormArgs a) {
  __shared__ float part[32];
  const NormProblem& p = a.p;
  const int sub = threadIdx.x / a.threads, tid = threadIdx.x - sub * a.threads;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / a.threads) + sub;
  const bool live = row < p.rows;
  constexpr int kSize = kBf16 ? 2 : 4;
  pdl_wait();
  pdl_trigger();
  float v[kVecs][kVec];
  {
    Raw<kBf16> x[kVecs], r[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int i = (tid + j * a.threads) * kVec, n = live ? min(kVec, p.width - i) : 0;
      x[j] = Raw<kBf16>{};
      if (n > 0) x[j].load(static_cast<const char*>(p.x) + row * p.x_stride * kSize, i, n, a.wide_x);
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int i = (tid + j * a.threads) * kVec, n = live && p.residual ? min(kVec, p.width - i) : 0;
      r[j] = Raw<kBf16>{};
      if (n > 0)
        r[j].load(static_cast<const char*>(p.residual) + row * p.residual_stride * kSize, i, n, a.wide_r);
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[j][k] = x[j].get(k) + r[j].get(k);
  }
  finish_row<kBf16, kVecs>(a, row, live, tid, v, part);
}

// A warp per latent: the non-RoPE dims eight a vector (a scale's 64 are eight
// lanes), the RoPE dims a pair a lane.
constexpr int kLatentWarps = 4;
struct LatentArgs {
  LatentWrite p;
  bool wide, wide_g;
};
template <bool kBf16>
__global__ void __launch_bounds__(32 * kLatentWarps) latent_write_kernel(const LatentArgs a) {
  const LatentWrite& p = a.p;
  const Fp8KvCache& c = p.cache;
  const int lane = threadIdx.x & 31;
  const long long i = static_cast<long long>(blockIdx.x) * kLatentWarps + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (i >= p.n) return;
  // all that it reads is asked for at once
  const void* x = static_cast<const char*>(p.kv) + i * p.stride * (kBf16 ? 2 : 4);
  auto value = [&](int k) {
    return kBf16 ? bf16_widen(static_cast<const uint16_t*>(x)[k]) : static_cast<const float*>(x)[k];
  };
  const int vecs = c.nope / kVec, pairs = c.rope_dim / 2;
  constexpr int kVecs = 2;  // 512 dims
  Raw<kBf16> in[kVecs];
  Raw<true> gain[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int at = lane + 32 * j;
    in[j] = Raw<kBf16>{};
    gain[j] = Raw<true>{};
    if (at < vecs) in[j].load(x, at * kVec, kVec, a.wide);
    if (at < vecs && p.gain) gain[j].load(p.gain, at * kVec, kVec, a.wide_g);
  }
  float p0 = 0.f, p1 = 0.f, co = 1.f, si = 0.f;  // the lane's first pair
  if (lane < pairs) {
    p0 = value(c.nope + 2 * lane);
    p1 = value(c.nope + 2 * lane + 1);
    if (p.rope_cos) {
      co = p.rope_cos[i * pairs + lane];
      si = p.rope_sin[i * pairs + lane];
    }
  }
  const long long r = p.rows[i];
  if (r < 0 || r >= c.rows) return;
  float v[kVecs][kVec];
  float squares = fmaf(p0, p0, p1 * p1);
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      v[j][k] = in[j].get(k);
      squares = fmaf(v[j][k], v[j][k], squares);
    }
  for (int q = lane + 32; q < pairs; q += 32) {
    const float x0 = value(c.nope + 2 * q), x1 = value(c.nope + 2 * q + 1);
    squares = fmaf(x0, x0, fmaf(x1, x1, squares));
  }
  float rs = 1.f, scale = 1.f;
  if (p.gain) {
    const float d = static_cast<float>(c.nope + c.rope_dim);
    auto warp_sum = [](float s) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      return s;
    };
    float mean = warp_sum(squares) / d, eps = p.eps;
    if (square_odd(mean + eps)) {
      scale = square_scale(mean + eps);
      squares = 0.f;
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int k = 0; k < kVec; ++k) squares = fmaf(v[j][k] * scale, v[j][k] * scale, squares);
      for (int q = lane; q < pairs; q += 32) {
        const float x0 = value(c.nope + 2 * q) * scale, x1 = value(c.nope + 2 * q + 1) * scale;
        squares = fmaf(x0, x0, fmaf(x1, x1, squares));
      }
      mean = warp_sum(squares) / d;
      eps = eps * scale * scale;
    }
    rs = rsqrtf(mean + eps);
  }
  uint8_t* codes = c.codes + r * c.nope;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int at = lane + 32 * j;
    if (p.gain) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[j][k] = v[j][k] * scale * rs * gain[j].get(k);
    }
    uint32_t top = top8(v[j]);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    // (the attention tells a broken latent by its codes: NaN under a scale of 1)
    uint2 q = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
    uint32_t e8 = 127;
    if (top < 0x7F800000u) {
      e8 = __float_as_uint(pow2_scale_448(__uint_as_float(top))) >> 23;
      q = codes8(v[j], __uint_as_float((254u - e8) << 23));
    }
    if (at >= vecs) continue;
    *reinterpret_cast<uint2*>(codes + at * kVec) = q;
    if ((lane & 7) == 0) c.scales[r * kKvScaleSlots + at / 8] = static_cast<uint8_t>(e8);
  }
  for (int q = lane; q < pairs; q += 32) {
    float x0 = p0, x1 = p1;
    if (q != lane) { x0 = value(c.nope + 2 * q); x1 = value(c.nope + 2 * q + 1); }
    if (p.gain) {
      x0 = x0 * scale * rs * bf16_widen(p.gain[c.nope + 2 * q]);
      x1 = x1 * scale * rs * bf16_widen(p.gain[c.nope + 2 * q + 1]);
    }
    if (p.rope_cos) {
      if (q != lane) { co = p.rope_cos[i * pairs + q]; si = p.rope_sin[i * pairs + q]; }
      const float y0 = x0 * co - x1 * si;
      x1 = x0 * si + x1 * co;
      x0 = y0;
    }
    uint16_t* to = c.rope + r * c.rope_dim + 2 * q;
    *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(x0, x1);  // rope_dim is even, rope aligned
  }
}

// Rows of whole vectors that start on a 16-byte boundary.
bool whole_vectors(const void* base, long long stride, int rows, int width, int size) {
  return width % kVec == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
         (rows <= 1 || stride * size % 16 == 0);
}

}  // namespace

cudaError_t norm_quant(const NormProblem& p, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  NormArgs a;
  a.p = p;
  const int size = p.bf16 ? 2 : 4;
  a.wide_x = whole_vectors(p.x, p.x_stride, p.rows, p.width, size);
  a.wide_r = whole_vectors(p.residual, p.residual_stride, p.rows, p.width, size);
  a.wide_s = whole_vectors(p.sum, p.sum_stride, p.rows, p.width, size);
  a.wide_o = whole_vectors(p.out, p.out_stride, p.rows, p.width, size);
  a.wide_g = p.width % kVec == 0 && reinterpret_cast<uintptr_t>(p.gain) % 16 == 0;
  a.wide_c = p.width % kVec == 0 && reinterpret_cast<uintptr_t>(p.codes) % 8 == 0;
  const int vecs = (p.width + kVec - 1) / kVec;
  // Vectors of a thread: rows of at most 256 threads while four are enough (4096
  // rows of 7168: 57 us; with two a thread 58, with one 85), wider rows up to
  // 1024.
  int per = 1;
  while (per < 4 && vecs > 256 * per) per *= 2;
  a.threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  if (a.threads > 1024) return cudaErrorInvalidValue;
  const int rows = a.threads >= 128 ? 1 : 128 / a.threads;
  const dim3 grid(static_cast<unsigned>((p.rows - 1) / rows + 1)), block(rows * a.threads);
  auto run = [&](auto bf16) {
    constexpr bool kB = decltype(bf16)::value;
    auto kernel = per == 1 ? norm_quant_kernel<kB, 1, 256> : per == 2 ? norm_quant_kernel<kB, 2, 256>
                  : a.threads <= 256 ? norm_quant_kernel<kB, 4, 256> : norm_quant_kernel<kB, 4, 1024>;
    return launch_pdl(kernel, grid, block, 0, st, a);
  };
  return p.bf16 ? run(std::true_type{}) : run(std::false_type{});
}

cudaError_t latent_write(const LatentWrite& p, cudaStream_t st) {
  if (p.n <= 0) return cudaSuccess;
  LatentArgs a;
  a.p = p;
  const int size = p.bf16 ? 2 : 4;
  a.wide = reinterpret_cast<uintptr_t>(p.kv) % 16 == 0 && (p.n <= 1 || p.stride * size % 16 == 0);
  a.wide_g = reinterpret_cast<uintptr_t>(p.gain) % 16 == 0;
  auto kernel = p.bf16 ? latent_write_kernel<true> : latent_write_kernel<false>;
  return launch_pdl(kernel, dim3(static_cast<unsigned>((p.n - 1) / kLatentWarps + 1)),
                    dim3(32 * kLatentWarps), 0, st, a);
}

}  // namespace dsv4
