// umma.cuh - tcgen05 primitives shared by the attention kernels: descriptors,
// MMA issue, TMEM loads and stores, bounded waits, E4M3 to BF16 conversion.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bulk.cuh"
#include "dsv4_common.cuh"

namespace dsv4 {
namespace {

constexpr unsigned kErrWait = 2u;  // device error bit: a wait in an attention kernel or a grouped product timed out
constexpr float kLog2e = 1.4426950408889634f;

// Byte offset of the 16-byte chunk (row, dc) in a 128-byte-swizzled tile
// whose 64-dim column blocks are `rows` rows tall (dc = dim / 8).
__device__ __forceinline__ uint32_t sw128_off(int row, int dc, int rows) {
  return static_cast<uint32_t>((dc >> 3) * rows * 128 + (row >> 3) * 1024 + (row & 7) * 128 +
                               (((dc & 7) ^ (row & 7)) << 4));
}

// UMMA shared-memory descriptor, 128-byte swizzle (layout type 2), sm_100
// version bit; addresses and offsets in 16-byte units.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) |
         (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of kind::f16: FP32 accumulate, BF16 A and B.
__host__ __device__ constexpr uint32_t umma_idesc_bf16(int m, int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// MMA issue, warp-converged: every lane of the MMA warp executes these, one
// elected lane (the same one each time) issues. A rolled single-lane issue
// loop runs several times slower than the tensor pipe. The _ts form takes
// A (M x 16, BF16 pairs packed along K) from TMEM.
__device__ __forceinline__ void umma_bf16_e(uint32_t d_tmem, uint64_t a, uint64_t b,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_ts_e(uint32_t d_tmem, uint32_t a_tmem, uint64_t b,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_e(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
          smem_addr(bar))
      : "memory");
}

// 2^x on the MUFU unit (ex2.approx.ftz: relative error ~2^-22, 2^-inf = +0).
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

#define DSV4_R32(X)                                                                          \
  X(0), X(1), X(2), X(3), X(4), X(5), X(6), X(7), X(8), X(9), X(10), X(11), X(12), X(13),  \
      X(14), X(15), X(16), X(17), X(18), X(19), X(20), X(21), X(22), X(23), X(24), X(25),  \
      X(26), X(27), X(28), X(29), X(30), X(31)
#define DSV4_OUT(i) "=r"(r[i])
#define DSV4_INOUT(i) "+r"(r[i])
#define DSV4_IN(i) "r"(r[i])

// 32 consecutive TMEM columns of this thread's lane (32x32b shape).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : DSV4_R32(DSV4_OUT)
      : "r"(taddr));
  // The wait names the registers so no use is scheduled before it.
  asm volatile("tcgen05.wait::ld.sync.aligned;" : DSV4_R32(DSV4_INOUT)::"memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          taddr),
      DSV4_R32(DSV4_IN)
      : "memory");
}
// The first 16 of r.
template <int N>
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[N]) {
  static_assert(N >= 16, "16 registers");
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Bounded wait that also gives up once another role has aborted.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        unsigned* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      if (err) atomicOr(err, kErrWait);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Four E4M3 codes (low byte first) times a power of two -> 2 x bf16x2; exact.
__device__ __forceinline__ uint2 e4m3x4_to_bf16(uint32_t w, float sc) {
  const uint32_t h01 = e4m3x2_to_f16x2(w & 0xFFFFu), h23 = e4m3x2_to_f16x2(w >> 16);
  const float2 f01 = __half22float2(*reinterpret_cast<const __half2*>(&h01));
  const float2 f23 = __half22float2(*reinterpret_cast<const __half2*>(&h23));
  return make_uint2(pack_bf16x2(f01.x * sc, f01.y * sc), pack_bf16x2(f23.x * sc, f23.y * sc));
}

// Four E4M3 codes times 2^(c - 127) -> 2 x bf16x2 on the integer and FMA
// pipes. Each code's 7 magnitude bits placed at BF16 bits 4-10 read as a
// BF16 number equal to the E4M3 value times 2^-120 (subnormal codes become
// BF16 subnormals, zero stays zero), the sign goes to bit 15, and one BF16
// multiply by k2 = 2^(c - 7) (exponent field c + 120) in both halves scales
// exactly. Valid for 10 <= c <= 134 (every product a normal BF16) and codes
// other than 0x7F/0xFF (NaN); the caller checks.
__device__ __forceinline__ uint2 e4m3x4_to_bf16_mul(uint32_t w, uint32_t k2) {
  const uint32_t m = w & 0x7F7F7F7Fu;
  uint32_t t0, t1, s0, s1, r0, r1;
  asm("prmt.b32 %0, %1, 0, 0x4140;" : "=r"(t0) : "r"(m));  // [b0, 0, b1, 0]
  asm("prmt.b32 %0, %1, 0, 0x4342;" : "=r"(t1) : "r"(m));  // [b2, 0, b3, 0]
  asm("prmt.b32 %0, %1, 0, 0x9484;" : "=r"(s0) : "r"(w));  // sign bytes of b0, b1
  asm("prmt.b32 %0, %1, 0, 0xB4A4;" : "=r"(s1) : "r"(w));  // sign bytes of b2, b3
  const uint32_t v0 = (t0 << 4) | (s0 & 0x80008000u), v1 = (t1 << 4) | (s1 & 0x80008000u);
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r0) : "r"(v0), "r"(k2));
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r1) : "r"(v1), "r"(k2));
  return make_uint2(r0, r1);
}

// Nonzero iff a byte of w is an E4M3 NaN code (0x7F or 0xFF).
__device__ __forceinline__ uint32_t e4m3_nan_bytes(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

}  // namespace
}  // namespace dsv4
