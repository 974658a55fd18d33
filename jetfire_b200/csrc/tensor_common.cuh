// What the kernels on the fifth-generation tensor cores have in common: tcgen05 in inline PTX, bounded waits, arithmetic on pairs.
#pragma once

#include "jf_common.cuh"

namespace jf {

constexpr int kSlabBytes = 128 * 128;                 // 64 channels of a tile of 128 rows, 16 bits each, 128-byte swizzle
constexpr int kTileBytes = 2 * kSlabBytes;
constexpr uint64_t kTensorWaitNs = 2000000000ull;

// Where kernels of the current device that bring no record of their own note a wait that ran out.  An error that is there is taken and
// returned, unless `s` is being captured.
jf_status_t wait_record(cudaStream_t s, int32_t** device);

// ---- tcgen05 ------------------------------------------------------------------------------
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// all products issued so far by this thread, on `bar`
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
#define JF_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define JF_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of the lane's row
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* x) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : JF_R8(x, 0), JF_R8(x, 8), JF_R8(x, 16), JF_R8(x, 24)
      : "r"(at));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::JF_W8(x, 0), JF_W8(x, 8), JF_W8(x, 16), JF_W8(x, 24), "r"(at)
      : "memory");
}
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded.  An attempt lasts 120 cycles or so; the loop is four instructions, since warps that wait take issue slots from those that compute (the
// loop as the compiler makes it was 20, and half of what a kernel with many roles issued).  Most waits end within a few attempts; the
// clock that bounds the others is read only after that (a read of it in front of every wait that did not end at once took
// 0.4 us of each step).
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 0;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 q, n, 1000;\n\t"
      "@q bra AGAIN;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0 || mbar_wait(bar, parity, kTensorWaitNs);
}
// by a whole warp, which goes on or gives up together
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait(bar, parity)); }

// Shared-memory operand: 128-byte swizzle, rows of 128 bytes in groups of eight (1024 bytes).  K-major operands (Q, K) step
// through a row's 128 bytes; the MN-major one (V: rows are keys, the contraction) has its 64-channel slabs kSlabBytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t smem, uint32_t lead_bytes) {
  return static_cast<uint64_t>(smem >> 4 & 0x3FFFu) | static_cast<uint64_t>(lead_bytes >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         1ull << 46 | 2ull << 61;
}
template <int DT> __device__ constexpr uint32_t instruction(bool b_mn_major) {
  constexpr uint32_t type = DT == JF_DTYPE_BF16 ? 1u : 0u;
  return 1u << 4 | type << 7 | type << 10 | (b_mn_major ? 1u << 16 : 0u) | (128u >> 3) << 17 | (128u >> 4) << 24;
}

// ---- arithmetic on pairs ----------------------------------------------------------------------
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void split(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// two values as 16 bits each, rounded to nearest.  (One instruction; single values take 8 cycles each on the special functions' unit, which
// was most of an item's end: three short sequences 11.2 -> 10.3 us.)
template <int DT> __device__ __forceinline__ uint32_t round2(float lo, float hi) {
  uint32_t d;
  if (DT == JF_DTYPE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// the largest of three, a NaN if there is one
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A row's output so far goes to another reference.
__device__ __forceinline__ void rescale(uint32_t o_at, float f) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t o[32];
    tmem_ld32(o_at + c * 32, o);
    tc_wait_ld();
#pragma unroll
    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
    tmem_st32(o_at + c * 32, o);
  }
}

}  // namespace jf
