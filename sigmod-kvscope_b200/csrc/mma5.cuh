// The fifth-generation tensor cores' instructions (tcgen05) that the attention kernels use.
#pragma once

#include "ekv_common.cuh"

namespace ekv {

__device__ __forceinline__ void tmem_ld32(float* r, uint32_t addr) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}

// Waits for the loads; naming the values keeps their first use behind the wait.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One lane of the converged warp, always the same one. The issuing code goes by this vote and not by the lane's
// number, and its addresses are made of values that are the same in the whole warp: then the tensor-core instructions
// take them from uniform registers (with per-lane ones each instruction took 115 cycles to issue, twice its work).
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
  return chosen != 0;
}

// A shared-memory operand in the 128-byte swizzle, in two words: where it starts with the distance `lead` in bytes
// between 64-element groups of the major dimension, and (constant) 1024 bytes between groups of eight rows.
__device__ __forceinline__ uint32_t operand_low(uint32_t addr, uint32_t lead) { return (addr & 0x3ffff) >> 4 | (lead >> 4) << 16; }
constexpr uint32_t kOperandHigh = 1024u >> 4 | 1u << 14 | 2u << 29;

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kOperandHigh)
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kOperandHigh)
      : "memory");
}

// Two float32 values to an instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

// 2^x and 2^y, at least 2^-126, on the FMA pipes, for a part of the exponentials where the special-function units are what a
// kernel waits for. x = n + f with n the nearest whole number (adding 1.5 2^23 leaves it in the low bits) and |f| <= 1/2; 2^f
// by the polynomial of degree 5 through the Chebyshev nodes of [-1/2, 1/2], 2.2e-7 off at most with its float32 roundings
// (ex2.approx: 2^-22); 2^n from its exponent bits. NaN stays NaN.
__device__ __forceinline__ void exp2_pair(float& x, float& y) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(y));
  const uint64_t v = pair_of(x, y), t = add_pair(v, pair_of(12582912.f, 12582912.f));
  const uint64_t f = fma_pair(add_pair(t, pair_of(-12582912.f, -12582912.f)), pair_of(-1.f, -1.f), v);
  uint64_t r = fma_pair(f, pair_of(1.3390863e-3f, 1.3390863e-3f), pair_of(9.676032e-3f, 9.676032e-3f));
  r = fma_pair(r, f, pair_of(5.550357e-2f, 5.550357e-2f));
  r = fma_pair(r, f, pair_of(2.4022107e-1f, 2.4022107e-1f));
  r = fma_pair(r, f, pair_of(6.931472e-1f, 6.931472e-1f));
  r = fma_pair(r, f, pair_of(1.0000001f, 1.0000001f));
  float a, b;
  split(t, a, b);
  const float two_n = __int_as_float((__float_as_int(a) << 23) + 0x3f800000), two_m = __int_as_float((__float_as_int(b) << 23) + 0x3f800000);
  split(mul_pair(r, pair_of(two_n, two_m)), x, y);
}

// The instruction's shape and types: M query or token rows of 128, N columns, float32 sums; `values_rows`: the second
// operand's rows are the summed dimension (values), not its columns (keys).
template <bool HALF>
__host__ __device__ constexpr uint32_t mma_shape(uint32_t n, bool values_rows) {
  return 1u << 4 | (HALF ? 0u : 1u) << 7 | (HALF ? 0u : 1u) << 10 | (128u >> 4) << 24 | (n >> 3) << 17 | (values_rows ? 1u << 16 : 0u);
}

}  // namespace ekv
