// lowbit.cuh — what the operators over values of 4 bits share: the mma.sync product, nibbles as bf16 operands, launchers.
#pragma once
#include "common.cuh"

namespace b200 {

#ifdef __CUDACC__
// D += A·B, m16n8k16; lane 4r + c: D {(r, 2c), (r, 2c + 1), (r + 8, 2c), (r + 8, 2c + 1)}, A pairs of columns {(r, 2c), (r + 8, 2c), (r, 2c + 8), (r + 8, 2c + 8)},
// B pairs of rows {2c, 2c + 8} of column r
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
constexpr uint32_t kBf16Ones = 0x3f803f80u;

// Eight nibbles → 128 + nibble as four pairs of bf16: pair i is {bits 4i, bits 16 + 4i}.  0x4300 | v is 128 + v in bf16 (from 128 to 255 a step is 1).  The
// 128, and the 8 that makes a nibble a value, are taken off the sums: Σ (128 + nibble)·x − 136·Σ x, which costs one more product where a subtraction here
// would cost one instruction a pair; in fp32 the detour moves a sum by some 2^-17 of it.
constexpr float kNibbleOff = 136.f;
__device__ __forceinline__ void nibbles_128(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(a[i]) : "r"(w >> (4 * i)));   // (w & mask) | 128
}
// the same, less 136: exact
__device__ __forceinline__ void nibbles_bf16(uint32_t w, uint32_t (&a)[4]) {
  const uint32_t kOff = 0x43084308u;
  nibbles_128(w, a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a[i]), *reinterpret_cast<const __nv_bfloat162*>(&kOff));
    a[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}
#endif

// ---- Linears over weights of 4 bits (w4.cu; w4_gemm.cu: any number of rows, on tcgen05)
int launch_w4_gemm(void* y, const void* x, const b200_w4_weight& w, const void* bias, int64_t m, cudaStream_t st);
int64_t w4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k);
int launch_w4_linear(void* y, const void* x, const b200_w4_weight& w, const void* bias, int64_t m, void* workspace, cudaStream_t st);
int launch_w4_dequant(void* out, const b200_w4_weight& w, cudaStream_t st);

}  // namespace b200
