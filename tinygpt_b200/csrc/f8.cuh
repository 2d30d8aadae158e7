// f8.cuh — what the operators in 8 bits and those of routed experts share: e4m3 with a scale for every block of 128 entries, launchers.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kF8Block = 128;
constexpr int64_t f8_ld(int64_t k) { return (k + 15) / 16 * 16; }                           // bytes from row to row
constexpr int64_t f8_blocks(int64_t k) { return (k + kF8Block - 1) / kF8Block; }
constexpr int kMaxExperts = 1024;

#ifdef __CUDACC__
// The scale of a block whose largest magnitude has the bits `top` (as integers magnitudes order like numbers, and NaN comes out on top of them all).
// Never below the least normal number: its reciprocal is finite.
__device__ __forceinline__ float f8_scale(uint32_t top) {
  const float s = __fdiv_rn(__uint_as_float(top), 448.f);
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// fp32(t / s) of eight numbers → e4m3, nearest with ties to even, at most ±448, NaN stays.  With r = 1 / s, rounded, one correction of t·r is the
// quotient as a division rounds it (Markstein), as long as the remainder is not below the normal numbers: tiny blocks divide.
__device__ __forceinline__ uint2 f8_pack8(const float (&t)[8], float s) {
  const float r = __frcp_rn(s);
  const bool tiny = s < 1e-25f;
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = t[4 * h + e], a = v * r;
      q[e] = fmaf(fmaf(-a, s, v), r, a);
    }
    if (tiny) {
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(t[4 * h + e], s);
    }
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[1]), "f"(q[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[3]), "f"(q[2]));
    w[h] = (uint32_t)lo | (uint32_t)hi << 16;
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ uint32_t magnitude8(const float (&t)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
  return top;
}
// over the sixteen lanes that hold a block
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// four values of 8 bits as numbers
__device__ __forceinline__ float4 f8_unpack4(uint32_t w) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
  float4 v;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(v.x), "=f"(v.y) : "r"(lo));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(v.z), "=f"(v.w) : "r"(hi));
  return v;
}
#endif

// ---- rows in 8 bits (f8_rows.cu)
int launch_f8_rows(void* q, float* scale, const void* x, int64_t ld_x, int64_t x_rows, const int32_t* index, int64_t rows, int64_t k, cudaStream_t st);
int launch_silu_mul_f8(void* q, float* scale, const void* gate_up, int64_t rows, int64_t n, cudaStream_t st);

// ---- products, one matrix for all rows or one for each group of them (group_gemm.cu)
struct GroupProduct {
  void* y;
  const void* x;            // bf16 [rows, k], or 8 bits [rows, f8_ld(k)] with x_scale [f8_blocks(k), rows]
  const float* x_scale;     // null: bf16
  const void* w;            // [experts, n, k] alike, w_scale [experts, f8_blocks(n), f8_blocks(k)]
  const float* w_scale;
  const int32_t* starts;    // [experts + 1], or null: one group of all rows
  const void* bias;         // bf16 [n] or null
  int64_t rows, experts, n, k;
};
int launch_group_product(const GroupProduct& p, cudaStream_t st);

// ---- rows by expert and back (experts.cu)
int launch_expert_order(int32_t* starts, int32_t* source, int32_t* place, const int32_t* chosen, int64_t rows, int64_t top, int64_t experts, cudaStream_t st);
int launch_expert_combine(void* out, const void* y, const int32_t* place, const float* weights, int64_t rows, int64_t top, int64_t n, cudaStream_t st);

}  // namespace b200
