// f8.cuh — what the operators in 8 bits and those of routed experts share: e4m3 with a scale for every block of 128 entries, launchers.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kF8Block = 128;
constexpr int64_t f8_ld(int64_t k) { return (k + 15) / 16 * 16; }                           // bytes from row to row
constexpr int64_t f8_blocks(int64_t k) { return (k + kF8Block - 1) / kF8Block; }
constexpr int kMaxExperts = 1024;

#ifdef __CUDACC__
// two fp32 numbers in a 64-bit register: one instruction multiplies and adds both
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// A block of 128 numbers t, eight a lane, in 8 bits.  `top`: the bits of their largest magnitude (as integers magnitudes order like numbers, and NaN comes out on top of
// them all).  s = max(fp32(top / 448), 2^-126): never below the least normal number, so that its reciprocal is finite.  value = e4m3(fp32(t / s)), nearest with
// ties to even, at most ±448; NaN stays.  With r = 1 / s, rounded, one correction of t·r is the quotient as a division rounds it (Markstein), as
// long as nothing is infinite and no remainder falls below the normal numbers: blocks of tiny and of huge numbers divide.  Eight divisions a lane in all blocks
// take the rows of 8 192 × 2 048 from 14.3 µs to 17.6; corrections one by one instead of in pairs to 14.8.
__device__ __forceinline__ uint2 f8_block(const float (&t)[8], uint32_t top, float& s) {
  constexpr float kR = 1.f / 448.f;
  const float m = __uint_as_float(top), a = m * kR;
  s = fmaf(fmaf(-a, 448.f, m), kR, a);
  const bool plain = s > 1e-25f && s < 1e35f;
  if (!plain) {
    s = __fdiv_rn(m, 448.f);
    s = s < 1.17549435e-38f ? 1.17549435e-38f : s;
  }
  float q[8];
  if (plain) {
    const float r = __frcp_rn(s);
    const uint64_t rr = pair_of(r, r), minus_s = pair_of(-s, -s);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint64_t tt = pair_of(t[e], t[e + 1]), v = mul_pair(tt, rr);
      const float2 both = halves(fma_pair(fma_pair(v, minus_s, tt), rr, v));
      q[e] = both.x;
      q[e + 1] = both.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(t[e], s);
  }
  uint16_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(w[e]) : "f"(q[2 * e + 1]), "f"(q[2 * e]));
  return make_uint2((uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16);
}
__device__ __forceinline__ uint32_t magnitude8(const float (&t)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
  return top;
}
// of eight bf16
__device__ __forceinline__ uint32_t magnitude8(const uint4& u) {
  auto larger = [](uint32_t a, uint32_t b) {
    uint32_t v;
    asm("max.u16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
    return v;
  };
  constexpr uint32_t kMask = 0x7fff7fffu;
  const uint32_t v = larger(larger(u.x & kMask, u.y & kMask), larger(u.z & kMask, u.w & kMask));
  return max(v << 16, v & 0xffff0000u);
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
// row i of x in 8 bits to every row place[i][0 … top − 1] of q and scale (dest_rows of them; a place outside them: nowhere)
int launch_f8_rows_to(void* q, float* scale, const void* x, const int32_t* place, int64_t rows, int64_t top, int64_t dest_rows, int64_t k, cudaStream_t st);
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
  // In front in the stream is the kernel that makes x, launched by the same call, and it lets this one start when all that came before it is done: nothing but
  // x and its scales has to be waited for.  What is read before that wait comes from L2 (W by TMA, groups and bias past L1).
  bool x_in_front = false;
};
int launch_group_product(const GroupProduct& p, cudaStream_t st);
// rows of a tile (0: group_gemm_wide.cu's) and CTAs to a tile that such a call takes
void group_way(const GroupProduct& g, bool f8, int32_t* rows, int32_t* splits);

// ---- rows by expert and back (experts.cu)
int launch_expert_order(int32_t* starts, int32_t* source, int32_t* place, const int32_t* chosen, int64_t rows, int64_t top, int64_t experts, cudaStream_t st);
int launch_expert_combine(void* out, const void* y, const int32_t* place, const float* weights, int64_t rows, int64_t top, int64_t n, cudaStream_t st);

}  // namespace b200
