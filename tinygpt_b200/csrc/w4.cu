// w4.cu — Linears over weights of 4 bits with group scales:  y = x·Wᵀ (+ bias),  W[n, k] = scale[n, k / group]·(value − zero[n, k / group]).
//
// Values lie in tiles of 16 rows × 64 columns, 512 bytes, [row tile][column block][lane][16 bytes]: what a lane takes of a tile is one 16-byte
// load, and each of its four words is the lane's part of the A operand of one m16n8k16 product (rows = output channels, columns =
// rows of x).  Word 2h + t of lane 4r + c: columns 32h + 8c + 4t + {0 … 3} of rows r and r + 8, so that the lane's part of x for
// the same four products is two 16-byte loads, and a group of 32 columns is two whole products.  Scales and zeros lie as [row tile][group][r]
// {row r, row r + 8}.
#include "lowbit.cuh"
#include "ops.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ uint4 ld_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

struct W4Params {
  __nv_bfloat16* y;
  const __nv_bfloat16* x;
  const uint4* q;
  const uint32_t* scale;
  const uint32_t* zero;
  const __nv_bfloat16* bias;
  int m, n, k, blocks, groups;
};

// A warp takes every kWarps-th column block of RT row tiles; the CTA's warps are summed in shared memory in their order.  Values enter the
// products as value − 8, exact in bf16, and a group's sums are scaled in fp32: nothing is rounded to fewer bits before the result.
template <int NT, int RT, int GROUP, bool ZERO>
__global__ void __launch_bounds__(kWarps * 32) w4_linear_kernel(const W4Params p) {
  constexpr int kParts = GROUP == 32 ? 2 : 1;   // groups of a column block (of 128: one for two blocks)
  constexpr int kUnroll = NT * RT <= 2 ? 4 : NT * RT <= 4 ? 2 : 1;
  constexpr int kSums = RT * NT * 4;
  __shared__ float red[kWarps][kSums][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int tile0 = blockIdx.x * RT, tiles = (p.n + 15) / 16;
  pdl_wait();
  pdl_trigger();
  const uint4* q[RT];
  const uint32_t *scale[RT], *zero[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t tile = min(tile0 + t, tiles - 1);
    q[t] = p.q + tile * p.blocks * 32 + lane;
    scale[t] = p.scale + tile * p.groups * 8 + r;
    zero[t] = p.zero + tile * p.groups * 8 + r;
  }
  const __nv_bfloat16* x[NT];
  bool has[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    has[i] = i * 8 + r < p.m;
    x[i] = p.x + (int64_t)(i * 8 + r) * p.k + 8 * c;
  }
  float total[RT][NT][4] = {};
#pragma unroll kUnroll
  for (int b = warp; b < p.blocks; b += kWarps) {
    uint4 w[RT], xb[NT][2];
    uint32_t s[RT][kParts], z[RT][kParts];
#pragma unroll
    for (int t = 0; t < RT; ++t) w[t] = ld_once(q[t] + (int64_t)b * 32);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xb[i][h] = has[i] && b * 64 + h * 32 + c * 8 < p.k ? __ldg(reinterpret_cast<const uint4*>(x[i] + b * 64 + h * 32)) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const int g = GROUP == 32 ? min(2 * b + h, p.groups - 1) : GROUP == 64 ? b : b / 2;
        s[t][h] = __ldg(scale[t] + (int64_t)g * 8);
        z[t][h] = ZERO ? __ldg(zero[t] + (int64_t)g * 8) : 0;
      }
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      constexpr int kHalves = 2 / kParts;
      float sum[NT][4];   // Σ x of the group, the same for every row
      if constexpr (ZERO) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.f;
#pragma unroll
          for (int e = 0; e < kHalves; ++e) {
            const uint4 v = xb[i][h + e];
            mma16816(sum[i], kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.x, v.y);
            mma16816(sum[i], kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.z, v.w);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float acc[NT][4] = {};
#pragma unroll
        for (int e = 0; e < kHalves; ++e) {
          uint32_t a[4];
          nibbles_bf16(h + e == 0 ? w[t].x : w[t].z, a);
#pragma unroll
          for (int i = 0; i < NT; ++i) mma16816(acc[i], a[0], a[1], a[2], a[3], xb[i][h + e].x, xb[i][h + e].y);
          nibbles_bf16(h + e == 0 ? w[t].y : w[t].w, a);
#pragma unroll
          for (int i = 0; i < NT; ++i) mma16816(acc[i], a[0], a[1], a[2], a[3], xb[i][h + e].z, xb[i][h + e].w);
        }
        const float s0 = bf16_lo(s[t][h]), s1 = bf16_hi(s[t][h]);
        const float z0 = 8.f - bf16_lo(z[t][h]), z1 = 8.f - bf16_hi(z[t][h]);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if constexpr (ZERO) {
            acc[i][0] = fmaf(z0, sum[i][0], acc[i][0]);
            acc[i][1] = fmaf(z0, sum[i][1], acc[i][1]);
            acc[i][2] = fmaf(z1, sum[i][2], acc[i][2]);
            acc[i][3] = fmaf(z1, sum[i][3], acc[i][3]);
          }
          total[t][i][0] = fmaf(s0, acc[i][0], total[t][i][0]);
          total[t][i][1] = fmaf(s0, acc[i][1], total[t][i][1]);
          total[t][i][2] = fmaf(s1, acc[i][2], total[t][i][2]);
          total[t][i][3] = fmaf(s1, acc[i][3], total[t][i][3]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][(t * NT + i) * 4 + e][lane] = total[t][i][e];
  __syncthreads();
  for (int o = threadIdx.x; o < kSums * 32; o += kWarps * 32) {   // rows of W fastest
    const int row = o % (16 * RT), col = o / (16 * RT);
    const int from = ((row / 16) * NT + col / 8) * 4 + (row % 16 / 8) * 2 + col % 2, at = row % 8 * 4 + col % 8 / 2;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w][from][at];
    const int n = tile0 * 16 + row;
    if (n < p.n && col < p.m) p.y[(int64_t)col * p.n + n] = f_to_bf16(p.bias != nullptr ? v + bf16_to_f(p.bias[n]) : v);
  }
}

// W as bf16 [n, k], each value rounded once; with `bias`, that as fp32 behind it.  A warp takes a tile: eight values in a row to a lane, four times.
__global__ void __launch_bounds__(256) w4_dequant_kernel(__nv_bfloat16* out, const W4Params p, int group, float* bias_out) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int64_t tile = blockIdx.y;
  if (bias_out != nullptr && blockIdx.x == 0 && threadIdx.x < 16) {
    const int n = (int)tile * 16 + threadIdx.x;
    if (n < p.n) bias_out[n] = bf16_to_f(p.bias[n]);
  }
  const int b = blockIdx.x * 8 + threadIdx.x / 32;
  if (b >= p.blocks) return;
  const uint4 w = ld_once(p.q + (tile * p.blocks + b) * 32 + lane);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k0 = b * 64 + h * 32 + c * 8;
    if (k0 >= p.k) break;
    const int64_t at = (tile * p.groups + k0 / group) * 8 + r;
    const uint32_t s = __ldg(p.scale + at), z = p.zero != nullptr ? __ldg(p.zero + at) : 0x41004100u;   // 8, 8
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const float sc = hi ? bf16_hi(s) : bf16_lo(s), off = 8.f - (hi ? bf16_hi(z) : bf16_lo(z));
      uint32_t o[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t a[4];
        nibbles_bf16(words[2 * h + t], a);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t v = a[2 * e + hi];
          o[2 * t + e] = pack2((bf16_lo(v) + off) * sc, (bf16_hi(v) + off) * sc);
        }
      }
      const int64_t n = tile * 16 + r + 8 * hi;
      if (n < p.n) *reinterpret_cast<uint4*>(out + n * p.k + k0) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

W4Params params(const b200_w4_weight& w) {
  W4Params p{};
  p.q = (const uint4*)w.q;
  p.scale = (const uint32_t*)w.scale;
  p.zero = (const uint32_t*)w.zero;
  p.n = w.n;
  p.k = w.k;
  p.blocks = (w.k + 63) / 64;
  p.groups = (w.k + w.group - 1) / w.group;
  return p;
}

template <int NT, int RT>
int launch_rows(const W4Params& p, int group, cudaStream_t st) {
  const dim3 grid((unsigned)(((p.n + 15) / 16 + RT - 1) / RT));
  const bool pdl = op_pdl(st), zero = p.zero != nullptr;
  const auto k = group == 32 ? (zero ? w4_linear_kernel<NT, RT, 32, true> : w4_linear_kernel<NT, RT, 32, false>)
                 : group == 64 ? (zero ? w4_linear_kernel<NT, RT, 64, true> : w4_linear_kernel<NT, RT, 64, false>)
                               : (zero ? w4_linear_kernel<NT, RT, 128, true> : w4_linear_kernel<NT, RT, 128, false>);
  B200_CUDA(launch_pdl(k, grid, dim3(kWarps * 32), 0, st, pdl, p));
  return B200_OK;
}

int launch_dequant(void* out, const W4Params& p, int group, float* bias_out, cudaStream_t st) {
  const dim3 grid((unsigned)((p.blocks + 7) / 8), (unsigned)((p.n + 15) / 16));
  B200_CUDA(launch_pdl(w4_dequant_kernel, grid, dim3(256), 0, st, op_pdl(st), (__nv_bfloat16*)out, p, group, bias_out));
  return B200_OK;
}

// Rows of x for which W is laid out as bf16 for the tcgen05 GEMM.
bool as_gemm(int64_t m, int64_t n) { return m > 64 && n % 8 == 0; }
int64_t bf16_bytes(int64_t n, int64_t k) { return (n * k * 2 + 15) / 16 * 16; }

}  // namespace

int64_t w4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) { return as_gemm(m, n) ? bf16_bytes(n, k) + n * 4 : 0; }

int launch_w4_linear(void* y, const void* x, const b200_w4_weight& w, const void* bias, int64_t m, void* workspace, cudaStream_t st) {
  W4Params p = params(w);
  p.bias = (const __nv_bfloat16*)bias;
  if (as_gemm(m, w.n)) {
    float* b = bias != nullptr ? (float*)((char*)workspace + bf16_bytes(w.n, w.k)) : nullptr;
    const int rc = launch_dequant(workspace, p, w.group, b, st);
    if (rc != B200_OK) return rc;
    return b != nullptr ? launch_gemm_bf16_bias(y, x, workspace, b, m, w.n, w.k, st)
                        : launch_linear_split_bf16(y, x, workspace, m, w.n, w.k, nullptr, st);
  }
  for (int64_t r = 0; r < m; r += 64) {
    p.m = (int)std::min<int64_t>(m - r, 64);
    p.x = (const __nv_bfloat16*)x + r * w.k;
    p.y = (__nv_bfloat16*)y + r * w.n;
    const int rc = p.m <= 8 ? launch_rows<1, 1>(p, w.group, st) : p.m <= 16 ? launch_rows<2, 1>(p, w.group, st)
                 : p.m <= 32 ? launch_rows<4, 1>(p, w.group, st) : launch_rows<8, 1>(p, w.group, st);
    if (rc != B200_OK) return rc;
  }
  return B200_OK;
}

int launch_w4_dequant(void* out, const b200_w4_weight& w, cudaStream_t st) { return launch_dequant(out, params(w), w.group, nullptr, st); }

}  // namespace b200

static int check_w4(const b200_w4_weight* w, const char* what) {
  using namespace b200;
  B200_CHECK_ARG(w && w->q && w->scale, "%s: null pointer", what);
  B200_CHECK_ARG(w->n >= 1 && w->n <= 16 * 65535 && w->k >= 8 && w->k % 8 == 0 && w->k <= 1 << 24, "%s: W [%d, %d] out of range (k a multiple of 8)", what,
                 w->n, w->k);
  B200_CHECK_ARG(w->group == 32 || w->group == 64 || w->group == 128, "%s: groups of %d (32, 64 or 128)", what, w->group);
  B200_CHECK_ARG(aligned16(w->q) && ((uintptr_t)w->scale & 3) == 0 && ((uintptr_t)w->zero & 3) == 0, "%s: misaligned weight", what);
  return B200_OK;
}

extern "C" {

int64_t b200_w4_workspace_bytes(int64_t m, int64_t n, int64_t k) { return m < 1 || n < 1 || k < 1 ? -1 : b200::w4_linear_workspace_bytes(m, n, k); }

int b200_w4_linear_bf16(void* y, const void* x, const b200_w4_weight* w, const void* bias, int64_t m, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_w4(w, "w4_linear")) != B200_OK) return rc;
  B200_CHECK_ARG(y && x && m >= 1 && m < 1 << 24, "w4_linear: m=%lld out of range, or a null pointer", (long long)m);
  B200_CHECK_ARG(aligned16(x), "w4_linear: x must be 16-byte aligned");
  B200_CHECK_ARG(w4_linear_workspace_bytes(m, w->n, w->k) == 0 || (workspace && aligned16(workspace, y)),
                 "w4_linear: %lld rows need a workspace, it and y 16-byte aligned", (long long)m);
  return launch_w4_linear(y, x, *w, bias, m, workspace, (cudaStream_t)stream);
}

int b200_w4_dequant_bf16(void* out, const b200_w4_weight* w, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_w4(w, "w4_dequant")) != B200_OK) return rc;
  B200_CHECK_ARG(out && aligned16(out), "w4_dequant: out must be 16-byte aligned");
  return launch_w4_dequant(out, *w, (cudaStream_t)stream);
}

}  // extern "C"
