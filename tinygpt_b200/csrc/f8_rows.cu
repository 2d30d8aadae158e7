// f8_rows.cu — rows of numbers → rows in 8 bits with a scale for every 128 entries, from bf16 rows (which may be picked by a list), from an RMS norm with or
// without the residual's sum in front, from a SiLU product; and back to fp32.
//
//   t: the row's numbers in fp32;  of every block of 128:  s = max(fp32(max|t| / 448), 2^-126),  value = e4m3(fp32(t / s))
//
// A norm needs no second look at its row: with z the row, t = z·w and inv = rsqrt(mean(z²) + eps) the normed row is inv·t, its blocks' largest entries
// are inv·max|t|, and in value = inv·t / (inv·s) the inv cancels.  So values come from t alone (a product of two bf16 numbers: exact) and
// inv only meets the scale.  All of it is bound by HBM: a row is read once, 16 bytes a lane, and sixteen lanes that hold a block find its largest entry by
// four shuffles.
#include "f8.cuh"

#include <algorithm>

namespace b200 {

namespace {

// eight entries i … i + 7 of a row of k bf16; zero behind its end.  WIDE: rows are whole 16-byte pieces.
template <bool WIDE>
__device__ __forceinline__ void load8(const __nv_bfloat16* row, int i, int k, float (&v)[8]) {
  if constexpr (WIDE) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (i < k) u = *reinterpret_cast<const uint4*>(row + i);
    unpack8(u, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e < k ? bf16_to_f(row[i + e]) : 0.f;
  }
}

// value and scale of eight entries of a block; a row's last piece may reach past its ld bytes
__device__ __forceinline__ void store8(uint8_t* q, float* scale, int64_t row, int64_t rows, int i, int64_t ld, int blocks, uint2 w, float s) {
  if (i < ld) *reinterpret_cast<uint2*>(q + row * ld + i) = w;
  if (i % kF8Block == 0 && i / kF8Block < blocks) scale[(int64_t)(i / kF8Block) * rows + row] = s;
}

// Sixteen lanes to a block, blocks in a row's order.  kList: row i of the result is row list[i] of x (list null: i).  kSilu: rows
// of x are [gate | up], k entries each.  kTo: row i of x goes to the rows list[i][0 … top − 1] of the result, whose `rows` there are.
// U blocks of a lane are on their way together: one at a time, 8 192 × 2 048 picked by a list took 20 µs, a kernel's length of latencies.
enum RowsKind { kList, kSilu, kTo };
// g / (1 + exp(−g)) within 2^-20 of it: exp2 (2^-22) of the product's rounded part, and what was rounded off it to first order, a reciprocal (2^-23), roundings; below 2^-119
// it may be 0.  A power past 2^126 is that, and what is then rounded off it is positive: no infinity meets a negative factor.  From 200 on the exponential is 0, and taken
// of 200: g times the constant passes the largest number at 2.36e38, and what is rounded off an infinity is one that the 0 would meet.  (12.3 µs for a product of 8 192 ×
// 1 024, 12.1 without that.)  The quotient and expf of silu_f took it from 12.5 to 16.5 µs.
__device__ __forceinline__ float silu_fast(float g) {
  const float h = fminf(g, 200.f);
  const float p = fminf(h * -1.44269504f, 126.f), rest = fmaf(h, -1.44269504f, -p) + h * -1.92596303e-8f;   // −log2 e in two parts
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(p));
  e = fmaf(e, rest * 0.693147181f, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;   // (a NaN of g is one here)
}
template <bool WIDE, RowsKind KIND, int U>
__global__ void __launch_bounds__(256) f8_rows_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const __nv_bfloat16* __restrict__ x, int64_t ld_x,
                                                      int64_t x_rows, const int32_t* __restrict__ list, int top, int64_t rows, int k, int blocks) {
  pdl_wait();
  pdl_trigger();
  constexpr int LOADS = KIND == kSilu ? 2 : 1;
  const int64_t ld = f8_ld(k), all = (KIND == kTo ? x_rows : rows) * blocks;
  const bool small = all < 1ll << 31;   // (a division of 64 bits: a hundred instructions)
  for (int64_t first = (int64_t)blockIdx.x * (16 * U); first < all; first += (int64_t)gridDim.x * (16 * U)) {   // (lanes of a warp stay together)
    int64_t row[U], from[U];
    int i[U];
    bool in[U];
    uint4 raw[U][LOADS];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t at = first + 16 * j + threadIdx.x / 16;
      row[j] = small ? (int64_t)((uint32_t)at / (uint32_t)blocks) : at / blocks;
      i[j] = (int)(at - row[j] * blocks) * kF8Block + threadIdx.x % 16 * 8;
      if (at >= all) row[j] = -1;
      from[j] = row[j];
    }
    if (KIND == kList && list != nullptr) {
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (row[j] >= 0) from[j] = list[row[j]];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      in[j] = row[j] >= 0 && from[j] >= 0 && from[j] < x_rows && i[j] < k;
      if constexpr (WIDE) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
          raw[j][l] = make_uint4(0, 0, 0, 0);
          if (in[j]) raw[j][l] = *reinterpret_cast<const uint4*>(x + from[j] * ld_x + l * k + i[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float t[8], s;
      uint32_t m;
      if constexpr (WIDE) {
        unpack8(raw[j][0], t);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = 0.f;
        if (in[j]) load8<false>(x + from[j] * ld_x, i[j], k, t);
      }
      if constexpr (KIND == kSilu) {
        float u[8];
        if constexpr (WIDE) {
          unpack8(raw[j][LOADS - 1], u);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = 0.f;
          if (in[j]) load8<false>(x + from[j] * ld_x + k, i[j], k, u);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = silu_fast(t[e]) * u[e];
      }
      if constexpr (WIDE && KIND != kSilu) m = magnitude8(raw[j][0]);
      else m = magnitude8(t);
      const uint2 w = f8_block(t, block_max(m), s);
      if (row[j] < 0) continue;
      if constexpr (KIND == kTo) {
        for (int l = 0; l < top; ++l) {
          const int64_t to = list[row[j] * top + l];
          if (to >= 0 && to < rows) store8(q, scale, to, rows, i[j], ld, blocks, w, s);
        }
      } else {
        store8(q, scale, row[j], rows, i[j], ld, blocks, w, s);
      }
    }
  }
}

// One CTA to a row, V pieces of 8 entries a thread; the CTA's next row is asked for before this one is summed (4 096 × 4 096 with a residual, a CTA for every row: 23.8 µs).
// The sum may lie where the row or the residual does: an entry is read and written by one thread.
template <bool WIDE, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) norm_f8_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, __nv_bfloat16* sum, const __nv_bfloat16* x,
                                                          const __nv_bfloat16* residual, const __nv_bfloat16* __restrict__ w, int64_t rows, int dim, int blocks,
                                                          float eps) {
  __shared__ float red[2][THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const int64_t ld = f8_ld(dim);
  uint4 rx[V], rr[V];   // WIDE: the row that comes next
  auto ask = [&](int64_t row) {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = (threadIdx.x + j * THREADS) * 8;
        rx[j] = rr[j] = make_uint4(0, 0, 0, 0);
        if (row < rows && i < dim) {
          rx[j] = *reinterpret_cast<const uint4*>(x + row * dim + i);
          if (residual != nullptr) rr[j] = *reinterpret_cast<const uint4*>(residual + row * dim + i);
        }
      }
    }
  };
  ask(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const int64_t base = row * dim;
    float t[V][8];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (threadIdx.x + j * THREADS) * 8;
      if constexpr (WIDE) unpack8(rx[j], t[j]);
      else load8<false>(x + base, i, dim, t[j]);
      if (residual != nullptr) {
        float r[8];
        uint32_t z[4];
        if constexpr (WIDE) unpack8(rr[j], r);
        else load8<false>(residual + base, i, dim, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[e] = pack2(t[j][2 * e] + r[2 * e], t[j][2 * e + 1] + r[2 * e + 1]);
          t[j][2 * e] = bf16_lo(z[e]);
          t[j][2 * e + 1] = bf16_hi(z[e]);
        }
        if constexpr (WIDE) {
          if (i < dim) *reinterpret_cast<uint4*>(sum + base + i) = make_uint4(z[0], z[1], z[2], z[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (i + e < dim) sum[base + i + e] = f_to_bf16(t[j][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(t[j][e], t[j][e], ss);
    }
    ask(row + gridDim.x);
    ss = warp_sum(ss);
    if (threadIdx.x % 32 == 0) red[turn][threadIdx.x / 32] = ss;   // (two of them: a warp may be a row ahead)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (threadIdx.x + j * THREADS) * 8;
      if (w != nullptr) {
        float g[8];
        load8<WIDE>(w, i, dim, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[j][e] *= g[e];
      }
    }
    __syncthreads();
    float tot = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) tot += red[turn][i];
    const float inv = __frsqrt_rn(tot / (float)dim + eps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float s;
      const uint2 v = f8_block(t[j], block_max(magnitude8(t[j])), s);
      store8(q, scale, row, rows, (threadIdx.x + j * THREADS) * 8, ld, blocks, v, s * inv);
    }
  }
}

// Rows that no CTA holds in registers: once over them for the sum, a second time (from L2) for the values.  512 × 32 768 23.8 µs (2.1 TB/s: four CTAs for every SM,
// and both ways' latencies in each).
template <bool WIDE>
__global__ void __launch_bounds__(1024) norm_f8_long_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, __nv_bfloat16* sum,
                                                            const __nv_bfloat16* x, const __nv_bfloat16* residual,
                                                            const __nv_bfloat16* __restrict__ w, int64_t rows, int dim, int blocks, float eps) {
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x, base = row * dim, ld = f8_ld(dim);
  float ss = 0.f;
  auto entry = [&](int i, float (&t)[8]) {
    load8<WIDE>(x + base, i, dim, t);
    if (residual != nullptr) {
      float r[8];
      load8<WIDE>(residual + base, i, dim, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = round_bf16(t[e] + r[e]);
    }
  };
  for (int i = threadIdx.x * 8; i < dim; i += 8192) {
    float t[8];
    entry(i, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(t[e], t[e], ss);
  }
  ss = warp_sum(ss);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = ss;
  __syncthreads();
  const float inv = __frsqrt_rn(warp_sum(red[threadIdx.x % 32]) / (float)dim + eps);
  for (int first = 0; first < blocks * kF8Block; first += 8192) {   // (all lanes take every turn)
    const int i = first + threadIdx.x * 8;
    float t[8], g[8];
    entry(i, t);
    if (residual != nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < dim) sum[base + i + e] = f_to_bf16(t[e]);
    }
    if (w != nullptr) {
      load8<WIDE>(w, i, dim, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] *= g[e];
    }
    float s;
    const uint2 v = f8_block(t, block_max(magnitude8(t)), s);
    store8(q, scale, row, rows, i, ld, blocks, v, s * inv);
  }
}

// Four entries a thread, four times; 16 bytes a lane side by side on the way out.  Bound by what it writes: 4 096 × 4 096 15.3 µs, 5.5 TB/s.
template <bool WIDE>
__global__ void __launch_bounds__(256) f8_dequant_kernel(float* __restrict__ out, const uint8_t* __restrict__ q, const float* __restrict__ scale, int64_t rows, int k,
                                                         int pieces) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = 4;
  const int64_t ld = f8_ld(k), all = rows * pieces;
  const bool small = all < 1ll << 31;
  for (int64_t first = (int64_t)blockIdx.x * (256 * U) + threadIdx.x; first < all; first += (int64_t)gridDim.x * (256 * U)) {
    uint32_t w[U];
    float s[U];
    int64_t row[U];
    int i[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t at = min(first + 256 * j, all - 1);   // (the last piece more than once)
      row[j] = small ? (int64_t)((uint32_t)at / (uint32_t)pieces) : at / pieces;
      i[j] = (int)(at - row[j] * pieces) * 4;
      w[j] = *reinterpret_cast<const uint32_t*>(q + row[j] * ld + i[j]);
      s[j] = scale[(int64_t)(i[j] / kF8Block) * rows + row[j]];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float4 a = f8_unpack4(w[j]);
      const float v[4] = {a.x * s[j], a.y * s[j], a.z * s[j], a.w * s[j]};
      float* const o = out + row[j] * k + i[j];
      if constexpr (WIDE) {
        *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i[j] + e < k) o[e] = v[e];
      }
    }
  }
}

unsigned ctas_for(int64_t work, int64_t each, int64_t most) { return (unsigned)std::max<int64_t>(1, std::min((work + each - 1) / each, most)); }

template <RowsKind KIND>
int launch_rows(void* q, float* scale, const void* x, int64_t ld_x, int64_t x_rows, const int32_t* list, int64_t top, int64_t rows, int64_t k, cudaStream_t st) {
  const int64_t blocks = f8_blocks(k), all = KIND == kTo ? x_rows : rows;
  const bool wide = k % 8 == 0 && ld_x % 8 == 0 && aligned16(x);
  // few blocks: one a lane, over as many SMs as there are
  const bool many = all * blocks >= 148 * 8 * 16 * 2;
  const auto f = !many ? (wide ? f8_rows_kernel<true, KIND, 1> : f8_rows_kernel<false, KIND, 1>) : wide ? f8_rows_kernel<true, KIND, 4> : f8_rows_kernel<false, KIND, 2>;
  const int each = !many ? 1 : wide ? 4 : 2;
  B200_CUDA(launch_pdl(f, dim3(ctas_for(all * blocks, 16 * each, 148 * 64)), dim3(256), 0, st, op_pdl(st), (uint8_t*)q, scale,
                       (const __nv_bfloat16*)x, ld_x, x_rows, list, (int)top, rows, (int)k, (int)blocks));
  return B200_OK;
}

template <bool WIDE>
auto norm_kernel(int64_t dim, int* threads) {
  const int64_t pieces = f8_blocks(dim) * 16;   // whole blocks: their lanes stay together
  struct Form { int threads, v; decltype(&norm_f8_kernel<WIDE, 64, 1>) f; };
  const Form forms[] = {{64, 1, norm_f8_kernel<WIDE, 64, 1>}, {128, 1, norm_f8_kernel<WIDE, 128, 1>}, {256, 1, norm_f8_kernel<WIDE, 256, 1>},
                        {256, 2, norm_f8_kernel<WIDE, 256, 2>}, {512, 2, norm_f8_kernel<WIDE, 512, 2>}, {512, 4, norm_f8_kernel<WIDE, 512, 4>}};
  for (const Form& f : forms)
    if (pieces <= f.threads * f.v) {
      *threads = f.threads;
      return f.f;
    }
  *threads = 1024;
  return decltype(&norm_f8_kernel<WIDE, 64, 1>)(norm_f8_long_kernel<WIDE>);
}

int check_rows(const char* what, const void* q, const void* scale, int64_t rows, int64_t k) {
  B200_CHECK_ARG(q && scale && rows >= 1 && k >= 1 && rows < 1ll << 31 && k <= 1 << 24, "%s: %lld rows of %lld out of range, or a null pointer", what, (long long)rows,
                 (long long)k);
  B200_CHECK_ARG(aligned16(q), "%s: rows of 8 bits must be 16-byte aligned", what);
  return B200_OK;
}

}  // namespace

int launch_f8_rows(void* q, float* scale, const void* x, int64_t ld_x, int64_t x_rows, const int32_t* index, int64_t rows, int64_t k, cudaStream_t st) {
  return launch_rows<kList>(q, scale, x, ld_x, x_rows, index, 0, rows, k, st);
}
int launch_f8_rows_to(void* q, float* scale, const void* x, const int32_t* place, int64_t rows, int64_t top, int64_t dest_rows, int64_t k, cudaStream_t st) {
  return launch_rows<kTo>(q, scale, x, k, rows, place, top, dest_rows, k, st);
}
int launch_silu_mul_f8(void* q, float* scale, const void* gate_up, int64_t rows, int64_t n, cudaStream_t st) {
  return launch_rows<kSilu>(q, scale, gate_up, 2 * n, rows, nullptr, 0, rows, n, st);
}

}  // namespace b200

extern "C" {

int b200_f8_rows_bf16(void* q, float* scale, const void* x, int64_t ld_x, int64_t x_rows, const int32_t* index, int64_t rows, int64_t k, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_rows("f8_rows", q, scale, rows, k)) != B200_OK) return rc;
  B200_CHECK_ARG(x && ld_x >= k && ld_x < 1ll << 40 && x_rows >= (index ? 1 : rows) && x_rows < 1ll << 31, "f8_rows: %lld rows %lld apart, or a null pointer",
                 (long long)x_rows, (long long)ld_x);
  return launch_f8_rows(q, scale, x, ld_x, x_rows, index, rows, k, (cudaStream_t)stream);
}

int b200_silu_mul_f8(void* q, float* scale, const void* gate_up, int64_t rows, int64_t n, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_rows("silu_mul_f8", q, scale, rows, n)) != B200_OK) return rc;
  B200_CHECK_ARG(gate_up, "silu_mul_f8: null pointer");
  return launch_silu_mul_f8(q, scale, gate_up, rows, n, (cudaStream_t)stream);
}

int b200_rmsnorm_f8(void* q, float* scale, void* sum, const void* x, const void* residual, const void* w, int64_t rows, int64_t dim, float eps, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_rows("rmsnorm_f8", q, scale, rows, dim)) != B200_OK) return rc;
  B200_CHECK_ARG(x && (residual == nullptr) == (sum == nullptr), "rmsnorm_f8: null pointer, or a sum without a residual");
  int threads = 0;
  const bool wide = dim % 8 == 0 && aligned16(x, residual, sum, w);
  const auto f = wide ? norm_kernel<true>(dim, &threads) : norm_kernel<false>(dim, &threads);
  const cudaStream_t st = (cudaStream_t)stream;
  const unsigned ctas = threads == 1024 ? (unsigned)rows : (unsigned)std::min<int64_t>(rows, 148 * (1024 / threads));   // 32 warps to an SM
  B200_CUDA(launch_pdl(f, dim3(ctas), dim3(threads), 0, st, op_pdl(st), (uint8_t*)q, scale, (__nv_bfloat16*)sum, (const __nv_bfloat16*)x,
                       (const __nv_bfloat16*)residual, (const __nv_bfloat16*)w, rows, (int)dim, (int)f8_blocks(dim), eps));
  return B200_OK;
}

int b200_f8_rows_dequant(float* out, const void* q, const float* scale, int64_t rows, int64_t k, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_rows("f8_rows_dequant", q, scale, rows, k)) != B200_OK) return rc;
  B200_CHECK_ARG(out, "f8_rows_dequant: null pointer");
  const int pieces = (int)((k + 3) / 4);
  const cudaStream_t st = (cudaStream_t)stream;
  const auto f = k % 4 == 0 && aligned16(out) ? f8_dequant_kernel<true> : f8_dequant_kernel<false>;
  B200_CUDA(launch_pdl(f, dim3(ctas_for(rows * pieces, 256 * 4, 148 * 32)), dim3(256), 0, st, op_pdl(st), out, (const uint8_t*)q, scale, rows, (int)k, pieces));
  return B200_OK;
}

}  // extern "C"
