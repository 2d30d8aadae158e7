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

__device__ __forceinline__ uint4 ld_once(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
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

// A CTA takes RT row tiles, a warp one of WARPS equal pieces of their columns, which come through a ring of its own in shared memory, 128 columns a stage; the
// pieces are summed in shared memory in their order.  Values enter the products exactly and a group's sums are scaled in fp32, so nothing is rounded to
// fewer bits before the result: as 128 + nibble, with Σ x of the group from a product with ones (kSums: with one tile of columns that costs less than
// the subtraction, and a zero needs the sum anyway), or as nibble − 8.  Nothing is saturated: one row × 28 672 × 4 096 with zeros takes 16.5 µs (3.8 TB/s), in which the ALU, which
// unpacks eight values in seven instructions of half rate, is busy for 53 % of the cycles, the issue slots for 55 and DRAM for 37; its 896 CTAs are two rounds on the SMs' 592
// places, and each fills rings of its own and sums over its warps.  32 rows (448 CTAs, one to an SM, 44.7 µs): tensor cores 39 %, issue 33, DRAM 15.
template <int NT, int RT, int WARPS, int GROUP, bool ZERO>
struct W4Shape {
  static constexpr int kStages = 2;   // (more take the room of a third and a fourth CTA: 1 / 16 / 32 rows × 28 672 × 4 096 with two 16.8 / 24.7 / 45.0 µs, three 17.8 / 25.5 / 46.8, four 19.1 / 27.4 / 47.9)
  static constexpr bool kSums = ZERO || NT == 1;
  static constexpr int kParts = 128 / GROUP;   // groups of a stage
  static constexpr int kSmall = RT * kParts * (ZERO ? 2 : 1) * 32;   // bytes of scales and zeros
  static constexpr int kStage = RT * 1024 + kSmall;
  static constexpr int kTotals = RT * NT * 4;
  static constexpr int kRing = kStages * kStage > kTotals * 128 ? kStages * kStage : kTotals * 128;
  static constexpr int kSmem = WARPS * kRing;
};
template <int NT, int RT, int WARPS, int GROUP, bool ZERO>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 32 / WARPS : 1) w4_linear_kernel(const W4Params p) {
  using S = W4Shape<NT, RT, WARPS, GROUP, ZERO>;
  constexpr int kSteps = 8 / S::kParts;   // products of a group
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int tiles = (p.n + 15) / 16, tile0 = blockIdx.x * RT;
  const int all = (p.blocks + 1) / 2, from = all * warp / WARPS, to = all * (warp + 1) / WARPS;
  uint8_t* const ring = smem + warp * S::kRing;
  pdl_wait();
  pdl_trigger();

  const uint4* q[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) q[t] = p.q + ((int64_t)min(tile0 + t, tiles - 1) * p.blocks + 2 * from) * 32 + lane;
  // this lane's part of the small numbers: of row tile and group of the stage j / 8, the scale or the zero of rows lane % 8, + 8
  constexpr int kEach = RT * S::kParts * (ZERO ? 2 : 1) * 8;
  const uint32_t* small[(kEach + 31) / 32];
#pragma unroll
  for (int e = 0; e < (kEach + 31) / 32; ++e) {
    const int j = (lane + 32 * e) / 8, t = j / S::kParts % RT;
    small[e] = (j >= RT * S::kParts ? p.zero : p.scale) + (int64_t)min(tile0 + t, tiles - 1) * p.groups * 8 + lane % 8;
  }
  auto fetch = [&](int i) {
    if (i < to) {
      uint8_t* dst = ring + i % S::kStages * S::kStage;
      const bool both = 2 * i + 1 < p.blocks;   // (an odd last block's neighbour meets zeros of x)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        cp_async16(dst + t * 1024 + lane * 16, q[t]);
        if (both) cp_async16(dst + t * 1024 + 512 + lane * 16, q[t] + 32);
        q[t] += 64;
      }
#pragma unroll
      for (int e = 0; e < (kEach + 31) / 32; ++e) {
        const int g = min(i * S::kParts + (lane + 32 * e) / 8 % S::kParts, p.groups - 1);
        if (kEach % 32 == 0 || lane + 32 * e < kEach) cp_async4(dst + RT * 1024 + (lane + 32 * e) * 4, small[e] + g * 8);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int a = 0; a < S::kStages - 1; ++a) fetch(from + a);
  // rows past m have the last row's numbers: their columns of the products go nowhere
  const __nv_bfloat16* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = p.x + (int64_t)min(t * 8 + r, p.m - 1) * p.k + 8 * c;
  float total[RT][NT][4] = {};
  for (int i = from; i < to; ++i) {
    uint4 xb[NT][4];
    const bool full = (i + 1) * 128 <= p.k;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (full) xb[t][h] = *reinterpret_cast<const uint4*>(x[t] + i * 128 + h * 32);
        else xb[t][h] = i * 128 + h * 32 + c * 8 < p.k ? *reinterpret_cast<const uint4*>(x[t] + i * 128 + h * 32) : make_uint4(0, 0, 0, 0);
      }
    fetch(i + S::kStages - 1);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    const uint8_t* stage = ring + i % S::kStages * S::kStage;
    const uint32_t* nums = reinterpret_cast<const uint32_t*>(stage + RT * 1024);
    uint4 w[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[t][h] = *reinterpret_cast<const uint4*>(stage + t * 1024 + h * 512 + lane * 16);
#pragma unroll
    for (int h = 0; h < S::kParts; ++h) {
      float sum[NT][4] = {};
      if constexpr (S::kSums) {
#pragma unroll
        for (int j = h * kSteps; j < (h + 1) * kSteps; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma16816(sum[n], kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, j % 2 ? xb[n][j / 2].z : xb[n][j / 2].x, j % 2 ? xb[n][j / 2].w : xb[n][j / 2].y);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float acc[NT][4] = {};
#pragma unroll
        for (int j = h * kSteps; j < (h + 1) * kSteps; ++j) {
          const uint4 v = w[t][j / 4];
          const uint32_t word = j % 4 == 0 ? v.x : j % 4 == 1 ? v.y : j % 4 == 2 ? v.z : v.w;
          uint32_t f[4];
          if constexpr (S::kSums) nibbles_128(word, f);
          else nibbles_bf16(word, f);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma16816(acc[n], f[0], f[1], f[2], f[3], j % 2 ? xb[n][j / 2].z : xb[n][j / 2].x, j % 2 ? xb[n][j / 2].w : xb[n][j / 2].y);
        }
        const uint32_t s = nums[(t * S::kParts + h) * 8 + r], z = ZERO ? nums[((RT + t) * S::kParts + h) * 8 + r] : 0;
        const float s0 = bf16_lo(s), s1 = bf16_hi(s);
        const float z0 = ZERO ? -128.f - bf16_lo(z) : -kNibbleOff, z1 = ZERO ? -128.f - bf16_hi(z) : -kNibbleOff;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (S::kSums) {
            acc[n][0] = fmaf(z0, sum[n][0], acc[n][0]);
            acc[n][1] = fmaf(z0, sum[n][1], acc[n][1]);
            acc[n][2] = fmaf(z1, sum[n][0], acc[n][2]);
            acc[n][3] = fmaf(z1, sum[n][1], acc[n][3]);
          }
          total[t][n][0] = fmaf(s0, acc[n][0], total[t][n][0]);
          total[t][n][1] = fmaf(s0, acc[n][1], total[t][n][1]);
          total[t][n][2] = fmaf(s1, acc[n][2], total[t][n][2]);
          total[t][n][3] = fmaf(s1, acc[n][3], total[t][n][3]);
        }
      }
    }
    __syncwarp();   // the stage is free
  }
  cp_async_wait<0>();
  __syncwarp();
  float* const own = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) own[((t * NT + n) * 4 + e) * 32 + lane] = total[t][n][e];
  __syncthreads();
  constexpr int kRows = RT * 16;
  for (int o = threadIdx.x; o < kRows * NT * 8; o += WARPS * 32) {   // rows of W fastest
    const int row = o % kRows, col = o / kRows, n = blockIdx.x * kRows + row;
    if (col >= p.m) break;
    if (n >= p.n) continue;
    const int of = ((row / 16 * NT + col / 8) * 4 + row % 16 / 8 * 2 + col % 2) * 32 + row % 8 * 4 + col % 8 / 2;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float*>(smem + w * S::kRing)[of];
    p.y[(int64_t)col * p.n + n] = f_to_bf16(p.bias != nullptr ? v + bf16_to_f(p.bias[n]) : v);
  }
}

// W as bf16 [n, k], each value rounded once; with `bias_out`, the bias as fp32 too.  A warp takes kDequantBlocks tiles in a row: eight values in a row to a lane, four
// times a tile.
constexpr int kDequantBlocks = 2;
__global__ void __launch_bounds__(256) w4_dequant_kernel(__nv_bfloat16* out, const W4Params p, int group, float* bias_out) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int64_t tile = blockIdx.y;
  if (bias_out != nullptr && blockIdx.x == 0 && threadIdx.x < 16) {
    const int n = (int)tile * 16 + threadIdx.x;
    if (n < p.n) bias_out[n] = bf16_to_f(p.bias[n]);
  }
  const int b0 = (blockIdx.x * 8 + threadIdx.x / 32) * kDequantBlocks;
  if (b0 >= p.blocks) return;
  uint4 w[kDequantBlocks];
  uint32_t s[kDequantBlocks][2], z[kDequantBlocks][2];
#pragma unroll
  for (int b = 0; b < kDequantBlocks; ++b) {
    w[b] = ld_once(p.q + (tile * p.blocks + min(b0 + b, p.blocks - 1)) * 32 + lane);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t at = (tile * p.groups + min(((b0 + b) * 64 + h * 32) / group, p.groups - 1)) * 8 + r;
      s[b][h] = __ldg(p.scale + at);
      z[b][h] = p.zero != nullptr ? __ldg(p.zero + at) : 0x41004100u;   // 8, 8
    }
  }
#pragma unroll
  for (int b = 0; b < kDequantBlocks; ++b) {
    const uint32_t words[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k0 = (b0 + b) * 64 + h * 32 + c * 8;
      if (k0 >= p.k) continue;
      uint32_t v[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) nibbles_128(words[2 * h + t], v[t]);
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        // scale·value − scale·zero: the second product has 16 bits, so that one rounding is left to fp32
        const float sc = hi ? bf16_hi(s[b][h]) : bf16_lo(s[b][h]), off = -sc * (hi ? bf16_hi(z[b][h]) : bf16_lo(z[b][h]));
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2(fmaf(sc, bf16_lo(v[e / 2][2 * (e % 2) + hi]) - 128.f, off), fmaf(sc, bf16_hi(v[e / 2][2 * (e % 2) + hi]) - 128.f, off));
        const int64_t n = tile * 16 + r + 8 * hi;
        if (n < p.n) *reinterpret_cast<uint4*>(out + n * p.k + k0) = make_uint4(o[0], o[1], o[2], o[3]);
      }
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

template <int NT, int RT, int WARPS, int GROUP, bool ZERO>
int launch_kernel(const W4Params& p, cudaStream_t st) {
  using S = W4Shape<NT, RT, WARPS, GROUP, ZERO>;
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(w4_linear_kernel<NT, RT, WARPS, GROUP, ZERO>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); }));
  const int rows = RT * 16;
  B200_CUDA(launch_pdl(w4_linear_kernel<NT, RT, WARPS, GROUP, ZERO>, dim3((unsigned)((p.n + rows - 1) / rows)), dim3(WARPS * 32), S::kSmem, st, op_pdl(st), p));
  return B200_OK;
}
template <int NT, int RT, int WARPS>
int launch_rows(const W4Params& p, int group, cudaStream_t st) {
  const bool zero = p.zero != nullptr;
  if (group == 32) return zero ? launch_kernel<NT, RT, WARPS, 32, true>(p, st) : launch_kernel<NT, RT, WARPS, 32, false>(p, st);
  if (group == 64) return zero ? launch_kernel<NT, RT, WARPS, 64, true>(p, st) : launch_kernel<NT, RT, WARPS, 64, false>(p, st);
  return zero ? launch_kernel<NT, RT, WARPS, 128, true>(p, st) : launch_kernel<NT, RT, WARPS, 128, false>(p, st);
}

int launch_dequant(void* out, const W4Params& p, int group, float* bias_out, cudaStream_t st) {
  const dim3 grid((unsigned)((p.blocks + 8 * kDequantBlocks - 1) / (8 * kDequantBlocks)), (unsigned)((p.n + 15) / 16));
  B200_CUDA(launch_pdl(w4_dequant_kernel, grid, dim3(256), 0, st, op_pdl(st), (__nv_bfloat16*)out, p, group, bias_out));
  return B200_OK;
}

// Which way rows of x go.  Values exact (w4_linear_kernel): up to 32 rows, and up to 64 over a W whose unpacking for each eight of them costs little (µs at 64 rows,
// exact / on tcgen05: 4 096 × 4 096 17.7 / 11.2, 14 336 × 4 096 45.8 / 22.0).  That 32 rows are exact is a choice for exactness and not for speed: the widest weights would be as fast or
// faster on tcgen05 from some 20 rows on (28 672 × 4 096: 16 rows 24.3 / 38.7, 24 42.0 / 39.9, 32 44.7 / 40.2, with zeros of 32 columns 71 / 48; 32 × 14 336 × 4 096 24.5 / 20.8; 32 × 8 192 ×
// 4 096 12.6 / 13.6, 32 × 4 096 × 4 096 8.8 / 9.9).  W as bf16, unpacked into the products of 128 rows (w4_gemm.cu), up to 256.  More: W laid out
// as bf16 once, which costs its writing, and the general GEMM (µs, unpacked / laid out: 128 × 1 024 × 1 024 8.8 / 13.0, 128 × 4 096 × 4 096 12.9 / 18.8, 256 × 4 096 × 4 096
// 17.1 / 22.4, 256 × 4 096 × 14 336 37.7 / 62, 256 × 28 672 × 4 096 96 / 104; 300 × 896 × 896 9.9 / 8.8, 512 × 4 096 × 4 096 25.9 / 25.3, 512 × 14 336 × 4 096 94 / 72).  Both want n to be a
// multiple of 8; other widths go the exact way, 64 rows a launch, each of which reads W (128 × 50 257 × 1 024 118 µs, 50 264 channels 36).
enum class W4Way { exact, unpacked, laid_out };
W4Way w4_way(int64_t m, int64_t n, int64_t k) {
  if (n % 8 != 0 || m <= 32 || (m <= 64 && n * k <= 6 * 1000 * 1000)) return W4Way::exact;
  return m <= 256 ? W4Way::unpacked : W4Way::laid_out;
}
int64_t bf16_bytes(int64_t n, int64_t k) { return (n * k * 2 + 15) / 16 * 16; }

}  // namespace

int64_t w4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) { return w4_way(m, n, k) == W4Way::laid_out ? bf16_bytes(n, k) + n * 4 : 0; }

int launch_w4_linear(void* y, const void* x, const b200_w4_weight& w, const void* bias, int64_t m, void* workspace, cudaStream_t st) {
  W4Params p = params(w);
  p.bias = (const __nv_bfloat16*)bias;
  const W4Way way = w4_way(m, w.n, w.k);
  if (way == W4Way::unpacked) return launch_w4_gemm(y, x, w, bias, m, st);
  if (way == W4Way::laid_out) {
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
    // Two row tiles to a warp share the loads of x and its sums, where CTAs are left for all SMs (µs, one / two: 1 × 28 672 × 4 096 19.1 / 16.9, 8 × 8 192 × 4 096
    // 7.2 / 6.6, 32 × 4 096 × 4 096 11.8 / 8.8, but 1 × 4 096 × 4 096 4.3 / 4.5; 8 × 2 048 × 4 896 4.4 / 6.0, 32 × 1 024 × 4 096 6.2 / 8.1).  All warps of a CTA share a row tile's
    // columns: fewer warps to a tile are fewer sums, and lost at every size (28 672 × 4 096: 17.7, four warps a tile 19.3).
    // Four where the loads of x weigh more, at 17 to 32 rows, or its sums, at 9 to 16 with zeros of many groups, and a CTA is left for most SMs (two / four: 32 × 28 672 ×
    // 4 096 51.4 / 44.8, 24 × 8 192 × 4 096 14.6 / 11.8, 12 × 8 192 × 4 096 with zeros of 64 columns 10.7 / 8.6; with zeros of 128, 16 × 28 672 × 4 096 26.4 / 29.6, without
    // 24.5 / 28.3, one row of it 16.5 / 16.6).  What they hold does not always fit 255 registers: four tiles spill 8 to 256 bytes (all but those of 128 columns without zeros), two
    // with eight tiles of x 28 to 308, one with eight up to 156; one tile of x, kept to 64 registers for four CTAs to an SM, up to 32.
    const int tiles = (p.n + 15) / 16;
    const bool two = tiles >= 256, four = tiles >= 512;
    const int rc = p.m <= 8 ? (two ? launch_rows<1, 2, 8>(p, w.group, st) : launch_rows<1, 1, 8>(p, w.group, st))
                 : p.m <= 16 ? (four && p.zero != nullptr && w.group == 32 ? launch_kernel<2, 4, 8, 32, true>(p, st)
                                : four && p.zero != nullptr && w.group == 64 ? launch_kernel<2, 4, 8, 64, true>(p, st)
                                : two ? launch_rows<2, 2, 8>(p, w.group, st) : launch_rows<2, 1, 8>(p, w.group, st))
                 : p.m <= 32 ? (four ? launch_rows<4, 4, 8>(p, w.group, st)
                                : two ? launch_rows<4, 2, 8>(p, w.group, st) : launch_rows<4, 1, 8>(p, w.group, st))
                             : (two ? launch_rows<8, 2, 8>(p, w.group, st) : launch_rows<8, 1, 8>(p, w.group, st));
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
