// w4_gemm.cu — Linears over weights of 4 bits for many rows, on the 5th-generation tensor cores:  yᵀ = W·xᵀ, [channels, rows].
//
// W is the A operand and comes from tensor memory: sixteen warps unpack its nibbles to bf16 (each weight rounded once) and store them there, 128 columns of W a
// stage, while TMA brings x as the B operand to shared memory.  W through shared memory would have to be written to it and read from it again
// for every product.  A stage takes 0.45 µs where 64 rows meet it and 0.54 at 128, of which the products need 0.27; without products and unpacking (170 instructions
// for 16 × 64 values) 0.42, without W's loads alone 0.42, without all three 0.22: what a stage needs goes on side by side and slows each other.  64 rows of
// 4 096 × 4 096 take 11.2 µs, of 14 336 × 4 096 22.0 (1.4 TB/s of W); 7 to 8 µs of a call are launch, first loads and the epilogue.  Pairs of CTAs that share x took as long
// (25 µs at 512 rows of 4 096 × 4 096), and so did shuffles in place of the neighbours' words below.
//
// The layout of W (w4.cu) has eight columns in a row together; the lane that stores to tensor memory wants two of every eight.  So it reads words of its
// three neighbours from shared memory, too, where they lie in an order that lets 32 lanes read side by side, and takes a byte of each for two columns.
#include "lowbit.cuh"
#include "tc.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kChannels = 128, kDepth = 128;     // of a tile; columns of W in a stage
constexpr int kStages = 4;                       // of x in shared memory and of W in tensor memory
constexpr int kAhead = 3;                        // of a warp's nibbles
constexpr int kUnpackers = 16, kThreads = 64 + 32 * kUnpackers;   // half of them take the even stages, half the odd ones
constexpr int kMaxRows = 128;                    // of x in a tile
constexpr int kBox = kMaxRows * 128;             // 64 columns of x
constexpr int kXStage = 2 * kBox;
constexpr int kWStage = 2 * 512 + 256;           // of a warp: two tiles, scales and zeros
constexpr int kXBytes = kStages * kXStage, kWBytes = kUnpackers * kAhead * kWStage;
constexpr int kSmem = 1024 + kXBytes + kWBytes + 128;
constexpr int kDepthCols = kDepth / 2;           // of tensor memory
constexpr int kTmem = 512, kTmemW = 128;         // the sums lie in front
constexpr int kMaxSplits = 8;
constexpr unsigned kWaitCode = 0x64000000u;
static_assert(kTmemW + kStages * kDepthCols <= kTmem && kSmem <= 232448, "room");

struct W4Gemm {
  __nv_bfloat16* y;
  const uint4* q;
  const uint32_t *scale, *zero;
  const __nv_bfloat16* bias;
  unsigned* err;
  int m, n, k, blocks, groups, group_shift;
  int rows, row_tiles, splits;   // rows of x in a tile, tiles of rows, CTAs to a tile
  bool wide;                     // y takes 8-byte stores
};

__device__ __forceinline__ void tmem_st_rows16(uint32_t taddr, const uint32_t (&r)[16]) {   // 16 rows, lane 4r + c: rows r, r + 8 of column c of every four
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint32_t sub_mul2(uint32_t v, uint32_t off, uint32_t scale) {   // (v − off)·scale of two bf16; the difference is exact
  const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off)),
                                   *reinterpret_cast<const __nv_bfloat162*>(&scale));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t fma_pack2(uint32_t v, float off, float scale) {   // scale·(v − 128) + off, one rounding to fp32 and one to bf16
  return pack2(fmaf(scale, bf16_lo(v) - 128.f, off), fmaf(scale, bf16_hi(v) - 128.f, off));
}

// Where 16 bytes of lane 4r + c of a tile lie in shared memory: eight lanes in a row store them side by side, and so do the eight r of a c read them.
__device__ __forceinline__ int chunk_at(int r, int c) { return (c * 8 + (r + 2 * c) % 8) * 16; }
// One tile of 16 rows × 64 columns at `tile`: out[2i], out[2i + 1] are rows r and r + 8 of columns 8i + 2c, + 1.  128 + zero is a bf16 number where the zero is whole
// (WHOLE); else the difference would be rounded, too, and is taken in fp32.
template <bool WHOLE, int PARTS>
__device__ __forceinline__ void unpack_tile(const uint8_t* tile, const uint32_t (&scale)[PARTS], const uint32_t (&zero)[PARTS], int r, int c, uint32_t (&out)[16]) {
  const uint32_t pick = c & 1 ? 0x7351 : 0x6240;   // bytes p, 2 + p of both words in turn
  const uint8_t* const mine = tile + (c & 2) * 2;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    uint32_t v[4];   // of the first 32 columns rows r, r + 8; of the second
    const uint8_t* const from = mine + chunk_at(r, s);
    nibbles_128(__byte_perm(*reinterpret_cast<const uint32_t*>(from), *reinterpret_cast<const uint32_t*>(from + 8), pick), v);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t sc = scale[PARTS == 2 ? h : 0], z = zero[PARTS == 2 ? h : 0];
      if constexpr (WHOLE) {   // z: 128 + zero
        out[8 * h + 2 * s] = sub_mul2(v[2 * h], __byte_perm(z, z, 0x1010), __byte_perm(sc, sc, 0x1010));
        out[8 * h + 2 * s + 1] = sub_mul2(v[2 * h + 1], __byte_perm(z, z, 0x3232), __byte_perm(sc, sc, 0x3232));
      } else {
        const float s0 = bf16_lo(sc), s1 = bf16_hi(sc);
        out[8 * h + 2 * s] = fma_pack2(v[2 * h], -s0 * bf16_lo(z), s0);
        out[8 * h + 2 * s + 1] = fma_pack2(v[2 * h + 1], -s1 * bf16_hi(z), s1);
      }
    }
  }
}

__device__ __forceinline__ bool is_whole(float zero, float sum) { return zero >= 0.f && zero < 128.f && sum - 128.f == zero; }   // (nibble − zero is exact, too)

// PARTS: groups in 64 columns (two of 32, else one).  A cluster of `splits` CTAs shares a tile's stages; their sums meet in shared memory, in order.
template <int PARTS, bool ZERO>
__global__ void __launch_bounds__(kThreads, 1) w4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const W4Gemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const sx = smem;                                   // [stages][2][rows × 128 bytes]
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + kXBytes + kWBytes);   // x has come and the stage's unpackers have stored
  uint64_t* const empty = full + kStages;
  uint64_t* const done = empty + kStages;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* const gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = (int)cluster_rank(), tile = blockIdx.x / p.splits, row0 = tile % p.row_tiles * p.rows, ch0 = tile / p.row_tiles * kChannels;
  const int all = (p.k + kDepth - 1) / kDepth, from = (int)((int64_t)all * split / p.splits), to = (int)((int64_t)all * (split + 1) / p.splits);
  bool ok = true;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], kUnpackers / 2 + 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    *gave_up = 0;
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      for (int i = from; i < to; ++i) {
        const int u = i - from, s = u % kStages;
        if (u >= kStages && !(ok = mbar_wait_limited(&empty[s], (u / kStages + 1) & 1, p.err, kWaitCode | 1))) break;
        mbar_arrive_expect_tx(&full[s], 2 * p.rows * 128);
#pragma unroll
        for (int h = 0; h < 2; ++h) tma_load_2d(sx + s * kXStage + h * kBox, &tmap_x, i * kDepth + h * 64, row0, &full[s]);
      }
      if (!ok) drain_async();
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t x0 = desc_lo(smem_u32(sx)), idesc = umma_idesc(kChannels, p.rows);
      for (int i = from; i < to; ++i) {
        const int u = i - from, s = u % kStages;
        if (!(ok = mbar_wait_limited(&full[s], (u / kStages) & 1, p.err, kWaitCode | 2))) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kDepth / 16; ++kk)
          umma_ts(tmem, tmem + kTmemW + s * kDepthCols + kk * 8, x0 + ((s * kXStage + kk / 4 * kBox + kk % 4 * 32) >> 4), idesc, u > 0 || kk > 0 ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      if (ok) umma_commit(done);
      else drain_async();
    }
  } else {
    // 32 rows in quarter warp % 4 of the tensor memory's, of every second 64 columns of every second stage
    const int unpacker = warp - 2, quad = warp & 3, half = unpacker >> 2 & 1, set = unpacker >> 3, c = lane % 4, r = lane / 4;
    uint8_t* const own = smem + kXBytes + unpacker * kAhead * kWStage;
    const int last_tile = (p.n + 15) / 16 - 1, tile0 = ch0 / 16 + quad * 2;
    const int64_t at[2] = {min(tile0, last_tile), min(tile0 + 1, last_tile)};
    const uint4* const q0 = p.q + at[0] * p.blocks * 32 + lane;
    const uint4* const q1 = p.q + at[1] * p.blocks * 32 + lane;
    constexpr int kWords = 2 * PARTS * (ZERO ? 2 : 1) * 8, kEach = (kWords + 31) / 32;   // [scale, zero][row tile][part][r]
    const uint32_t* small[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int j = (lane + 32 * e) / 8;
      small[e] = (j >= 2 * PARTS ? p.zero : p.scale) + at[j / PARTS % 2] * p.groups * 8 + lane % 8;
    }
    auto fetch = [&](int i, uint8_t* dst) {
      if (i < to) {
        const int block = min(2 * i + half, p.blocks - 1);    // (behind the last one x is zero)
        cp_async16(dst + chunk_at(r, c), q0 + block * 32);
        cp_async16(dst + 512 + chunk_at(r, c), q1 + block * 32);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int g = min((block * 64 + (lane + 32 * e) / 8 % PARTS * 32) >> p.group_shift, p.groups - 1);
          if (kWords % 32 == 0 || lane + 32 * e < kWords) cp_async4(dst + 1024 + (lane + 32 * e) * 4, small[e] + g * 8);
        }
      }
      cp_async_commit();
    };
    const int first = from + set;
#pragma unroll
    for (int a = 0; a < kAhead - 1; ++a) fetch(first + 2 * a, own + a * kWStage);
    const uint32_t to_tmem = tmem + ((uint32_t)(quad * 32) << 16) + kTmemW + half * 32;
    uint8_t *stage = own, *into = own + (kAhead - 1) * kWStage;
    int s = set, lap = 0;
    for (int i = first; i < to; i += 2) {
      fetch(i + 2 * (kAhead - 1), into);
      cp_async_wait<kAhead - 1>();
      __syncwarp();
      if (lap > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait_limited(&empty[s], (lap + 1) & 1, p.err, kWaitCode | 3)))) break;
      tc_fence_after();
      const uint32_t* const nums = reinterpret_cast<const uint32_t*>(stage + 1024) + r;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t v[16], scale[PARTS], zero[PARTS], whole[PARTS];
        bool all_whole = true;
#pragma unroll
        for (int h = 0; h < PARTS; ++h) {
          scale[h] = nums[(t * PARTS + h) * 8];
          zero[h] = ZERO ? nums[((2 + t) * PARTS + h) * 8] : 0;
          whole[h] = ZERO ? pack2(128.f + bf16_lo(zero[h]), 128.f + bf16_hi(zero[h])) : 0x43084308u;
          if (ZERO) all_whole = all_whole && is_whole(bf16_lo(zero[h]), bf16_lo(whole[h])) && is_whole(bf16_hi(zero[h]), bf16_hi(whole[h]));
        }
        if (!ZERO || __all_sync(0xffffffffu, all_whole)) unpack_tile<true, PARTS>(stage + t * 512, scale, whole, r, c, v);
        else unpack_tile<false, PARTS>(stage + t * 512, scale, zero, r, c, v);
        tmem_st_rows16(to_tmem + ((uint32_t)(t * 16) << 16) + s * kDepthCols, v);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      into = stage;
      stage = stage == own + (kAhead - 1) * kWStage ? own : stage + kWStage;
      if ((s += 2) >= kStages) {
        s -= kStages;
        ++lap;
      }
    }
    cp_async_wait<0>();
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_limited(done, 0, p.err, kWaitCode | 4));
    if (ok) {   // the sums, [row of x][channel] fp32, where x was
      tc_fence_after();
      float* const part = reinterpret_cast<float*>(sx) + quad * 32 + lane;
#pragma unroll 1
      for (int j0 = unpacker / 4 * 32; j0 < p.rows; j0 += kUnpackers / 4 * 32) {
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + j0, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j0 + j < p.rows) part[(j0 + j) * kChannels] = __uint_as_float(v[j]);
      }
    }
  }
  if (!ok) *gave_up = 1;
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (p.splits > 1) cluster_sync_all();
  // a warp takes a row of x, a lane four channels
  const bool lost = __any_sync(0xffffffffu, lane < p.splits && ld_cluster_i32(mapa_u32(smem_u32(gave_up), min(lane, p.splits - 1))) != 0);
  const int rows = lost ? 0 : min(p.rows, p.m - row0), ch = ch0 + 4 * lane;
  float bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) bias[j] = p.bias != nullptr && ch + j < p.n ? bf16_to_f(p.bias[ch + j]) : 0.f;
  for (int row = split + p.splits * warp; row < rows; row += p.splits * (kThreads / 32)) {
    const uint32_t at = smem_u32(sx) + (row * kChannels + 4 * lane) * 4;
    float4 of[kMaxSplits];
#pragma unroll
    for (int e = 0; e < kMaxSplits; ++e) of[e] = e < p.splits ? ld_cluster_f4(mapa_u32(at, e)) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v = of[0];
#pragma unroll
    for (int e = 1; e < kMaxSplits; ++e) v = make_float4(v.x + of[e].x, v.y + of[e].y, v.z + of[e].z, v.w + of[e].w);
    v = make_float4(v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]);
    __nv_bfloat16* const out = p.y + (int64_t)(row0 + row) * p.n + ch;
    if (p.wide) {
      if (ch < p.n) *reinterpret_cast<uint2*>(out) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    } else {
      if (ch < p.n) out[0] = f_to_bf16(v.x);
      if (ch + 1 < p.n) out[1] = f_to_bf16(v.y);
      if (ch + 2 < p.n) out[2] = f_to_bf16(v.z);
      if (ch + 3 < p.n) out[3] = f_to_bf16(v.w);
    }
  }
  __syncthreads();
  if (p.splits > 1) cluster_sync_all();   // nobody reads this CTA's sums any more
  if (warp == 1) {
    tc_fence_after();
    tmem_free<1>(tmem, kTmem);
  }
}

template <int PARTS, bool ZERO>
int launch(const CUtensorMap& tx, const W4Gemm& p, int64_t ctas, cudaStream_t st) {
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(w4_gemm_kernel<PARTS, ZERO>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); }));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = op_pdl(st) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  B200_CUDA(cudaLaunchKernelEx(&cfg, w4_gemm_kernel<PARTS, ZERO>, tx, p));
  return B200_OK;
}

}  // namespace

int launch_w4_gemm(void* y, const void* x, const b200_w4_weight& w, const void* bias, int64_t m, cudaStream_t st) {
  W4Gemm p{};
  int rc = wait_word(&p.err);
  if (rc != B200_OK) return rc;
  p.y = (__nv_bfloat16*)y;
  p.q = (const uint4*)w.q;
  p.scale = (const uint32_t*)w.scale;
  p.zero = (const uint32_t*)w.zero;
  p.bias = (const __nv_bfloat16*)bias;
  p.m = (int)m;
  p.n = w.n;
  p.k = w.k;
  p.blocks = (w.k + 63) / 64;
  p.groups = (w.k + w.group - 1) / w.group;
  p.group_shift = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
  p.row_tiles = (int)((m + kMaxRows - 1) / kMaxRows);
  p.rows = (int)(((m + p.row_tiles - 1) / p.row_tiles + 15) / 16 * 16);
  p.wide = w.n % 4 == 0 && ((uintptr_t)y & 7) == 0;
  // CTAs to a tile: as many as the SMs hold at once (clusters of 8: 15, of 4: 33), and two stages for each at least
  const int64_t tiles = (int64_t)p.row_tiles * ((w.n + kChannels - 1) / kChannels);
  p.splits = tiles <= 15 ? 8 : tiles <= 33 ? 4 : tiles <= 74 ? 2 : 1;
  while (p.splits > 1 && (p.k + kDepth - 1) / kDepth < 2 * p.splits) p.splits /= 2;
  CUtensorMap tx;
  if ((rc = make_tmap_sw128(&tx, 2, x, 1, m, w.k, m * w.k, w.k, p.rows)) != B200_OK) return rc;
  const int64_t ctas = tiles * p.splits;
  if (w.group == 32) return w.zero != nullptr ? launch<2, true>(tx, p, ctas, st) : launch<2, false>(tx, p, ctas, st);
  return w.zero != nullptr ? launch<1, true>(tx, p, ctas, st) : launch<1, false>(tx, p, ctas, st);
}

}  // namespace b200
