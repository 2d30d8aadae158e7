// group_gemm.cu — products of rows with the matrix of their group, on the 5th-generation tensor cores:  y[r] = W[e]·x[r] for the rows r of group e.
//
// One kernel for bf16 and for 8 bits with scales, for one matrix (a Linear) and for many (experts, rows sorted by expert).  W is the A operand: a tile is
// 128 of its rows (channels) × up to NT rows of x, and the product's N is what the tile really holds, rounded up to 16.  So a group of three rows costs a stream of its
// matrix and little else, and a group that ends inside a tile costs no idle rows.
//
// Warp-specialised, persistent over the tiles:
//   warp 0   TMA: of every 128 bytes of k 128 rows of W and the tile's rows of x, into a ring of shared memory
//   warp 1   one thread issues four products (K = 32 bytes) per 128 bytes
//   warp 2   8 bits: the products of x's and W's scales, NT of them for each block of 128 entries
//   warp 3   rows of no group are zeroed
//   warps 4 … 11   the sums: a lane holds a channel, a warp a quarter of the channels and half of the rows
// 8 bits: W has a scale for 128 × 128 entries and x one for 128 entries of a row, so that 128 entries of k meet one factor per row of x, and the sums of 128
// entries — a slot of tensor memory each — are scaled and added in fp32 registers; two to four slots keep the tensor cores running meanwhile.
// bf16: a slot holds the sums over all of k.
#include "f8.cuh"
#include "tc.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kCh = 128, kWBytes = kCh * 128, kThreads = 384, kEpiWarps = 8;
constexpr int kMaxSplits = 8;
constexpr unsigned kWaitCode = 0x67000000u;

struct Args {
  __nv_bfloat16* y;
  const float *sx, *sw;
  const int32_t* starts;
  const __nv_bfloat16* bias;
  unsigned* err;
  int64_t rows;
  int n, k_blocks, experts, ch_tiles, splits;
  bool pairs;   // y takes stores of two channels
};

template <int NT>
struct Form {
  static constexpr int per_sm = NT <= 64 ? 2 : 1;
  static constexpr int x_bytes = NT * 128, stage = kWBytes + x_bytes;
  static constexpr int stages = NT == 16 ? 5 : NT == 32 ? 5 : NT == 64 ? 4 : NT == 128 ? 6 : 4;
  static constexpr int box = NT < 64 ? NT : 64;        // rows of x in a TMA box
  static constexpr int slots8 = NT == 256 ? 2 : 4;     // of tensor memory, 8 bits
  static constexpr int cols = NT / 2;                  // rows of x a thread sums
  static constexpr int ring = stages * stage;
  static constexpr int smem = 1024 + ring + slots8 * NT * 4 + 512 + (kMaxExperts + 1) * 4;
  static constexpr int tmem(int slots) { return slots * NT < 32 ? 32 : slots * NT; }
};
static_assert(Form<16>::smem * 2 <= 228 * 1024 - 2048 && Form<32>::smem * 2 <= 228 * 1024 - 2048 && Form<64>::smem * 2 <= 228 * 1024 - 2048, "two CTAs to an SM");
static_assert(Form<128>::smem <= 227 * 1024 && Form<256>::smem <= 227 * 1024, "room");
static_assert(Form<256>::ring >= 256 * kCh * 4 && Form<128>::ring >= 128 * kCh * 4, "a partial tile fits in the drained ring");

// D[tmem] (+)= A·B over 32 entries of 8 bits
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f8f6f4: D = F32 (bits 4-5 = 1), A = B = e4m3 (0), both K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28
__device__ __forceinline__ uint32_t idesc_of(bool eight, int n) {
  const uint32_t shape = ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kCh >> 4) << 24) | (1u << 4);
  return eight ? shape : shape | (1u << 7) | (1u << 10);
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 8) tmem_ld8(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld32(taddr, r);
}

// Which rows and channels a tile has.  Tiles run over the row tiles of a group first (its matrix's rows stay in L2), then over channels, then over groups.
struct Tile {
  int64_t row0;
  int rows, ch0, expert;
};
// rows of group e: inside the call's, whatever the starts say
__device__ __forceinline__ void group_span(const int32_t* starts, int64_t rows, int e, int64_t& from, int64_t& count) {
  from = starts == nullptr ? 0 : min(max((int64_t)starts[e], (int64_t)0), rows);
  count = starts == nullptr ? rows : max(min((int64_t)starts[e + 1], rows) - from, (int64_t)0);
}

template <bool F8, int NT>
__global__ void __launch_bounds__(kThreads, Form<NT>::per_sm) group_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                                                                               const Args p) {
  using F = Form<NT>;
  constexpr int ST = F::stages, SLOTS = F8 ? F::slots8 : 2, COLS = F::cols, TMEM = F::tmem(SLOTS);
  constexpr int PIECE = COLS < 32 ? COLS : 32;      // sums loaded at once
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const sx = smem + ST * kWBytes;
  float* const factors = reinterpret_cast<float*>(smem + F::ring);                 // [slots][NT]
  uint64_t* const full = reinterpret_cast<uint64_t*>(factors + F::slots8 * NT);    // [stages]
  uint64_t* const empty = full + ST;
  uint64_t* const sums_full = empty + ST;                                          // [slots]
  uint64_t* const sums_empty = sums_full + 4;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sums_empty + 4);
  int* const gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  int* const ends = reinterpret_cast<int*>(smem + F::ring + F::slots8 * NT * 4 + 512);   // [experts] row tiles up to and with e
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  bool ok = true;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < SLOTS; ++a) {
      mbar_init(&sums_full[a], F8 ? 2 : 1);
      mbar_init(&sums_empty[a], kEpiWarps);
    }
    fence_mbar_init();
    *gave_up = 0;
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, TMEM);
  pdl_wait();
  pdl_trigger();
  auto span = [&](int e, int64_t& from, int64_t& count) { group_span(p.starts, p.rows, e, from, count); };
  if (warp == 3) {   // every lane a run of groups
    const int each = (p.experts + 31) / 32, e0 = min(lane * each, p.experts), e1 = min(e0 + each, p.experts);
    int mine = 0;
    for (int e = e0; e < e1; ++e) {
      int64_t from, count;
      span(e, from, count);
      mine += (int)((count + NT - 1) / NT);
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto -= mine;
    for (int e = e0; e < e1; ++e) {
      int64_t from, count;
      span(e, from, count);
      upto += (int)((count + NT - 1) / NT);
      ends[e] = upto;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int split = p.splits > 1 ? (int)cluster_rank() : 0;
  const int64_t tiles = (int64_t)ends[p.experts - 1] * p.ch_tiles;
  const int64_t first = blockIdx.x / p.splits, step = p.splits > 1 ? tiles : gridDim.x;   // a cluster takes one tile
  const int kb0 = (int)((int64_t)p.k_blocks * split / p.splits), kb1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
  auto tile_at = [&](int64_t t) {
    const int64_t at = t / p.ch_tiles;   // this group's: ends[e − 1] ≤ at < ends[e]
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (ends[mid] > at) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo > 0 ? ends[lo - 1] : 0, row_tiles = ends[lo] - before;
    const int64_t local = t - (int64_t)before * p.ch_tiles;
    int64_t from, count;
    span(lo, from, count);
    const int64_t i = local % row_tiles, each = ((count + row_tiles - 1) / row_tiles + 15) / 16 * 16;   // alike, and none is empty
    return Tile{from + i * each, (int)max((int64_t)0, min(min(each, (int64_t)NT), count - i * each)), (int)(local / row_tiles) * kCh, lo};
  };

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      for (int64_t t = first; t < tiles && ok; t += step) {
        const Tile tile = tile_at(t);
        const int boxes = max(1, (tile.rows + F::box - 1) / F::box), w_row = tile.expert * p.n + tile.ch0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait_limited(&empty[s], ph, p.err, kWaitCode | 1))) break;
          mbar_arrive_expect_tx(&full[s], kWBytes + boxes * F::box * 128);
          tma_load_2d(smem + s * kWBytes, &tmap_w, kb * (F8 ? 128 : 64), w_row, &full[s]);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(sx + s * F::x_bytes + b * F::box * 128, &tmap_x, kb * (F8 ? 128 : 64), (int)tile.row0 + b * F::box, &full[s]);
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) drain_async();
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t w0 = desc_lo(smem_u32(smem)), x0 = desc_lo(smem_u32(sx));
      int s = 0, slot = 0;
      uint32_t ph = 0, slot_ph = 1;
      for (int64_t t = first; t < tiles && ok; t += step) {
        const Tile tile = tile_at(t);
        const uint32_t idesc = idesc_of(F8, max(16, (tile.rows + 15) / 16 * 16));
        for (int kb = kb0; kb < kb1; ++kb) {
          if (F8 || kb == kb0) {
            if (!(ok = mbar_wait_limited(&sums_empty[slot], slot_ph, p.err, kWaitCode | 2))) break;
          }
          if (!(ok = mbar_wait_limited(&full[s], ph, p.err, kWaitCode | 3))) break;
          tc_fence_after();
          const uint32_t w = w0 + s * (kWBytes >> 4), x = x0 + s * (F::x_bytes >> 4), d = tmem + slot * NT;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (F8) umma_f8(d, w + 2 * k, x + 2 * k, idesc, k > 0 ? 1u : 0u);
            else umma_lo<1>(d, w + 2 * k, x + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
          }
          umma_commit(&empty[s]);
          if (F8 || kb == kb1 - 1) {
            umma_commit(&sums_full[slot]);
            if (++slot == SLOTS) {
              slot = 0;
              slot_ph ^= 1;
            }
          }
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) drain_async();
    }
  } else if (warp == 2) {
    if constexpr (F8) {
      constexpr int PER = (NT + 31) / 32;
      int slot = 0;
      uint32_t slot_ph = 1;
      for (int64_t t = first; t < tiles && ok; t += step) {
        const Tile tile = tile_at(t);
        const float* const sw = p.sw + ((int64_t)tile.expert * p.ch_tiles + tile.ch0 / kCh) * p.k_blocks;
        const float* const from = p.sx + tile.row0;
        for (int kb = kb0; kb < kb1; ++kb) {
          float v[PER];
          const float w = sw[kb];
#pragma unroll
          for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < tile.rows ? from[(int64_t)kb * p.rows + lane + 32 * i] * w : 0.f;
          if (!(ok = __all_sync(0xffffffffu, mbar_wait_limited(&sums_empty[slot], slot_ph, p.err, kWaitCode | 4)))) break;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (NT % 32 == 0 || lane + 32 * i < NT) factors[slot * NT + lane + 32 * i] = v[i];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sums_full[slot]);
          if (++slot == SLOTS) {
            slot = 0;
            slot_ph ^= 1;
          }
        }
      }
    }
  } else if (warp == 3) {
    if (p.starts != nullptr) {   // rows in front of the first group and behind the last
      const int64_t from = min(max((int64_t)p.starts[0], (int64_t)0), p.rows), to = min(max((int64_t)p.starts[p.experts], from), p.rows);
      for (int64_t r = blockIdx.x; r < p.rows - (to - from); r += gridDim.x) {
        __nv_bfloat16* const out = p.y + (r < from ? r : r - from + to) * p.n;
        for (int i = lane; i < p.n; i += 32) out[i] = f_to_bf16(0.f);
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 4) >> 2, ch_lane = quad * 32 + lane;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + half * COLS;
    int slot = 0;
    uint32_t slot_ph = 0;
    for (int64_t t = first; t < tiles; t += step) {
      const Tile tile = tile_at(t);
      const int mine = tile.rows - half * COLS;   // rows of this half
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
      for (int kb = F8 ? kb0 : kb1 - 1; kb < kb1; ++kb) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_limited(&sums_full[slot], slot_ph, p.err, kWaitCode | 5)))) break;
        tc_fence_after();
        const float* const factor = factors + slot * NT + half * COLS;
#pragma unroll
        for (int c = 0; c < COLS; c += PIECE) {
          if (c < mine) {
            uint32_t d[PIECE];
            tmem_ld<PIECE>(from + slot * NT + c, d);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < PIECE; j += 4) {
              if constexpr (F8) {
                const float4 f = *reinterpret_cast<const float4*>(factor + c + j);
                acc[c + j] = fmaf(__uint_as_float(d[j]), f.x, acc[c + j]);
                acc[c + j + 1] = fmaf(__uint_as_float(d[j + 1]), f.y, acc[c + j + 1]);
                acc[c + j + 2] = fmaf(__uint_as_float(d[j + 2]), f.z, acc[c + j + 2]);
                acc[c + j + 3] = fmaf(__uint_as_float(d[j + 3]), f.w, acc[c + j + 3]);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[c + j + e] = __uint_as_float(d[j + e]);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sums_empty[slot]);
        if (++slot == SLOTS) {
          slot = 0;
          slot_ph ^= 1;
        }
      }
      if (!ok) break;
      if (p.splits > 1) {   // [row][channel] where the operands were: every product has read them
        float* const part = reinterpret_cast<float*>(smem) + (int64_t)half * COLS * kCh + ch_lane;
#pragma unroll
        for (int j = 0; j < COLS; ++j)
          if (j < mine) part[j * kCh] = acc[j];
      } else {
        const int ch = tile.ch0 + ch_lane;
        const float bias = p.bias != nullptr && ch < p.n ? bf16_to_f(p.bias[ch]) : 0.f;
        __nv_bfloat16* const out = p.y + (tile.row0 + half * COLS) * p.n + ch;
        if (p.pairs) {   // a lane and its neighbour swap every second row: an even one stores both channels of row j, an odd one of row j + 1
          const bool odd = lane & 1;
          __nv_bfloat16* const to = out + (odd ? p.n - 1 : 0);
#pragma unroll
          for (int j = 0; j < COLS; j += 2) {
            if (j < mine) {
              const float a = acc[j] + bias, b = acc[j + 1] + bias;
              const float other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
              if (j + odd < mine && ch < p.n) *reinterpret_cast<uint32_t*>(to + (int64_t)j * p.n) = odd ? pack2(other, b) : pack2(a, other);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < COLS; ++j)
            if (j < mine && ch < p.n) out[(int64_t)j * p.n] = f_to_bf16(acc[j] + bias);
        }
      }
    }
  }
  if (!ok) *gave_up = 1;
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (p.splits > 1) {
    cluster_sync_all();
    // a warp takes a row of x, a lane four channels; the CTAs' sums in order
    const bool lost = __any_sync(0xffffffffu, lane < p.splits && ld_cluster_i32(mapa_u32(smem_u32(gave_up), min(lane, p.splits - 1))) != 0);
    if (first < tiles && !lost) {
      const Tile tile = tile_at(first);
      const int ch = tile.ch0 + 4 * lane;
      float bias[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bias[j] = p.bias != nullptr && ch + j < p.n ? bf16_to_f(p.bias[ch + j]) : 0.f;
      for (int row = split + p.splits * warp; row < tile.rows; row += p.splits * (kThreads / 32)) {
        const uint32_t at = smem_u32(smem) + (row * kCh + 4 * lane) * 4;
        float4 of[kMaxSplits];
#pragma unroll
        for (int e = 0; e < kMaxSplits; ++e) of[e] = e < p.splits ? ld_cluster_f4(mapa_u32(at, e)) : make_float4(0.f, 0.f, 0.f, 0.f);
        float4 v = of[0];
#pragma unroll
        for (int e = 1; e < kMaxSplits; ++e) v = make_float4(v.x + of[e].x, v.y + of[e].y, v.z + of[e].z, v.w + of[e].w);
        __nv_bfloat16* const out = p.y + (tile.row0 + row) * p.n + ch;
        const float r[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
        if (p.pairs) {
          if (ch < p.n) *reinterpret_cast<uint32_t*>(out) = pack2(r[0], r[1]);
          if (ch + 2 < p.n) *reinterpret_cast<uint32_t*>(out + 2) = pack2(r[2], r[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (ch + j < p.n) out[j] = f_to_bf16(r[j]);
        }
      }
    }
    __syncthreads();
    cluster_sync_all();   // nobody reads this CTA's sums any more
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_free<1>(tmem, TMEM);
  }
}

template <bool F8, int NT>
int launch(const GroupProduct& g, Args& p, cudaStream_t st) {
  using F = Form<NT>;
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(group_gemm_kernel<F8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::smem); }));
  CUtensorMap tw, tx;
  int rc;
  if constexpr (F8) {
    if ((rc = make_tmap_sw128_u8(&tw, g.w, g.experts * g.n, g.k, f8_ld(g.k), kCh)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128_u8(&tx, g.x, g.rows, g.k, f8_ld(g.k), F::box)) != B200_OK) return rc;
  } else {
    if ((rc = make_tmap_sw128(&tw, 2, g.w, 1, g.experts * g.n, g.k, 0, g.k, kCh)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128(&tx, 2, g.x, 1, g.rows, g.k, 0, g.k, F::box)) != B200_OK) return rc;
  }
  // tiles that there can be: every group's last one may be short
  const int64_t row_tiles = g.rows / NT + std::min<int64_t>(g.experts, g.rows), most = std::max<int64_t>(1, g.starts ? row_tiles : (g.rows + NT - 1) / NT) * p.ch_tiles;
  const int64_t room = 148 * F::per_sm;
  p.splits = 1;
  while (p.splits < kMaxSplits && most * p.splits * 2 <= room && p.k_blocks >= 4 * p.splits) p.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.splits > 1 ? most * p.splits : std::min(most, room)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = F::smem;
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
  B200_CUDA(cudaLaunchKernelEx(&cfg, group_gemm_kernel<F8, NT>, tw, tx, (const Args)p));
  return B200_OK;
}

template <bool F8>
int launch_for(const GroupProduct& g, Args& p, cudaStream_t st) {
  // rows of a tile: a group's, or twice its share of them (groups are unlike)
  const int64_t want = g.starts == nullptr ? g.rows : 2 * g.rows / std::min<int64_t>(g.experts, g.rows);
  if (want <= 16) return launch<F8, 16>(g, p, st);
  if (want <= 32) return launch<F8, 32>(g, p, st);
  if (want <= 64) return launch<F8, 64>(g, p, st);
  if (want <= 128) return launch<F8, 128>(g, p, st);
  return launch<F8, 256>(g, p, st);
}

}  // namespace

int launch_group_product(const GroupProduct& g, cudaStream_t st) {
  Args p{};
  const int rc = wait_word(&p.err);
  if (rc != B200_OK) return rc;
  p.y = (__nv_bfloat16*)g.y;
  p.sx = g.x_scale;
  p.sw = g.w_scale;
  p.starts = g.starts;
  p.bias = (const __nv_bfloat16*)g.bias;
  p.rows = g.rows;
  p.n = (int)g.n;
  p.experts = (int)g.experts;
  p.ch_tiles = (int)((g.n + kCh - 1) / kCh);
  p.k_blocks = (int)(g.x_scale != nullptr ? f8_blocks(g.k) : (g.k + 63) / 64);
  p.pairs = g.n % 2 == 0 && ((uintptr_t)g.y & 3) == 0;
  return g.x_scale != nullptr ? launch_for<true>(g, p, st) : launch_for<false>(g, p, st);
}

}  // namespace b200

extern "C" {

static int check_product(const char* what, const void* y, const void* x, const void* w, int64_t rows, int64_t experts, int64_t n, int64_t k) {
  using namespace b200;
  B200_CHECK_ARG(y && x && w && rows >= 1 && rows < 1 << 24, "%s: %lld rows out of range, or a null pointer", what, (long long)rows);
  B200_CHECK_ARG(experts >= 1 && experts <= kMaxExperts && n >= 1 && n <= 1 << 20 && k >= 1 && k <= 1 << 24 && experts * n < 1ll << 31,
                 "%s: %lld matrices [%lld, %lld] out of range", what, (long long)experts, (long long)n, (long long)k);
  B200_CHECK_ARG(aligned16(x, w), "%s: x and the weight must be 16-byte aligned", what);
  return B200_OK;
}

int b200_f8_linear_bf16(void* y, const void* q, const float* scale, const b200_f8_weight* w, const void* bias, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(w && scale && w->scale && w->experts == 1, "f8_linear: null pointer, or a weight of experts");
  if ((rc = check_product("f8_linear", y, q, w->q, rows, 1, w->n, w->k)) != B200_OK) return rc;
  return launch_group_product({y, q, scale, w->q, w->scale, nullptr, bias, rows, 1, w->n, w->k}, (cudaStream_t)stream);
}

int b200_f8_grouped_bf16(void* y, const void* q, const float* scale, const b200_f8_weight* w, const int32_t* starts, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(w && scale && w->scale && starts, "f8_grouped: null pointer");
  if ((rc = check_product("f8_grouped", y, q, w->q, rows, w->experts, w->n, w->k)) != B200_OK) return rc;
  return launch_group_product({y, q, scale, w->q, w->scale, starts, nullptr, rows, w->experts, w->n, w->k}, (cudaStream_t)stream);
}

int b200_grouped_bf16(void* y, const void* x, const void* w, const int32_t* starts, int64_t rows, int64_t experts, int64_t n, int64_t k, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_product("grouped", y, x, w, rows, experts, n, k)) != B200_OK) return rc;
  B200_CHECK_ARG(starts && k % 8 == 0, "grouped: null pointer, or k=%lld that is no multiple of 8", (long long)k);
  return launch_group_product({y, x, nullptr, w, nullptr, starts, nullptr, rows, experts, n, k}, (cudaStream_t)stream);
}

}  // extern "C"
