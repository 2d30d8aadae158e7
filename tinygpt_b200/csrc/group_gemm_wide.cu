// group_gemm_wide.cu — grouped products for groups of many rows: 256 channels and, in 8 bits, 128 rows of x to a CTA, in bf16 256 rows to a pair of them (cta_group::2).
//
// x is the A operand here: a lane of tensor memory is a row of x, so that in 8 bits a summing thread — a row, one block of 128 channels — needs one factor for 128
// sums.  With W as A (group_gemm.cu) factors differ from sum to sum: adding 128 entries of k for 128 × 256 sums took 620 to 660 cycles alone for 313 here, and
// 4 096 × 28 672 × 4 096 took 754 µs for 465 (2.07 PFLOP/s; 530 in a run of them, under the power cap).  The roles of the warps are those of group_gemm.cu; two slots of 256
// columns of tensor memory.
// 8 bits: a block of k takes some 950 cycles where its products need 512.  What is known of them: a slot goes around — products, 646 cycles until they are seen; factors, loads
// and sums, 450; back to the issuing warp — and there is room for two, so a block every 550 to 575; reading sums holds the products up (a block's loads by 124 cycles); x and W of
// 48 KB a block are written to and read from shared memory in 768.  None of these is 950: the last 180 cycles are not accounted for.  Tried and
// as slow or slower: pairs with 256 rows (32 KB a block; longer ways from CTA to CTA), four slots of 128 columns (the issue of four products alone takes 249 cycles), halves of a slot by themselves, sums in pairs or one by one, an earlier look at the next slot.
// A pair in 8 bits ends groups in tiles of 256 rows: 2 048 rows with four of 32 experts each 146 µs for 125, and 4 096 × 4 096 × 4 096 82 for 75.
// bf16: tensor memory sums over all of k; 4 096 × 4 096 × 4 096 93.5 µs (1.47 PFLOP/s).  A CTA by itself took 127 where a pair took 97.
// A summing warp stores what it summed itself, 32 channels at a time through two kilobytes: with whole tiles handed to a storing warp the last one of a CTA came 5 µs
// behind its sums, and their room is a stage of operands now.  With the tiles found by warp 3, ahead, that took 8 192 rows over 32 experts, as many for each, 2 048 × 2 048, from 52.2 to
// 48.1 µs in 8 bits and 72 to 65.6 in bf16.
#include "group_gemm.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kRows = 128;                        // of a CTA
constexpr int kXBytes = kRows * 128;              // of a stage
constexpr int kThreads = 384, kEpiWarps = 8;
constexpr unsigned kWaitCode = 0x68000000u;
constexpr int CH = 256, COLS = CH / 2, BLOCKS = CH / 128;   // channels of a tile, of a summing warp; blocks that share a scale of W
constexpr int SLOTS = 512 / CH;
constexpr int kPiece = 32 * 64;                   // of a summing warp: 32 rows of 32 finished channels
template <bool F8>
struct Wide {
  static constexpr int group = F8 ? 1 : 2;        // CTAs to a tile
  static constexpr int w_rows = CH / group, w_bytes = w_rows * 128, stage = kXBytes + w_bytes;
  static constexpr int stages = F8 ? 4 : 6;
  static constexpr int lag = 4, ahead = F8 ? 2 * SLOTS + 1 + lag : 0;   // blocks of factors that are asked for ahead, and kept: see group_gemm.cu
  static constexpr int ring = stages * stage;
  static constexpr int tables = 1024 + ring + kEpiWarps * kPiece + ahead * BLOCKS * kRows * 4 + 512;
  static constexpr int smem(int experts) { return tables + Groups::bytes(experts); }
};
// A thread that sums 8-bit products holds 128 sums: the four warps that hold none give registers up.
constexpr int kRegsFew = 72, kRegsMany = 216, kRegsLaunch = 168;
static_assert(128 * kRegsFew + 256 * kRegsMany <= kThreads * kRegsLaunch, "no warp waits for registers that the launch does not have");
static_assert(Wide<true>::smem(kWideExperts8) <= 227 * 1024 && Wide<false>::smem(kMaxExperts) <= 227 * 1024, "room");

#define B200_R8(b) "+r"(r[b]), "+r"(r[b + 1]), "+r"(r[b + 2]), "+r"(r[b + 3]), "+r"(r[b + 4]), "+r"(r[b + 5]), "+r"(r[b + 6]), "+r"(r[b + 7])
// the wait for what tmem_ld32 has loaded holds it: nothing that uses it moves in front of the wait
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : B200_R8(0), B200_R8(8));
  asm volatile("" : B200_R8(16), B200_R8(24));
}

template <bool F8>
__global__ void __launch_bounds__(kThreads, 1)
group_wide_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const GemmArgs p) {
  using F = Wide<F8>;
  constexpr int GROUP = F::group, ST = F::stages, AHEAD = F::ahead, F_SLOT = BLOCKS * kRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const sx = smem;                                                        // [stages][128 rows × 128 bytes]
  uint8_t* const sw = smem + ST * kXBytes;                                         // this CTA's rows of W alike
  uint8_t* const pieces = smem + F::ring;                                          // [summing warps][32][32]: bf16
  float* const factors = reinterpret_cast<float*>(pieces + kEpiWarps * kPiece);    // [AHEAD][blocks][128]: of a block of channels, of a row
  uint64_t* const full = reinterpret_cast<uint64_t*>(factors + AHEAD * F_SLOT);    // [stages], CTA 0's count the pair's bytes
  uint64_t* const empty = full + ST;
  uint64_t* const sums_full = empty + ST;                                          // [slots]
  uint64_t* const sums_empty = sums_full + SLOTS;                                  // CTA 0's
  TileRing ring(sums_empty + SLOTS);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sums_empty + SLOTS) + TileRing::bytes / 4;
  float* const w_scale = reinterpret_cast<float*>(tmem_slot + 1);                  // [AHEAD][blocks]
  Groups groups(reinterpret_cast<int*>(smem + F::tables - 1024), p.experts);
  const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
  const int rank = GROUP == 2 ? (int)cluster_rank() : 0;
  bool ok = true;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < SLOTS; ++a) {
      mbar_init(&sums_full[a], F8 ? 2 : 1);   // products done, factors there
      mbar_init(&sums_empty[a], GROUP * kEpiWarps);
    }
    ring.init(kEpiWarps + (F8 ? 2 : 1));
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc<GROUP>(tmem_slot, 512);
  pdl_wait();
  pdl_trigger();
  if (warp == 3) groups.make<GROUP * kRows>(p.starts, p.rows, lane);
  tc_fence_before();
  __syncthreads();
  if constexpr (GROUP == 2) cluster_sync_all();   // the pair's barriers exist
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const int tiles = groups.ends[p.experts - 1] * p.ch_tiles, first = blockIdx.x / GROUP, step = gridDim.x / GROUP;
  const int k_blocks = p.k_blocks;
  Tile tile{};   // row0 and rows of this CTA: none where the tile ends in the pair's first half
  auto next_tile = [&]() { return ok = ring.take(tile, lane, p.err, kWaitCode | 6); };

  if (warp < 4) {
    if constexpr (F8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0) {
      int s = 0;
      uint32_t ph = 1;
      for (int t = first; t < tiles && ok; t += step) {
        if (!next_tile()) break;
        if (lane == 0) {
          const int x_row = (int)tile.row0, w_row = tile.expert * p.n + tile.ch0 + rank * F::w_rows;   // (what lies past the operands is zero)
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (!(ok = wait_asleep(&empty[s], ph, p.err, kWaitCode | 1))) break;
            const int k0 = kb * (F8 ? 128 : 64);
            if constexpr (GROUP == 2) {
              const uint32_t bar = mapa_u32(smem_u32(&full[s]), 0);
              if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * F::stage);
              tma_load_2d_pair(sx + s * kXBytes, &tmap_x, k0, x_row, bar);
              tma_load_2d_pair(sw + s * F::w_bytes, &tmap_w, k0, w_row, bar);
            } else {
              mbar_arrive_expect_tx(&full[s], F::stage);
              tma_load_2d(sx + s * kXBytes, &tmap_x, k0, x_row, &full[s]);
              tma_load_2d(sw + s * F::w_bytes, &tmap_w, k0, w_row, &full[s]);
            }
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        __syncwarp();
      }
      if (lane == 0 && !ok) drain_async();
    } else if (warp == 1) {
      if (GROUP == 1 || rank == 0) {
        const uint32_t x0 = desc_lo(smem_u32(sx)), w0 = desc_lo(smem_u32(sw)), idesc = idesc_of(F8, GROUP * kRows, CH), lead = elect_one();
        int s = 0, slot = 0;
        uint32_t ph = 0, slot_ph = 1;
        bool ready = false;   // the next stage, looked at behind the products of this one
        for (int t = first; t < tiles && ok; t += step) {
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (!ready && !(ok = warp_wait(&full[s], ph, p.err, kWaitCode | 2))) break;
            if ((F8 || kb == 0) && !(ok = warp_wait(&sums_empty[slot], slot_ph, p.err, kWaitCode | 3))) break;
            tc_fence_after();
            const uint32_t x = x0 + s * (kXBytes >> 4), w = w0 + s * (F::w_bytes >> 4), d = tmem + slot * CH;
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_by<F8, GROUP>(lead, d, x + 2 * k, w + 2 * k, idesc, k > 0 || (!F8 && kb > 0) ? 1u : 0u);
            commit_by<GROUP>(lead, &empty[s]);
            if (F8 || kb == k_blocks - 1) {
              commit_by<GROUP>(lead, &sums_full[slot]);
              if (++slot == SLOTS) {
                slot = 0;
                slot_ph ^= 1;
              }
            }
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
            ready = __all_sync(0xffffffffu, mbar_test(&full[s], ph));
          }
        }
        if (!ok) drain_async();
      }
    } else if (warp == 2) {
      if constexpr (F8) {   // as in group_gemm.cu, which says why the ring is never written where it is read
        const int64_t units = first < tiles ? (int64_t)((tiles - first + step - 1) / step) * k_blocks : 0;
        int kb = 0, into = 0, from_slot = 0, slot = 0;
        uint32_t ph = 1;
        auto ask = [&]() {
          if (kb == 0 && !next_tile()) return false;
          const float* const from = p.sx + (int64_t)kb * p.rows + tile.row0 + lane;
          float* const to = factors + into * F_SLOT + lane;
#pragma unroll
          for (int i = 0; i < kRows / 32; ++i)
            if (lane + 32 * i < tile.rows) cp_async4(to + 32 * i, from + 32 * i);
          if (lane < BLOCKS)
            cp_async4(&w_scale[BLOCKS * into + lane], p.sw + ((int64_t)tile.expert * p.ch_blocks + min(tile.ch0 / 128 + lane, p.ch_blocks - 1)) * k_blocks + kb);
          if (++kb == k_blocks) kb = 0;
          if (++into == AHEAD) into = 0;
          return true;
        };
        for (int64_t u = -F::lag; u < units; ++u) {
          if (u >= 0 && !(ok = warp_wait(&sums_full[slot], ph, p.err, kWaitCode | 4))) break;
          if (u + F::lag < units && !ask()) break;
          cp_async_commit();
          if (u >= 0) {
            cp_async_wait<F::lag>();
            __syncwarp();
            const float w_lo = w_scale[BLOCKS * from_slot], w_hi = w_scale[BLOCKS * from_slot + 1];
            float* const at = factors + from_slot * F_SLOT + lane;
#pragma unroll
            for (int i = 0; i < kRows / 32; ++i) {   // (places behind the tile's rows hold anything: nobody stores what they scale)
              const float v = at[32 * i];
              at[32 * i] = v * w_lo;
              at[kRows + 32 * i] = v * w_hi;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sums_full[slot]);
            if (++from_slot == AHEAD) from_slot = 0;
            if (++slot == SLOTS) {
              slot = 0;
              ph ^= 1;
            }
          }
        }
        cp_async_wait<0>();
      }
    } else {
      int e = 0;   // the group of the last tile
      for (int t = first; t < tiles && ok; t += step) {
        int local, row_tiles;
        groups.walk(t, p.ch_tiles, lane, e, local, row_tiles);   // a group's row tiles first: its rows of W stay in L2
        const int channels = row_tiles == 1 ? local : local / row_tiles, row = (local - channels * row_tiles) * (GROUP * kRows) + rank * kRows;
        ok = ring.give(groups.froms[e] + row, max(0, min(kRows, groups.counts[e] - row)), channels * CH, e, lane, p.err, kWaitCode | 7);
      }
      zero_other_rows(p, lane);
    }
  } else {
    if constexpr (F8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
    const int quad = warp & 3, half = (warp - 4) >> 2, row = quad * 32 + lane;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + half * COLS, free_bar = GROUP == 2 ? mapa_u32(smem_u32(sums_empty), 0) : 0;
    uint8_t* const piece = pieces + (warp - 4) * kPiece;
    const float* const my_factors = factors + half * kRows + row;
    int slot = 0, fslot = 0;
    uint32_t slot_ph = 0;
    for (int t = first; t < tiles; t += step) {
      if (!next_tile()) break;
      const bool mine = quad * 32 < tile.rows;   // some row of this warp is one
      auto release = [&]() {   // the slot may be filled again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (GROUP == 1 || rank == 0) mbar_arrive(&sums_empty[slot]);
          else arrive_at(free_bar + slot * 8);
        }
        if (++slot == SLOTS) {
          slot = 0;
          slot_ph ^= 1;
        }
      };
      // channels 32i … 32i + 31 of this half, as pairs, → y
      auto put = [&](int i, auto pair_at) {
        const int ch0 = tile.ch0 + half * COLS + 32 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float2 f = pair_at(4 * j + c);
            if (p.bias != nullptr) {
              const int ch = ch0 + 8 * j + 2 * c;
              f = make_float2(f.x + (ch < p.n ? bf16_to_f(p.bias[ch]) : 0.f), f.y + (ch + 1 < p.n ? bf16_to_f(p.bias[ch + 1]) : 0.f));
            }
            v[c] = pack2(f.x, f.y);
          }
          *reinterpret_cast<uint4*>(piece + piece_at(lane, j)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
        store_piece(p.y + (tile.row0 + quad * 32) * p.n + ch0, piece, min(32, tile.rows - quad * 32), p.n - ch0, p, lane);
        __syncwarp();
      };
      if constexpr (F8) {
        constexpr int PIECES = COLS / 32;
        uint64_t acc[COLS / 2];
#pragma unroll
        for (int j = 0; j < COLS / 2; ++j) acc[j] = 0;
        if (mine) {
          // One load is always on its way while another's sums are added, the next unit's first one too where its products are done by then.
          uint32_t d[2][32];
          if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
          tc_fence_after();
          tmem_ld32(from + slot * CH, d[0]);
          for (int kb = 0; kb < k_blocks; ++kb) {
            const float f = my_factors[fslot * F_SLOT];
            const uint64_t ff = pair_of(f, f);
            const uint32_t at = from + slot * CH;
            bool next = false;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              loaded(d[i % 2]);
              if (i + 1 < PIECES) {
                tmem_ld32(at + 32 * (i + 1), d[(i + 1) % 2]);
              } else {
                release();
                next = kb + 1 < k_blocks && __all_sync(0xffffffffu, mbar_test(&sums_full[slot], slot_ph));
                if (next) {
                  tc_fence_after();
                  tmem_ld32(from + slot * CH, d[0]);
                }
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[16 * i + j] = fma_pair(pair_of(d[i % 2][2 * j], d[i % 2][2 * j + 1]), ff, acc[16 * i + j]);
            }
            if (++fslot == AHEAD) fslot = 0;
            if (!next && kb + 1 < k_blocks) {
              if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
              tc_fence_after();
              tmem_ld32(from + slot * CH, d[0]);
            }
          }
        } else {
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
            release();
            if (++fslot == AHEAD) fslot = 0;
          }
        }
        if (!ok) break;
        if (mine) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i) put(i, [&](int j) { return halves(acc[16 * i + j]); });
        }
      } else {
        if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
        tc_fence_after();
        if (mine) {
#pragma unroll 1
          for (int i = 0; i < COLS / 32; ++i) {
            uint32_t d[32];
            tmem_ld32(from + slot * CH + 32 * i, d);
            loaded(d);
            if (i + 1 == COLS / 32) release();
            put(i, [&](int j) { return make_float2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])); });
          }
        } else {
          release();
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if constexpr (GROUP == 2) cluster_sync_all();   // neither CTA still reads the pair's operands, barriers or sums
  if (warp == 1) {
    tc_fence_after();
    tmem_free<GROUP>(tmem, 512);
  }
  if constexpr (GROUP == 2) cluster_sync_all();
}

template <bool F8>
int launch(const GroupProduct& g, GemmArgs& p, cudaStream_t st) {
  using F = Wide<F8>;
  static PerDevice attrs;
  B200_CUDA(attrs([] {
    cudaFuncAttributes a{};
    const cudaError_t e = cudaFuncGetAttributes(&a, group_wide_kernel<F8>);
    if (e != cudaSuccess) return e;
    if (F8 && a.numRegs != kRegsLaunch) return cudaErrorInvalidDeviceFunction;   // (the shares would not add up)
    return cudaFuncSetAttribute(group_wide_kernel<F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::smem(F8 ? kWideExperts8 : kMaxExperts));
  }));
  CUtensorMap tw, tx;
  int rc;
  if constexpr (F8) {
    if ((rc = make_tmap_sw128_u8(&tw, g.w, g.experts * g.n, g.k, f8_ld(g.k), F::w_rows)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128_u8(&tx, g.x, g.rows, g.k, f8_ld(g.k), kRows)) != B200_OK) return rc;
  } else {
    if ((rc = make_tmap_sw128(&tw, 2, g.w, 1, g.experts * g.n, g.k, 0, g.k, F::w_rows)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128(&tx, 2, g.x, 1, g.rows, g.k, 0, g.k, kRows)) != B200_OK) return rc;
  }
  p.ch_blocks = (int)((g.n + 127) / 128);
  p.ch_tiles = (int)((g.n + CH - 1) / CH);
  p.splits = 1;
  // tiles that there can be: every group's last one may be short
  constexpr int GROUP = F::group, kTileRows = GROUP * kRows;
  const int64_t row_tiles = g.starts ? g.rows / kTileRows + std::min<int64_t>(g.experts, g.rows) : (g.rows + kTileRows - 1) / kTileRows;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(GROUP * std::min<int64_t>(row_tiles * p.ch_tiles, 148 / GROUP)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = F::smem((int)g.experts);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = GROUP;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = op_pdl(st) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  B200_CUDA(cudaLaunchKernelEx(&cfg, group_wide_kernel<F8>, tw, tx, (const GemmArgs)p));
  return B200_OK;
}

}  // namespace

int launch_group_wide(const GroupProduct& g, GemmArgs& p, cudaStream_t st) { return g.x_scale == nullptr ? launch<false>(g, p, st) : launch<true>(g, p, st); }

}  // namespace b200
