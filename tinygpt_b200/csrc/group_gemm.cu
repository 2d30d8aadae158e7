// group_gemm.cu — products of rows with the matrix of their group, on the 5th-generation tensor cores:  y[r] = W[e]·x[r] for the rows r of group e.
//
// For bf16 and for 8 bits with scales, for one matrix (a Linear) and for many (experts, rows sorted by expert).  W is the A operand: a tile is 128 of its rows (channels) ×
// up to NT rows of x, and the product's N is what the tile really holds, rounded up to 16.  So a group of three rows costs a stream of its matrix and little else, and a
// group that ends inside a tile costs no idle rows.  Few rows are bound by that stream: one row × 28 672 × 4 096 in 8 bits 21.3 µs, 5.5 TB/s; launch, the first loads' way
// and the end are 5 µs of any call.
//
// Warp-specialised, persistent over the tiles:
//   warp 0   TMA: of every 128 bytes of k 128 rows of W and the tile's rows of x, into a ring of shared memory
//   warp 1   issues four products (K = 32 bytes) per 128 bytes, as a whole warp with one leading lane (umma_by)
//   warp 2   8 bits: the products of x's and W's scales, NT of them for each block of 128 entries, fetched some blocks ahead
//   warp 3   finds the CTA's tiles; rows of no group are zeroed
//   warps 4 … 11   the sums: a warp has a quarter of the channels and half of the rows, as fragments of 8 × 8 (lane 4r + c: channel r, rows 2c and 2c + 1), so
//            that a lane needs a quarter of the factors and a transposing store to shared memory makes rows of y of them, which the warp stores
// 8 bits: W has a scale for 128 × 128 entries and x one for 128 entries of a row, so that 128 entries of k meet one factor per row of x, and the sums of 128
// entries — a slot of tensor memory each — are scaled and added in fp32 registers; two to four slots keep the tensor cores running meanwhile.
// bf16: a slot holds the sums over all of k.
// Where there are few tiles, a cluster of CTAs shares a tile's k and each sums its rows of the partial tiles, sent through distributed shared memory.
// Many rows go to tiles of 256 channels with x as the A operand (group_gemm_wide.cu); choose() says when.
#include "group_gemm.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {

namespace {

constexpr int kCh = 128, kWBytes = kCh * 128, kThreads = 384, kEpiWarps = 8;
constexpr int kMaxSplits = 8;
constexpr int kPartLd = kCh + 4;            // floats from row to row of a partial tile: a fragment's lanes meet 32 banks
constexpr unsigned kWaitCode = 0x67000000u;
// Blocks of W that are asked into L2 beside the kernel in front.  Behind a norm 16 × 6 144 × 4 096 take 12.1 µs for 12.5 without, 48 × 4 096 × 4 096 13.0 for 13.4, in a run of
// its own 128 × 4 096 × 4 096 11.8 for 12.3 and 1 × 28 672 × 4 096 21.3 for 21.6 (1 × 4 096 × 14 336 15.2 for 14.9); more blocks compete with the running kernel's: with 16 and
// 32 1 × 28 672 × 4 096 takes 22.6 and 25.1.
constexpr int kWToL2 = 4;

template <int NT>
struct Form {
  static constexpr int per_sm = NT <= 64 ? 2 : 1;
  static constexpr int x_bytes = NT * 128, stage = kWBytes + x_bytes;
  static constexpr int stages = NT == 16 ? 5 : NT == 64 ? 3 : 4;
  static constexpr int box = NT < 64 ? NT : 64;  // rows of x in a TMA box
  static constexpr int slots8 = 4;                     // of tensor memory, 8 bits
  static constexpr int lag = 3;                        // blocks that factors are asked for ahead
  static constexpr int ahead = 2 * slots8 + 1 + lag;   // blocks of factors in shared memory: see where they are written
  static constexpr int f_slot = NT < 32 ? 32 : NT;
  static constexpr int cols = NT / 2;                  // rows of x of a summing warp
  static constexpr int ring = stages * stage;
  static constexpr int out_bytes = NT * kPartLd * 4;   // a finished tile in bf16, the warps' pieces one behind the other, or what the CTAs of a cluster send of theirs in fp32
  static constexpr int tables = 1024 + ring + out_bytes + ahead * f_slot * 4 + 512;
  static constexpr int smem(int experts) { return tables + Groups::bytes(experts); }
  static constexpr int tmem(int slots) { return slots * NT < 32 ? 32 : slots * NT; }
};
static_assert(Form<16>::smem(64) <= 113 * 1024 && Form<32>::smem(64) <= 114 * 1024 && Form<64>::smem(64) <= 114 * 1024, "two CTAs to an SM");
static_assert(Form<128>::smem(kMaxExperts) <= 227 * 1024, "room");
static_assert(Form<128>::ring >= 128 * kPartLd * 4 && Form<64>::ring >= 64 * kPartLd * 4 && Form<16>::ring >= 16 * kPartLd * 4, "a partial tile fits in the drained ring");

// 16 lanes of tensor memory × 8·N columns as N fragments: lane 4r + c takes {(r, 2c), (r, 2c + 1), (r + 8, 2c), (r + 8, 2c + 1)} of each.  What was loaded is held by the
// wait (tmem_ready), so that nothing that uses it moves in front of that.
__device__ __forceinline__ void tmem_frag(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_frag(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_frag(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]));
}
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]));
}
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
// four 8 × 8 matrices of 16 bits, each transposed; lane 8m + i holds the address of row i of matrix m
__device__ __forceinline__ void store_transposed(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// what a load at these coordinates would read, to L2
__device__ __forceinline__ void tma_to_l2(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// where the factor of row j of a tile lies: a lane that holds rows 8i + 2c, + 1 finds those of four i side by side
__device__ __forceinline__ int factor_at(int j) { return (j & ~31) + (j % 8 / 2) * 8 + (j % 32 / 8) * 2 + j % 2; }
template <bool F8, int NT>
__global__ void __launch_bounds__(kThreads, Form<NT>::per_sm) group_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                                                                               const GemmArgs p) {
  using F = Form<NT>;
  constexpr int ST = F::stages, SLOTS = F8 ? F::slots8 : 2, COLS = F::cols, TMEM = F::tmem(SLOTS), AHEAD = F::ahead, LAG = F::lag;
  constexpr int PIECE = COLS < 32 ? COLS : 32;      // rows of 16 channels that are loaded at once
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const sx = smem + ST * kWBytes;
  uint8_t* const done_tile = smem + F::ring;
  float* const factors = reinterpret_cast<float*>(done_tile + F::out_bytes);       // [AHEAD][NT]
  uint64_t* const full = reinterpret_cast<uint64_t*>(factors + AHEAD * F::f_slot);   // [stages]
  uint64_t* const empty = full + ST;
  uint64_t* const sums_full = empty + ST;                                          // [slots]
  uint64_t* const sums_empty = sums_full + 4;
  TileRing ring(sums_empty + 4);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sums_empty + 4) + TileRing::bytes / 4;
  int* const gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  int* const gave_up_of = gave_up + 1;                                                // [splits]
  float* const w_scale = reinterpret_cast<float*>(gave_up_of + kMaxSplits);                       // [AHEAD]
  Groups groups(reinterpret_cast<int*>(smem + F::tables - 1024), p.experts);
  const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
  const int split = p.splits > 1 ? (int)cluster_rank() : 0;
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
      mbar_init(&sums_empty[a], kEpiWarps);
    }
    ring.init(kEpiWarps + (F8 ? 3 : 2));
    fence_mbar_init();
    *gave_up = 0;
  }
  if (p.splits > 1) cluster_arrive_relaxed();
  if (warp == 1) tmem_alloc<1>(tmem_slot, TMEM);
  // Where the kernel in front only makes x: the groups and, of the first tile, as many blocks of W as there are stages come beside it.  48 × 4 096 × 14 336
  // from bf16 rows 18.8 µs for 20.3, a layer of 32 experts over 8 rows 33.1 for 35.1.
  const bool ahead = F8 && p.ahead;
  const int first = blockIdx.x / p.splits;
  const int kb0 = (int)((int64_t)p.k_blocks * split / p.splits), kb1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
  if (!ahead) {
    if (p.starts == nullptr && threadIdx.x == 0) {   // rows that are given: W may be written by the kernel in front, but L2 has what is written
      const int ch0 = first / (int)((p.rows + NT - 1) / NT) * kCh;
      for (int kb = kb0; kb < kb1 && kb - kb0 < kWToL2 && ch0 < p.n; ++kb) tma_to_l2(&tmap_w, kb * 128, ch0);
    }
    pdl_wait();
    pdl_trigger();
  }
  if (warp == 3) groups.make<NT>(p.starts, p.rows, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const int tiles = groups.ends[p.experts - 1] * p.ch_tiles;
  const int step = p.splits > 1 ? max(tiles, 1) : (int)gridDim.x;   // a cluster that splits k takes one tile
  Tile tile{};
  auto next_tile = [&]() { return ok = ring.take(tile, lane, p.err, kWaitCode | 6); };
  auto up16 = [](int v) { return (v + 15) / 16 * 16; };

  if (warp < 4) {
    if (warp == 0) {
      int s = 0;
      uint32_t ph = 1;
      for (int t = first; t < tiles && ok; t += step) {
        if (!next_tile()) break;
        if (lane == 0) {
          const int row0 = (int)tile.row0;
          const int boxes = (tile.rows + F::box - 1) / F::box, w_row = tile.expert * p.n + tile.ch0;
          auto ask_w = [&](int kb, int s) {
            mbar_arrive_expect_tx(&full[s], kWBytes + boxes * F::box * 128);
            tma_load_2d(smem + s * kWBytes, &tmap_w, kb * (F8 ? 128 : 64), w_row, &full[s]);
          };
          int asked = kb0;   // blocks of W in front of this one are on their way
          if (ahead && t == first) {
            for (; asked < kb1 && asked - kb0 < ST; ++asked) ask_w(asked, asked - kb0);
            pdl_wait();
          }
          for (int kb = kb0; kb < kb1; ++kb) {
            if (kb >= asked) {
              if (!(ok = wait_asleep(&empty[s], ph, p.err, kWaitCode | 1))) break;
              ask_w(kb, s);
            }
            uint8_t* const x_to = sx + s * F::x_bytes;
            const int k0 = kb * (F8 ? 128 : 64);
            for (int b = 0; b < boxes; ++b) tma_load_2d(x_to + b * F::box * 128, &tmap_x, k0, row0 + b * F::box, &full[s]);
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
      }
      if (lane == 0 && !ok) drain_async();
    } else if (warp == 1) {
      const uint32_t w0 = desc_lo(smem_u32(smem)), x0 = desc_lo(smem_u32(sx)), lead = elect_one();
      int s = 0, slot = 0;
      uint32_t ph = 0, slot_ph = 1;
      bool ready = false;   // the next stage and slot, looked at behind the products of this one
      for (int t = first; t < tiles && ok; t += step) {
        if (!next_tile()) break;
        const uint32_t idesc = uniform(idesc_of(F8, kCh, up16(tile.rows)));
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ready) {
            if (!(ok = warp_wait(&sums_empty[slot], slot_ph, p.err, kWaitCode | 2))) break;
            if (!(ok = warp_wait(&full[s], ph, p.err, kWaitCode | 3))) break;
          }
          tc_fence_after();
          const uint32_t w = w0 + s * (kWBytes >> 4), x = x0 + s * (F::x_bytes >> 4), d = tmem + slot * NT;
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_by<F8, 1>(lead, d, w + 2 * k, x + 2 * k, idesc, k > 0 || (!F8 && kb > kb0) ? 1u : 0u);
          commit_by<1>(lead, &empty[s]);
          if (F8 || kb == kb1 - 1) {
            commit_by<1>(lead, &sums_full[slot]);
            if (++slot == SLOTS) {
              slot = 0;
              slot_ph ^= 1;
            }
          }
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
          ready = mbar_test(&full[s], ph);
          if (F8 || kb == kb1 - 1) ready = mbar_test(&sums_empty[slot], slot_ph) && ready;
          ready = __all_sync(0xffffffffu, ready);
        }
      }
      if (!ok) drain_async();
    } else if (warp == 2) {
      if constexpr (F8) {
        // Of unit u — a block of a tile — x's scales and W's are asked for LAG units before they are multiplied.  A slot's barrier takes unit u's arrival when its
        // phase before, unit u − SLOTS, is complete.  Then the products of that unit are done, so every warp has released unit u − 2·SLOTS and needs nothing of the units in
        // front of that one any more: a ring of 2·SLOTS + 1 + LAG units is never written where it is read.
        constexpr int PER = (NT + 31) / 32;
        if (ahead) {
          pdl_wait();
          pdl_trigger();
        }
        const int64_t units = first < tiles ? (int64_t)((tiles - first + step - 1) / step) * (kb1 - kb0) : 0;
        int kb = kb0, into = 0, from_slot = 0, slot = 0;
        uint32_t ph = 1;
        auto ask = [&]() {
          if (kb == kb0 && !next_tile()) return false;
          const float* const from = p.sx + (int64_t)kb * p.rows + tile.row0 + lane;
          float* const to = factors + into * F::f_slot + factor_at(lane);
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < tile.rows) cp_async4(to + 32 * i, from + 32 * i);
          if (lane == 0) cp_async4(&w_scale[into], p.sw + ((int64_t)tile.expert * p.ch_blocks + min(tile.ch0 / kCh, p.ch_blocks - 1)) * p.k_blocks + kb);
          if (++kb == kb1) kb = kb0;
          if (++into == AHEAD) into = 0;
          return true;
        };
        for (int64_t u = -LAG; u < units; ++u) {
          if (u >= 0 && !(ok = warp_wait(&sums_full[slot], ph, p.err, kWaitCode | 4))) break;
          if (u + LAG < units && !ask()) break;
          cp_async_commit();
          if (u >= 0) {
            cp_async_wait<LAG>();
            __syncwarp();
            const float w = w_scale[from_slot];
            float* const at = factors + from_slot * F::f_slot + lane;
#pragma unroll
            for (int i = 0; i < PER; ++i) at[32 * i] *= w;   // (places behind the tile's rows hold anything: nobody stores what they scale)
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
    } else if (warp == 3) {
      int e = 0;   // the group of the last tile
      for (int t = first; t < tiles && ok; t += step) {
        int local, row_tiles;
        groups.walk(t, p.ch_tiles, lane, e, local, row_tiles);   // a group's row tiles first: its rows of W stay in L2
        const int count = groups.counts[e], channels = row_tiles == 1 ? local : local / row_tiles, i = local - channels * row_tiles;
        const int each = row_tiles == 1 ? count : ((count + row_tiles - 1) / row_tiles + 15) / 16 * 16;   // alike, and none is empty
        ok = ring.give(groups.froms[e] + i * each, min(each, count - i * each), channels * kCh, e, lane, p.err, kWaitCode | 7);
      }
      if (ahead) pdl_wait();
      zero_other_rows(p, lane);
    }
  } else {
    const int quad = warp & 3, half = (warp - 4) >> 2, r = lane / 4, c = lane % 4;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + half * COLS;
    uint8_t* const piece = done_tile + (warp - 4) * (COLS * 64);
    const uint32_t put_at = smem_u32(piece) + piece_at(lane % 8, lane / 8);   // lane 8m + i of a transposing store: row i, channels 8m … 8m + 7 of 32
    int slot = 0, fslot = 0;
    uint32_t slot_ph = 0;
    for (int t = first; t < tiles; t += step) {
      if (!next_tile()) break;
      const int mine = tile.rows - half * COLS;   // rows of this half
      const int ch0 = tile.ch0 + quad * 32;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = p.bias != nullptr && ch0 + r + 8 * e < p.n ? bias_at(p.bias + ch0 + r + 8 * e) : 0.f;
      // Rows j … j + 7 of this half, 32 channels: v[e][i] is channel r + 8e, row j + 2c + i.
      auto put8 = [&](int j, float2 (&v)[4]) {
        if (p.splits > 1) {   // [row][channel] where the operands were: every product has read them
          float* const part = reinterpret_cast<float*>(smem) + (half * COLS + j + 2 * c) * kPartLd + quad * 32 + r;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            part[8 * e] = v[e].x;
            part[8 * e + kPartLd] = v[e].y;
          }
        } else {
          store_transposed(put_at + j * 64, pack2(v[0].x + bias[0], v[0].y + bias[0]), pack2(v[1].x + bias[1], v[1].y + bias[1]),
                           pack2(v[2].x + bias[2], v[2].y + bias[2]), pack2(v[3].x + bias[3], v[3].y + bias[3]));
        }
      };
      auto store = [&]() {
        if (p.splits > 1) return;
        __syncwarp();
        store_piece(p.y + (tile.row0 + half * COLS) * p.n + ch0, piece, min(mine, COLS), p.n - ch0, p, lane);
        __syncwarp();
      };
      auto release = [&]() {   // the slot may be filled again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sums_empty[slot]);
        if (++slot == SLOTS) {
          slot = 0;
          slot_ph ^= 1;
        }
      };
      if constexpr (F8) {
        // acc[g][e]: rows 8g + 2c, + 1, channel r + 8e
        uint64_t acc[COLS / 8][4];
#pragma unroll
        for (int g = 0; g < COLS / 8; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[g][e] = 0;
        auto unit = [&](auto all_rows) {
          constexpr bool ALL = decltype(all_rows)::value;
          const float* const factor = factors + fslot * F::f_slot + (half * COLS & ~31) + c * 8 + half * COLS % 32 / 4;
          const uint32_t at = from + slot * NT;
          constexpr int PIECES = COLS / PIECE;
          const int pieces = ALL ? PIECES : (mine + PIECE - 1) / PIECE;
          uint32_t d[2][2][PIECE / 2];   // channels 0 … 15, 16 … 31
          float2 f[PIECE / 8];
          tmem_frag(at, d[0][0]);
          tmem_frag(at + (16u << 16), d[0][1]);
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            if (!ALL && i >= pieces) break;
            if constexpr (PIECE >= 16) {
#pragma unroll
              for (int g = 0; g < PIECE / 8; g += 2) {
                const float4 both = *reinterpret_cast<const float4*>(factor + i * PIECE + 2 * g);
                f[g] = make_float2(both.x, both.y);
                f[g + 1] = make_float2(both.z, both.w);
              }
            } else {
              f[0] = *reinterpret_cast<const float2*>(factor);
            }
            tmem_ready(d[i % 2][0]);
            tmem_ready(d[i % 2][1]);
            if (i + 1 < PIECES && (ALL || i + 1 < pieces)) {
              tmem_frag(at + (i + 1) * PIECE, d[(i + 1) % 2][0]);
              tmem_frag(at + (i + 1) * PIECE + (16u << 16), d[(i + 1) % 2][1]);
            } else {
              release();
            }
#pragma unroll
            for (int g = 0; g < PIECE / 8; ++g) {
              const uint64_t fg = pair_of(f[g].x, f[g].y);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[i * (PIECE / 8) + g][e] = fma_pair(pair_of(d[i % 2][e / 2][4 * g + e % 2 * 2], d[i % 2][e / 2][4 * g + e % 2 * 2 + 1]), fg, acc[i * (PIECE / 8) + g][e]);
            }
          }
        };
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
          tc_fence_after();
          if (mine >= COLS) unit(Is<true>{});
          else if (mine > 0) unit(Is<false>{});
          else release();
          if (++fslot == AHEAD) fslot = 0;
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < COLS / 8; ++g)
          if (8 * g < mine) {
            float2 v[4] = {halves(acc[g][0]), halves(acc[g][1]), halves(acc[g][2]), halves(acc[g][3])};
            put8(8 * g, v);
          }
        store();
      } else {
        if (!(ok = warp_wait(&sums_full[slot], slot_ph, p.err, kWaitCode | 5))) break;
        tc_fence_after();
#pragma unroll 1
        for (int j = 0; j < COLS && j < mine; j += PIECE) {
          uint32_t a[PIECE / 2], b[PIECE / 2];
          tmem_frag(from + slot * NT + j, a);
          tmem_frag(from + slot * NT + j + (16u << 16), b);
          tmem_ready(a);
          tmem_ready(b);
          if (j + PIECE >= COLS || j + PIECE >= mine) release();
#pragma unroll
          for (int g = 0; g < PIECE / 8; ++g)
            if (j + 8 * g < mine) {
              float2 v[4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                v[e] = make_float2(__uint_as_float(a[4 * g + 2 * e]), __uint_as_float(a[4 * g + 2 * e + 1]));
                v[2 + e] = make_float2(__uint_as_float(b[4 * g + 2 * e]), __uint_as_float(b[4 * g + 2 * e + 1]));
              }
              put8(j + 8 * g, v);
            }
        }
        if (mine <= 0) release();
        store();
      }
    }
  }
  if (!ok) *gave_up = 1;
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (p.splits > 1) {
    // Every row has an owner among the CTAs, which get their rows of everybody's partial tile (a warp a row, a lane four channels) and sum them in order.
    // Reading them from the others instead takes a round trip and a second meeting: 48 × 4 096 × 14 336 from bf16 rows 0.5 µs more.
    const int owned = NT / p.splits;
    const int4 only = first < tiles ? ring.tiles[0] : make_int4(0, 0, 0, 0);
    tile = Tile{only.x, only.y, only.z, only.w};
    cluster_wait();   // all CTAs have started
    for (int row = warp; row < tile.rows; row += kThreads / 32) {
      const int owner = row / owned;
      const float4 v = *reinterpret_cast<const float4*>(smem + (row * kPartLd + 4 * lane) * 4);
      st_cluster_f4(mapa_u32(smem_u32(done_tile), owner) + ((split * owned + row - owner * owned) * kPartLd + 4 * lane) * 4, v);
    }
    if (lane == 0) st_cluster_i32(mapa_u32(smem_u32(gave_up_of), warp % p.splits) + split * 4, *gave_up);
    cluster_sync_all();
    const bool lost = __any_sync(0xffffffffu, lane < p.splits && gave_up_of[lane] != 0);
    const int ch = tile.ch0 + 4 * lane;
    float bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = p.bias != nullptr && ch + j < p.n ? bias_at(p.bias + ch + j) : 0.f;
    for (int i = warp; i < owned && !lost; i += kThreads / 32) {
      const int row = split * owned + i;
      if (row >= tile.rows) break;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int e = 0; e < p.splits; ++e) {
        const float4 u = *reinterpret_cast<const float4*>(done_tile + ((e * owned + i) * kPartLd + 4 * lane) * 4);
        v = e == 0 ? u : make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
      }
      const float r[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
      __nv_bfloat16* const out = p.y + (tile.row0 + row) * p.n + ch;
      if (p.wide) {
        if (ch < p.n) *reinterpret_cast<uint2*>(out) = make_uint2(pack2(r[0], r[1]), pack2(r[2], r[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (ch + j < p.n) out[j] = f_to_bf16(r[j]);
      }
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_free<1>(tmem, TMEM);
  }
}

template <bool F8, int NT>
int launch(const GroupProduct& g, GemmArgs& p, int splits, cudaStream_t st) {
  using F = Form<NT>;
  static PerDevice attrs;
  B200_CUDA(attrs([] {
    return cudaFuncSetAttribute(group_gemm_kernel<F8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::smem(kMaxExperts));
  }));
  CUtensorMap tw, tx;
  int rc;
  if constexpr (F8) {
    if ((rc = make_tmap_sw128_u8(&tw, g.w, g.experts * g.n, g.k, f8_ld(g.k), kCh)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128_u8(&tx, g.x, g.rows, g.k, f8_ld(g.k), F::box)) != B200_OK) return rc;
  } else {
    if ((rc = make_tmap_sw128(&tw, 2, g.w, 1, g.experts * g.n, g.k, 0, g.k, kCh)) != B200_OK) return rc;
    if ((rc = make_tmap_sw128(&tx, 2, g.x, 1, g.rows, g.k, 0, g.k, F::box)) != B200_OK) return rc;
  }
  p.ch_blocks = (int)((g.n + kCh - 1) / kCh);
  p.ch_tiles = p.ch_blocks;
  // tiles that there can be: every group's last one may be short
  const int64_t row_tiles = g.starts ? g.rows / NT + std::min<int64_t>(g.experts, g.rows) : (g.rows + NT - 1) / NT, most = row_tiles * p.ch_tiles;
  p.splits = splits;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.splits > 1 ? most * p.splits : std::min<int64_t>(most, 148 * F::per_sm)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = F::smem((int)g.experts);
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
  B200_CUDA(cudaLaunchKernelEx(&cfg, group_gemm_kernel<F8, NT>, tw, tx, (const GemmArgs)p));
  return B200_OK;
}

// Rows of a tile (16 to 128 here, or a tile of group_gemm_wide.cu) and CTAs to a tile: what the whole call is estimated to take, in µs.  W cannot come faster than
// memory gives it; a CTA needs 0.25 (16 rows) to 0.5 µs (128) for 128 bytes of k, a wide one 0.49 (bf16 0.38 a pair), and something for a tile's end; two CTAs on an SM 1.45
// times that each; partial tiles that meet cost 2 to 4.5 µs.  The rates are fitted to 189 calls — 1 to 4 096 rows, up to 20 000 over 8 to 64 experts, seven and five
// matrices — in all the forms that can run: 13 of those calls take more than 5 % longer than in the best form, the worst 12 %.  For one of each, the way that is taken and,
// in brackets, others: 200 × 4 096 × 14 336 33 µs in tiles of 128 rows and two CTAs to each (37, 64 and two; 42, 64 and four), 512 × 4 096 × 14 336 55 wide (53, 128: one of those that
// are not cut best), 768 × 4 096 × 4 096 22 wide (34, 128), 512 × 2 048 × 2 048 11.1 with 64 (12.0, 32; 12.3, 128), 1 × 896 × 4 864 7.0 with eight CTAs to a tile (8.0, four).
// b200_product_way tells the way that any call takes.
struct Way {
  int rows, splits;   // rows 0: wide
};
Way choose(const GroupProduct& g, bool f8) {
  auto up = [](double a, double b) { return std::ceil(a / b); };
  const double groups = g.starts ? (double)std::min<int64_t>(g.experts, g.rows) : 1, average = (double)g.rows / groups;
  const double k_blocks = up((double)g.k, f8 ? 128 : 64), stream = groups * (double)g.n * (double)g.k * (f8 ? 1 : 2) / 6.8e6;
  // groups are unlike: four tenths of a last tile are empty on average, and no group has less than a tile
  auto row_tiles = [&](int rows) { return g.starts ? groups * std::max(1.0, average / rows + 0.4) : up(average, rows); };
  Way best{0, 1};
  // wide: a CTA of 128 rows in 8 bits, a pair of 256 in bf16
  double least = f8 && g.experts > kWideExperts8
                     ? 1e30
                     : 5.0 + std::max(stream, up(row_tiles(f8 ? 128 : 256) * up((double)g.n, 256), f8 ? 148 : 74) * (k_blocks * (f8 ? 0.49 : 0.38) + 1.35));
  for (int rows = 16; rows <= 128; rows *= 2) {
    const double tiles = row_tiles(rows) * up((double)g.n, kCh), each = (f8 ? 0.24 : 0.25) + (f8 ? 0.0021 : 0.0009) * std::min<double>(rows, average);
    for (int splits = 1; splits <= kMaxSplits && (splits == 1 || k_blocks >= 2 * splits); splits *= 2) {
      constexpr int kOne[4] = {148, 74, 33, 15}, kTwo[4] = {296, 148, 70, 32};   // clusters that the SMs hold at once
      const int i = splits == 1 ? 0 : splits == 2 ? 1 : splits == 4 ? 2 : 3;
      const double share = rows <= 64 && tiles * splits > 148 ? 1.45 : 1.0;
      const int hold = rows <= 64 ? kTwo[i] : kOne[i];
      if (splits > 1 && (g.starts ? (g.rows / rows + groups) * up((double)g.n, kCh) : tiles) > hold) break;   // (a cluster that comes later starts from nothing)
      const double us =
          4.9 + (splits > 1 ? 1.2 + 0.3 * splits + 0.008 * rows : 0.0) + std::max(stream, up(tiles, hold) * (up(k_blocks, splits) * each * share + 0.6));
      if (us < least) {
        least = us;
        best = Way{rows, splits};
      }
    }
  }
  return best;
}

template <bool F8>
int launch_for(const GroupProduct& g, GemmArgs& p, cudaStream_t st) {
  const Way way = choose(g, F8);
  switch (way.rows) {
    case 16: return launch<F8, 16>(g, p, way.splits, st);
    case 32: return launch<F8, 32>(g, p, way.splits, st);
    case 64: return launch<F8, 64>(g, p, way.splits, st);
    case 128: return launch<F8, 128>(g, p, way.splits, st);
    default: return launch_group_wide(g, p, st);
  }
}

}  // namespace

void group_way(const GroupProduct& g, bool f8, int32_t* rows, int32_t* splits) {
  const Way way = choose(g, f8);
  *rows = way.rows;
  *splits = way.splits;
}

int launch_group_product(const GroupProduct& g, cudaStream_t st) {
  GemmArgs p{};
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
  p.k_blocks = (int)(g.x_scale != nullptr ? f8_blocks(g.k) : (g.k + 63) / 64);
  p.wide = g.n % 8 == 0 && aligned16(g.y);
  p.ahead = g.x_in_front;
  return g.x_scale != nullptr ? launch_for<true>(g, p, st) : launch_for<false>(g, p, st);
}

}  // namespace b200

extern "C" {

static int check_sizes(const char* what, int64_t rows, int64_t experts, int64_t n, int64_t k) {
  using namespace b200;
  B200_CHECK_ARG(rows >= 1 && rows < 1 << 24, "%s: %lld rows out of range", what, (long long)rows);
  B200_CHECK_ARG(experts >= 1 && experts <= kMaxExperts && n >= 1 && n <= 1 << 20 && k >= 1 && k <= 1 << 24 && experts * n < 1ll << 31,
                 "%s: %lld matrices [%lld, %lld] out of range", what, (long long)experts, (long long)n, (long long)k);
  return B200_OK;
}
static int check_product(const char* what, const void* y, const void* x, const void* w, int64_t rows, int64_t experts, int64_t n, int64_t k) {
  using namespace b200;
  const int rc = check_sizes(what, rows, experts, n, k);
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(y && x && w, "%s: null pointer", what);
  B200_CHECK_ARG(aligned16(x, w), "%s: x and the weight must be 16-byte aligned", what);
  return B200_OK;
}

int b200_product_way(int64_t rows, int64_t experts, int64_t n, int64_t k, int32_t eight_bits, int32_t* tile_rows, int32_t* ctas) {
  using namespace b200;
  B200_CHECK_ARG(tile_rows && ctas && (experts != 0 || eight_bits), "product_way: null pointer, or one matrix in bf16");
  const int rc = check_sizes("product_way", rows, experts == 0 ? 1 : experts, n, k);
  if (rc != B200_OK) return rc;
  GroupProduct g{};
  g.rows = rows;
  g.experts = experts == 0 ? 1 : experts;
  g.n = n;
  g.k = k;
  g.starts = experts == 0 ? nullptr : tile_rows;   // (whether there are groups: no estimate reads them)
  group_way(g, eight_bits != 0, tile_rows, ctas);
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

int b200_f8_linear_of_bf16(void* y, void* q, float* scale, const void* x, const b200_f8_weight* w, const void* bias, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(x && w && scale && w->scale && w->experts == 1, "f8_linear_of: null pointer, or a weight of experts");
  if ((rc = check_product("f8_linear_of", y, q, w->q, rows, 1, w->n, w->k)) != B200_OK) return rc;
  if ((rc = launch_f8_rows(q, scale, x, w->k, rows, nullptr, rows, w->k, (cudaStream_t)stream)) != B200_OK) return rc;
  return launch_group_product({y, q, scale, w->q, w->scale, nullptr, bias, rows, 1, w->n, w->k, true}, (cudaStream_t)stream);
}

int b200_f8_grouped_of_bf16(void* y, void* q, float* scale, const void* x, const b200_f8_weight* w, const int32_t* starts, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(x && w && scale && w->scale && starts, "f8_grouped_of: null pointer");
  if ((rc = check_product("f8_grouped_of", y, q, w->q, rows, w->experts, w->n, w->k)) != B200_OK) return rc;
  if ((rc = launch_f8_rows(q, scale, x, w->k, rows, nullptr, rows, w->k, (cudaStream_t)stream)) != B200_OK) return rc;
  return launch_group_product({y, q, scale, w->q, w->scale, starts, nullptr, rows, w->experts, w->n, w->k, true}, (cudaStream_t)stream);
}

int b200_grouped_bf16(void* y, const void* x, const void* w, const int32_t* starts, int64_t rows, int64_t experts, int64_t n, int64_t k, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_product("grouped", y, x, w, rows, experts, n, k)) != B200_OK) return rc;
  B200_CHECK_ARG(starts && k % 8 == 0, "grouped: null pointer, or k=%lld that is no multiple of 8", (long long)k);
  return launch_group_product({y, x, nullptr, w, nullptr, starts, nullptr, rows, experts, n, k}, (cudaStream_t)stream);
}

}  // extern "C"
