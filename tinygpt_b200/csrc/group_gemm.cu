// group_gemm.cu — products of rows with the matrix of their group, on the 5th-generation tensor cores:  y[r] = W[e]·x[r] for the rows r of group e.
//
// One kernel for bf16 and for 8 bits with scales, for one matrix (a Linear) and for many (experts, rows sorted by expert).  W is the A operand: a tile is
// 128 of its rows (channels) × up to NT rows of x, and the product's N is what the tile really holds, rounded up to 16.  So a group of three rows costs a stream of its
// matrix and little else, and a group that ends inside a tile costs no idle rows.
//
// Warp-specialised, persistent over the tiles:
//   warp 0   TMA: of every 128 bytes of k 128 rows of W and the tile's rows of x, into a ring of shared memory
//   warp 1   one thread issues four products (K = 32 bytes) per 128 bytes
//   warp 2   8 bits: the products of x's and W's scales, NT of them for each block of 128 entries, fetched some blocks ahead
//   warp 3   rows of no group are zeroed
//   warps 4 … 11   the sums: a warp has a quarter of the channels and half of the rows, as fragments of 8 × 8 (lane 4r + c: channel r, rows 2c and 2c + 1), so
//            that a lane needs a quarter of the factors and a transposing store to shared memory makes rows of y of them
// 8 bits: W has a scale for 128 × 128 entries and x one for 128 entries of a row, so that 128 entries of k meet one factor per row of x, and the sums of 128
// entries — a slot of tensor memory each — are scaled and added in fp32 registers; two to four slots keep the tensor cores running meanwhile.
// bf16: a slot holds the sums over all of k.
// Tiles of up to 256 rows belong to pairs of CTAs (cta_group::2): 256 channels, each CTA brings its 128 of them and half of the rows, and sums its own channels.
#include "f8.cuh"
#include "tc.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kCh = 128, kWBytes = kCh * 128, kThreads = 384, kEpiWarps = 8;
constexpr int kMaxSplits = 8;
constexpr int kPatch = 16 * 64;            // 16 rows of y, 32 channels of a warp
constexpr int kPartLd = kCh + 4;            // floats from row to row of a partial tile: a fragment's lanes meet 32 banks
constexpr int kRegsFew = 72, kRegsMany = 216, kRegsLaunch = 168;   // where they are shared out unevenly
static_assert(128 * kRegsFew + 256 * kRegsMany <= kThreads * kRegsLaunch, "no warp waits for registers that the launch does not have");
constexpr unsigned kWaitCode = 0x67000000u;

struct Args {
  __nv_bfloat16* y;
  const float *sx, *sw;
  const int32_t* starts;
  const __nv_bfloat16* bias;
  unsigned* err;
  int64_t rows;
  int n, k_blocks, experts, ch_tiles, ch_blocks, splits;   // ch_tiles: of 128 channels, a pair's of 256
  bool wide;    // y takes stores of 16 bytes
};

template <int NT>
struct Form {
  static constexpr int group = NT == 256 ? 2 : 1;      // CTAs to a tile
  static constexpr int per_sm = NT <= 64 ? 2 : 1;
  static constexpr int x_rows = NT / group, x_bytes = x_rows * 128, stage = kWBytes + x_bytes;   // of a CTA
  static constexpr int stages = NT <= 32 ? 5 : NT == 64 ? 4 : 6;
  static constexpr int box = x_rows < 32 ? x_rows : 32;  // rows of x in a TMA box
  static constexpr int slots8 = NT == 256 ? 2 : 4;     // of tensor memory, 8 bits
  static constexpr int lag = 3;                        // blocks that factors are asked for ahead
  static constexpr int ahead = 2 * slots8 + 1 + lag;   // blocks of factors in shared memory: see where they are written
  static constexpr int f_slot = NT < 32 ? 32 : NT;
  static constexpr int cols = NT / 2;                  // rows of x of a summing warp
  static constexpr int ring = stages * stage;
  static constexpr int tables = 1024 + ring + kEpiWarps * kPatch + ahead * f_slot * 4 + 512;
  static constexpr int smem(int experts) { return tables + experts * 12; }
  // 8 bits, 256 rows: a thread that sums holds 128 of them.  The four warps that do not give registers up: 128·72 + 256·216 of the launch's 384·168.
  static constexpr bool uneven = NT == 256;
  static constexpr int tmem(int slots) { return slots * NT < 32 ? 32 : slots * NT; }
};
static_assert(Form<16>::smem(64) <= 113 * 1024 && Form<32>::smem(64) <= 114 * 1024 && Form<64>::smem(64) <= 114 * 1024, "two CTAs to an SM");
static_assert(Form<128>::smem(kMaxExperts) <= 227 * 1024 && Form<256>::smem(kMaxExperts) <= 227 * 1024, "room");
static_assert(Form<128>::ring >= 128 * kPartLd * 4 && Form<64>::ring >= 64 * kPartLd * 4 && Form<16>::ring >= 16 * kPartLd * 4, "a partial tile fits in the drained ring");

// D[tmem] (+)= A·B over 32 entries of 8 bits
template <int GROUP>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  if constexpr (GROUP == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::f8f6f4: D = F32 (bits 4-5 = 1), A = B = e4m3 (0), both K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28
__device__ __forceinline__ uint32_t idesc_of(bool eight, int m, int n) {
  const uint32_t shape = ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24) | (1u << 4);
  return eight ? shape : shape | (1u << 7) | (1u << 10);
}

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
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// a wait of a whole warp that mostly finds what it waits for
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, err, code));
}
// where the factor of row j of a tile lies: a lane that holds rows 8i + 2c, + 1 finds those of four i side by side
__device__ __forceinline__ int factor_at(int j) { return (j & ~31) + (j % 8 / 2) * 8 + (j % 32 / 8) * 2 + j % 2; }
// Arrives in another CTA.  What it tells is that tensor memory was read (the fence in front); no memory is handed over, so that no release at the cluster's
// scope is needed, which takes some 700 cycles.
__device__ __forceinline__ void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// two fp32 numbers in a 64-bit register: one instruction multiplies and adds both
template <bool B>
struct Is {
  static constexpr bool value = B;
};
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

// Which rows and channels a tile has.  Tiles run over the row tiles of a group first (its matrix's rows stay in L2), then over channels, then over groups.
struct Tile {
  int64_t row0;
  int rows, ch0, expert;
};

template <bool F8, int NT>
__global__ void __launch_bounds__(kThreads, Form<NT>::per_sm) group_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                                                                               const Args p) {
  using F = Form<NT>;
  constexpr int GROUP = F::group, ST = F::stages, SLOTS = F8 ? F::slots8 : 2, COLS = F::cols, TMEM = F::tmem(SLOTS), AHEAD = F::ahead, LAG = F::lag;
  constexpr int PIECE = COLS < 32 ? COLS : 32;      // rows of 16 channels that are loaded at once
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const sx = smem + ST * kWBytes;
  uint8_t* const patches = smem + F::ring;                                         // [summing warps][16 rows][32 channels], bf16
  float* const factors = reinterpret_cast<float*>(patches + kEpiWarps * kPatch);   // [AHEAD][NT]
  uint64_t* const full = reinterpret_cast<uint64_t*>(factors + AHEAD * F::f_slot);   // [stages], a pair's first CTA's
  uint64_t* const empty = full + ST;
  uint64_t* const sums_full = empty + ST;                                          // [slots]
  uint64_t* const sums_empty = sums_full + 4;                                      // a pair's first CTA's
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sums_empty + 4);
  int* const gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  float* const w_scale = reinterpret_cast<float*>(gave_up + 1);                       // [AHEAD]
  int* const ends = reinterpret_cast<int*>(smem + F::tables - 1024);   // [experts] row tiles up to and with e
  int* const froms = ends + p.experts;                                               // first row, rows
  int* const counts = froms + p.experts;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = GROUP == 2 || p.splits > 1 ? (int)cluster_rank() : 0;
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
    fence_mbar_init();
    *gave_up = 0;
  }
  if (warp == 1) tmem_alloc<GROUP>(tmem_slot, TMEM);
  pdl_wait();
  pdl_trigger();
  if (warp == 3) {   // every lane a run of groups; their rows lie inside the call's, whatever the starts say
    const int each = (p.experts + 31) / 32, e0 = min(lane * each, p.experts), e1 = min(e0 + each, p.experts);
    int mine = 0;
    for (int e = e0; e < e1; ++e) {
      const int64_t from = p.starts == nullptr ? 0 : min(max((int64_t)p.starts[e], (int64_t)0), p.rows);
      const int64_t count = p.starts == nullptr ? p.rows : max(min((int64_t)p.starts[e + 1], p.rows) - from, (int64_t)0);
      froms[e] = (int)from;
      counts[e] = (int)count;
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
      upto += (counts[e] + NT - 1) / NT;
      ends[e] = upto;
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (GROUP == 2) cluster_sync_all();   // the pair's barriers exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int split = GROUP == 1 ? rank : 0;
  const int64_t tiles = (int64_t)ends[p.experts - 1] * p.ch_tiles;
  const int64_t first = blockIdx.x / (GROUP * p.splits), step = p.splits > 1 ? tiles : gridDim.x / GROUP;   // a cluster that splits k takes one tile
  const int kb0 = (int)((int64_t)p.k_blocks * split / p.splits), kb1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
  auto tile_at = [&](int64_t t) {
    const int at = (int)(t / p.ch_tiles);   // this group's: ends[e − 1] ≤ at < ends[e]
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (ends[mid] > at) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo > 0 ? ends[lo - 1] : 0, row_tiles = ends[lo] - before, count = counts[lo];
    const int local = (int)(t - (int64_t)before * p.ch_tiles);
    const int i = local % row_tiles, each = ((count + row_tiles - 1) / row_tiles + 15) / 16 * 16;   // alike, and none is empty
    return Tile{froms[lo] + (int64_t)i * each, min(each, count - i * each), (local / row_tiles * GROUP + (GROUP == 2 ? rank : 0)) * kCh, lo};
  };
  auto up16 = [](int v) { return (v + 15) / 16 * 16; };

  if (warp < 4) {
    if constexpr (F8 && F::uneven) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0) {
      if (lane == 0) {
        int s = 0;
        uint32_t ph = 1;
        for (int64_t t = first; t < tiles && ok; t += step) {
          const Tile tile = tile_at(t);
          const int mine = up16(tile.rows) / GROUP, row0 = (int)tile.row0 + (GROUP == 2 ? rank * mine : 0);
          const int boxes = (mine + F::box - 1) / F::box, w_row = tile.expert * p.n + tile.ch0;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!(ok = mbar_wait_limited(&empty[s], ph, p.err, kWaitCode | 1))) break;
            uint8_t *const w_to = smem + s * kWBytes, *const x_to = sx + s * F::x_bytes;
            const int k0 = kb * (F8 ? 128 : 64);
            if constexpr (GROUP == 2) {
              const uint32_t bar = mapa_u32(smem_u32(&full[s]), 0);
              if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (kWBytes + boxes * F::box * 128));
              tma_load_2d_pair(w_to, &tmap_w, k0, w_row, bar);
              for (int b = 0; b < boxes; ++b) tma_load_2d_pair(x_to + b * F::box * 128, &tmap_x, k0, row0 + b * F::box, bar);
            } else {
              mbar_arrive_expect_tx(&full[s], kWBytes + boxes * F::box * 128);
              tma_load_2d(w_to, &tmap_w, k0, w_row, &full[s]);
              for (int b = 0; b < boxes; ++b) tma_load_2d(x_to + b * F::box * 128, &tmap_x, k0, row0 + b * F::box, &full[s]);
            }
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
          }
        }
        if (!ok) drain_async();
      }
    } else if (warp == 1) {
      if ((GROUP == 1 || rank == 0) && elect_one()) {
        const uint32_t w0 = desc_lo(smem_u32(smem)), x0 = desc_lo(smem_u32(sx));
        int s = 0, slot = 0;
        uint32_t ph = 0, slot_ph = 1;
        bool ready = false;   // of the next stage, looked at before the products of this one go out
        for (int64_t t = first; t < tiles && ok; t += step) {
          const Tile tile = tile_at(t);
          const uint32_t idesc = idesc_of(F8, kCh * GROUP, up16(tile.rows));
          for (int kb = kb0; kb < kb1; ++kb) {
            if (F8 || kb == kb0) {
              if (!(ok = mbar_wait_limited(&sums_empty[slot], slot_ph, p.err, kWaitCode | 2))) break;
            }
            if (!ready && !(ok = mbar_wait_limited(&full[s], ph, p.err, kWaitCode | 3))) break;
            tc_fence_after();
            const uint32_t w = w0 + s * (kWBytes >> 4), x = x0 + s * (F::x_bytes >> 4), d = tmem + slot * NT;
            uint64_t* const done = &empty[s];
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
            ready = mbar_test(&full[s], ph);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (F8) umma_f8<GROUP>(d, w + 2 * k, x + 2 * k, idesc, k > 0 ? 1u : 0u);
              else umma_lo<GROUP>(d, w + 2 * k, x + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
            }
            if constexpr (GROUP == 2) umma_commit_pair(done);
            else umma_commit(done);
            if (F8 || kb == kb1 - 1) {
              if constexpr (GROUP == 2) umma_commit_pair(&sums_full[slot]);
              else umma_commit(&sums_full[slot]);
              if (++slot == SLOTS) {
                slot = 0;
                slot_ph ^= 1;
              }
            }
          }
        }
        if (!ok) drain_async();
      }
    } else if (warp == 2) {
      if constexpr (F8) {
        // Of unit u — a block of a tile — x's scales and W's are asked for LAG units before they are multiplied.  A slot's barrier takes unit u's arrival when its
        // phase before, unit u − SLOTS, is complete.  Then the products of that unit are done, so every warp has released unit u − 2·SLOTS and needs nothing of the units in
        // front of that one any more: a ring of 2·SLOTS + 1 + LAG units is never written where it is read.
        constexpr int PER = (NT + 31) / 32;
        const int64_t units = first < tiles ? ((tiles - first + step - 1) / step) * (kb1 - kb0) : 0;
        int64_t t = first;
        int kb = kb0, into = 0, from_slot = 0, slot = 0;
        uint32_t ph = 1;
        Tile tile{};
        auto ask = [&]() {
          if (kb == kb0) tile = tile_at(t);
          const float* const from = p.sx + (int64_t)kb * p.rows + tile.row0 + lane;
          float* const to = factors + into * F::f_slot + factor_at(lane);
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < tile.rows) cp_async4(to + 32 * i, from + 32 * i);
          if (lane == 0) cp_async4(&w_scale[into], p.sw + ((int64_t)tile.expert * p.ch_blocks + min(tile.ch0 / kCh, p.ch_blocks - 1)) * p.k_blocks + kb);
          if (++kb == kb1) {
            kb = kb0;
            t += step;
          }
          if (++into == AHEAD) into = 0;
        };
        for (int64_t u = -LAG; u < units; ++u) {
          if (u >= 0 && !(ok = warp_wait(&sums_full[slot], ph, p.err, kWaitCode | 4))) break;
          if (u + LAG < units) ask();
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
      if (p.starts != nullptr) {   // rows in front of the first group and behind the last
        const int64_t from = min(max((int64_t)p.starts[0], (int64_t)0), p.rows), to = min(max((int64_t)p.starts[p.experts], from), p.rows);
        for (int64_t r = blockIdx.x; r < p.rows - (to - from); r += gridDim.x) {
          __nv_bfloat16* const out = p.y + (r < from ? r : r - from + to) * p.n;
          for (int i = lane; i < p.n; i += 32) out[i] = f_to_bf16(0.f);
        }
      }
    }
  } else {
    if constexpr (F8 && F::uneven) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
    const int quad = warp & 3, half = (warp - 4) >> 2, r = lane / 4, c = lane % 4;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + half * COLS;
    uint8_t* const patch = patches + (warp - 4) * kPatch;
    // lane 8m + i of a transposing store: row i, channels 8m … of 32, at a place that lets eight rows meet all banks; and row 8 + i
    const uint32_t put_at = smem_u32(patch) + lane % 8 * 64 + (((lane / 8) ^ (lane % 8 / 2)) << 4);
    const uint8_t* const get_at = patch + lane / 4 * 64 + (((lane % 4) ^ (lane / 4 / 2)) << 4);
    int slot = 0, fslot = 0;
    uint32_t slot_ph = 0;
    for (int64_t t = first; t < tiles; t += step) {
      const Tile tile = tile_at(t);
      const int mine = tile.rows - half * COLS;   // rows of this half
      const int ch0 = tile.ch0 + quad * 32;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = p.bias != nullptr && ch0 + r + 8 * e < p.n ? bf16_to_f(p.bias[ch0 + r + 8 * e]) : 0.f;
      __nv_bfloat16* const out = p.y + (tile.row0 + half * COLS) * p.n + ch0;
      // Rows j … j + 7 of this half, 32 channels: v[e][i] is channel r + 8e, row j + 2c + i.  Every second call stores sixteen rows.
      auto put8 = [&](int j, float2 (&v)[4]) {
        if (GROUP == 1 && p.splits > 1) {   // [row][channel] where the operands were: every product has read them
          float* const part = reinterpret_cast<float*>(smem) + (half * COLS + j + 2 * c) * kPartLd + quad * 32 + r;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            part[8 * e] = v[e].x;
            part[8 * e + kPartLd] = v[e].y;
          }
          return;
        }
        store_transposed(put_at + j % 16 * 64, pack2(v[0].x + bias[0], v[0].y + bias[0]), pack2(v[1].x + bias[1], v[1].y + bias[1]),
                         pack2(v[2].x + bias[2], v[2].y + bias[2]), pack2(v[3].x + bias[3], v[3].y + bias[3]));
        if (j % 16 == 0 && j + 8 < COLS && j + 8 < mine) return;
        __syncwarp();
        const int j0 = j / 16 * 16;
        if (p.wide) {   // n is a multiple of 8: sixteen bytes lie inside a row or outside it
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = j0 + 8 * i + lane / 4;
            if (row < mine && row < COLS && ch0 + lane % 4 * 8 < p.n)
              *reinterpret_cast<uint4*>(out + (int64_t)row * p.n + lane % 4 * 8) = *reinterpret_cast<const uint4*>(get_at + i * 512);
          }
        } else if (ch0 + lane < p.n) {
          for (int i = 0; i < 16 && j0 + i < min(mine, COLS); ++i)
            out[(int64_t)(j0 + i) * p.n + lane] =
                *reinterpret_cast<const __nv_bfloat16*>(patch + i * 64 + (((lane / 8) ^ (i % 8 / 2)) << 4) + lane % 8 * 2);
        }
        __syncwarp();
      };
      auto release = [&]() {   // the slot may be filled again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (GROUP == 2) arrive_at(mapa_u32(smem_u32(&sums_empty[slot]), 0));
          else mbar_arrive(&sums_empty[slot]);
        }
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
          constexpr int PIECES = 2 * (COLS / PIECE);   // in turn channels 0 … 15 and 16 … 31
          const int pieces = ALL ? PIECES : 2 * ((mine + PIECE - 1) / PIECE);
          uint32_t d[2][PIECE / 2];
          float2 f[PIECE / 8];
          tmem_frag(at, d[0]);
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            if (!ALL && i >= pieces) break;
            uint32_t(&v)[PIECE / 2] = d[i % 2];
            if (i % 2 == 0) {
#pragma unroll
              for (int g = 0; g < PIECE / 8; ++g) {
                if constexpr (PIECE >= 16) {
                  if (g % 2 == 0) {
                    const float4 both = *reinterpret_cast<const float4*>(factor + i / 2 * PIECE + 2 * g);
                    f[g] = make_float2(both.x, both.y);
                    f[g + 1] = make_float2(both.z, both.w);
                  }
                } else {
                  f[g] = *reinterpret_cast<const float2*>(factor);
                }
              }
            }
            tmem_ready(v);
            if (i + 1 < PIECES && (ALL || i + 1 < pieces)) tmem_frag(at + (i + 1) / 2 * PIECE + ((uint32_t)((i + 1) % 2 * 16) << 16), d[(i + 1) % 2]);
            else release();
#pragma unroll
            for (int g = 0; g < PIECE / 8; ++g) {
              const uint64_t fg = pair_of(f[g].x, f[g].y);
              uint64_t(&sum)[4] = acc[i / 2 * (PIECE / 8) + g];
              sum[i % 2 * 2] = fma_pair(pair_of(v[4 * g], v[4 * g + 1]), fg, sum[i % 2 * 2]);
              sum[i % 2 * 2 + 1] = fma_pair(pair_of(v[4 * g + 2], v[4 * g + 3]), fg, sum[i % 2 * 2 + 1]);
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
      }
    }
  }
  if (!ok) *gave_up = 1;
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if constexpr (GROUP == 2) {
    cluster_sync_all();   // neither CTA still reads the pair's operands, barriers or sums
  } else if (p.splits > 1) {
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
        const uint32_t at = smem_u32(smem) + (row * kPartLd + 4 * lane) * 4;
        float4 of[kMaxSplits];
#pragma unroll
        for (int e = 0; e < kMaxSplits; ++e) of[e] = e < p.splits ? ld_cluster_f4(mapa_u32(at, e)) : make_float4(0.f, 0.f, 0.f, 0.f);
        float4 v = of[0];
#pragma unroll
        for (int e = 1; e < kMaxSplits; ++e) v = make_float4(v.x + of[e].x, v.y + of[e].y, v.z + of[e].z, v.w + of[e].w);
        __nv_bfloat16* const out = p.y + (tile.row0 + row) * p.n + ch;
        const float r[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
        if (p.wide) {
          if (ch < p.n) *reinterpret_cast<uint2*>(out) = make_uint2(pack2(r[0], r[1]), pack2(r[2], r[3]));
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
    tmem_free<GROUP>(tmem, TMEM);
  }
  if constexpr (GROUP == 2) cluster_sync_all();
}

template <bool F8, int NT>
int launch(const GroupProduct& g, Args& p, cudaStream_t st) {
  using F = Form<NT>;
  static PerDevice attrs;
  B200_CUDA(attrs([] {
    cudaFuncAttributes a{};
    const cudaError_t e = cudaFuncGetAttributes(&a, group_gemm_kernel<F8, NT>);
    if (e != cudaSuccess) return e;
    if (F8 && F::uneven && a.numRegs != kRegsLaunch) return cudaErrorInvalidDeviceFunction;   // (the shares would not add up)
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
  p.ch_tiles = (p.ch_blocks + F::group - 1) / F::group;
  // tiles that there can be: every group's last one may be short
  const int64_t row_tiles = g.starts ? g.rows / NT + std::min<int64_t>(g.experts, g.rows) : (g.rows + NT - 1) / NT, most = row_tiles * p.ch_tiles;
  const int64_t room = 148 / F::group * F::per_sm;
  p.splits = 1;
  while (F::group == 1 && p.splits < kMaxSplits && most * p.splits * 2 <= room && p.k_blocks >= 4 * p.splits) p.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.splits > 1 ? most * p.splits : std::min(most, room) * F::group));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = F::smem((int)g.experts);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)(p.splits * F::group);
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
  p.k_blocks = (int)(g.x_scale != nullptr ? f8_blocks(g.k) : (g.k + 63) / 64);
  p.wide = g.n % 8 == 0 && aligned16(g.y);
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
