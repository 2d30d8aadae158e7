// group_gemm.cuh — what the two kernels of grouped products share: arguments, 8-bit products, the groups' tiles, waits of a warp, stores of finished tiles.
#pragma once
#include "f8.cuh"
#include "tc.cuh"

namespace b200 {

struct GemmArgs {
  __nv_bfloat16* y;
  const float *sx, *sw;
  const int32_t* starts;
  const __nv_bfloat16* bias;
  unsigned* err;
  int64_t rows;
  int n, k_blocks, experts, ch_tiles, ch_blocks, splits;   // ch_tiles: of a tile's channels; ch_blocks: of 128 channels
  bool wide;    // y takes stores of 16 bytes
  bool ahead;   // W, groups and bias may be read before the kernel in front is done
};
// tiles of 256 channels (group_gemm_wide.cu); in 8 bits for so many matrices
constexpr int kWideExperts8 = 512;
int launch_group_wide(const GroupProduct& g, GemmArgs& p, cudaStream_t st);

#ifdef __CUDACC__
// D[tmem] (+)= A·B over 32 bytes of k, of 8-bit entries or bf16, where `lead`.  A whole warp comes here with the same operands and one of its lanes is the leading
// one: they stay in uniform registers.  Issued by a lane in a branch of its own four products and their commit take 445 cycles, however few columns they
// have, so 249 — a tile of 128 × 128 needs 256 — and the products of 128 × 256 are there 646 cycles after the first one's issue, for 801.
template <bool F8, int GROUP>
__device__ __forceinline__ void umma_by(uint32_t lead, uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
#define B200_UMMA(group, kind)                                                                                                                              \
  asm volatile(                                                                                                                                             \
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"     \
      "@q tcgen05.mma.cta_group::" group ".kind::" kind " [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc),          \
      "r"(accumulate), "r"(lead)                                                                                                                            \
      : "memory")
  if constexpr (GROUP == 2) {
    if constexpr (F8) B200_UMMA("2", "f8f6f4");
    else B200_UMMA("2", "f16");
  } else {
    if constexpr (F8) B200_UMMA("1", "f8f6f4");
    else B200_UMMA("1", "f16");
  }
#undef B200_UMMA
}
// the barrier at this offset — in both CTAs of a pair — hears when what the leading lane has issued is done
template <int GROUP>
__device__ __forceinline__ void commit_by(uint32_t lead, uint64_t* bar) {
  if constexpr (GROUP == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3), "r"(lead)
        : "memory");
  else
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
                 "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void st_cluster_i32(uint32_t addr, int v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// what is the same in all lanes of a warp, where the compiler sees that it is
template <typename T>
__device__ __forceinline__ T uniform(T v) { return __shfl_sync(0xffffffffu, v, 0); }
// kind::f8f6f4: D = F32 (bits 4-5 = 1), A = B = e4m3 (0), both K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28
__device__ __forceinline__ uint32_t idesc_of(bool eight, int m, int n) {
  const uint32_t shape = ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24) | (1u << 4);
  return eight ? shape : shape | (1u << 7) | (1u << 10);
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Waits as mbar_wait_limited does, but asleep: a thread that polls takes issue slots from the warps that sum.  False after about two seconds.
__device__ __forceinline__ bool try_wait_asleep(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u) : "memory");   // ns, at most
  return ok != 0;
}
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  if (try_wait_asleep(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!try_wait_asleep(bar, parity)) {
    if (global_timer_ns() - t0 > 2000000000ull) {
      *reinterpret_cast<volatile unsigned*>(err) = code;
      __threadfence_system();
      return false;
    }
  }
  return true;
}
// of a whole warp
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  return __all_sync(0xffffffffu, wait_asleep(bar, parity, err, code));
}
// Arrives in another CTA.  What it tells is that tensor memory was read (the fence in front); no memory is handed over, so that no release at the cluster's
// scope is needed, which takes some 700 cycles.
__device__ __forceinline__ void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Groups and bias where the warp that reads them may not have waited for the kernel in front (`ahead`): whoever wrote them is done and L2 has what was written, so
// they are read from there, past an L1 of which nothing is promised before the wait.
__device__ __forceinline__ int start_at(const int32_t* p) { return __ldcg(p); }
__device__ __forceinline__ float bias_at(const __nv_bfloat16* p) { return bf16_lo(__ldcg(reinterpret_cast<const unsigned short*>(p))); }
template <bool B>
struct Is {
  static constexpr bool value = B;
};

// The row tiles of all groups, made by one warp: a group's rows (inside the call's, whatever the starts say) and the tiles of ROWS rows up to and with it.
struct Groups {
  int *ends, *froms, *counts;   // shared memory
  int experts;
  static constexpr int bytes(int experts) { return experts * 12; }
  __device__ __forceinline__ Groups(int* at, int n) : ends(at), froms(at + n), counts(at + 2 * n), experts(n) {}
  template <int ROWS>
  __device__ __forceinline__ void make(const int32_t* starts, int64_t rows, int lane) {
    const int each = (experts + 31) / 32, e0 = min(lane * each, experts), e1 = min(e0 + each, experts);
    int mine = 0;
    for (int e = e0; e < e1; ++e) {
      const int64_t from = starts == nullptr ? 0 : min(max((int64_t)start_at(starts + e), (int64_t)0), rows);
      const int64_t count = starts == nullptr ? rows : max(min((int64_t)start_at(starts + e + 1), rows) - from, (int64_t)0);
      froms[e] = (int)from;
      counts[e] = (int)count;
      mine += (int)((count + ROWS - 1) / ROWS);
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto -= mine;
    for (int e = e0; e < e1; ++e) {
      upto += (counts[e] + ROWS - 1) / ROWS;
      ends[e] = upto;
    }
  }
  // The group e that tile t is one of — its row tiles times ch_tiles tiles — from the group of a tile in front of it; local: its number there, row_tiles: how many
  // row tiles the group has.  Of a whole warp.  (A call has fewer than 2^31 tiles.)
  __device__ __forceinline__ void walk(int t, int ch_tiles, int lane, int& e, int& local, int& row_tiles) const {
    int before = 0;
    if (experts > 1) {
      const int at = t / ch_tiles;
      for (int from = e; from < experts; from += 32) {   // ends[e − 1] ≤ at < ends[e]
        const unsigned past = __ballot_sync(0xffffffffu, from + lane < experts && ends[from + lane] > at);
        if (past != 0) {
          e = from + __ffs(past) - 1;
          break;
        }
      }
      before = e > 0 ? ends[e - 1] : 0;
    }
    row_tiles = ends[e] - before;
    local = t - before * ch_tiles;
  }
};
// A CTA's tiles, which one warp finds ahead of those that work on them: a search and divisions take 1 000 cycles and more, in which a summing warp would let its slots fill.
struct Tile {
  int64_t row0;
  int rows, ch0, expert;
};
struct TileRing {
  static constexpr int places = 4, bytes = places * 32;
  uint64_t *full, *empty;
  int4* tiles;
  int at = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ TileRing(void* room) : full((uint64_t*)room), empty(full + places), tiles((int4*)(empty + places)) {}
  __device__ __forceinline__ void init(int takers) {
    for (int i = 0; i < places; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], takers);
    }
  }
  __device__ __forceinline__ void step() {
    if (++at == places) {
      at = 0;
      ph ^= 1;
    }
  }
  // both of a whole warp
  __device__ __forceinline__ bool give(int row0, int rows, int ch0, int expert, int lane, unsigned* err, unsigned code) {
    if (!warp_wait(&empty[at], ph ^ 1, err, code)) return false;
    if (lane == 0) {
      tiles[at] = make_int4(row0, rows, ch0, expert);
      mbar_arrive(&full[at]);
    }
    step();
    return true;
  }
  __device__ __forceinline__ bool take(Tile& tile, int lane, unsigned* err, unsigned code) {
    if (!warp_wait(&full[at], ph, err, code)) return false;
    const int4 v = tiles[at];
    tile = Tile{v.x, v.y, v.z, v.w};
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[at]);
    step();
    return true;
  }
};
// rows in front of the first group and behind the last, by one warp of every CTA
__device__ __forceinline__ void zero_other_rows(const GemmArgs& p, int lane) {
  if (p.starts == nullptr) return;
  const int64_t from = min(max((int64_t)p.starts[0], (int64_t)0), p.rows), to = min(max((int64_t)p.starts[p.experts], from), p.rows);
  for (int64_t r = blockIdx.x; r < p.rows - (to - from); r += gridDim.x) {
    __nv_bfloat16* const out = p.y + (r < from ? r : r - from + to) * p.n;
    if (p.wide)
      for (int i = lane * 8; i < p.n; i += 256) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
    else
      for (int i = lane; i < p.n; i += 32) out[i] = f_to_bf16(0.f);
  }
}
// A summing warp stores what it summed itself, through a piece of shared memory of rows × 32 channels in bf16, for stores of 64 bytes.  A row's sixteen bytes c lie at
// piece_at: eight lanes meet all banks, writing and reading.
__device__ __forceinline__ int piece_at(int row, int c) { return row * 64 + (c ^ (row >> 1 & 3)) * 16; }
__device__ __forceinline__ void store_piece(__nv_bfloat16* out, const uint8_t* piece, int rows, int width, const GemmArgs& p, int lane) {
  if (p.wide) {
    const int c = lane & 3;
    for (int row0 = lane >> 2; row0 < rows; row0 += 32) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(piece + piece_at(min(row0 + 8 * j, rows - 1), c));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row0 + 8 * j < rows && 8 * c < width) *reinterpret_cast<uint4*>(out + (int64_t)(row0 + 8 * j) * p.n + 8 * c) = v[j];
    }
  } else if (lane < width) {   // a lane has a channel of every row
#pragma unroll 8
    for (int r = 0; r < rows; ++r) out[(int64_t)r * p.n + lane] = *reinterpret_cast<const __nv_bfloat16*>(piece + piece_at(r, lane >> 3) + (lane & 7) * 2);
  }
}
#endif

}  // namespace b200
