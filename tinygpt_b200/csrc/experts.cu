// experts.cu — a layer of routed experts around its products (group_gemm.cu): the pairs (row, chosen expert) in the order of their experts, and the weighted sum of
// the experts' rows back into the rows that they came from.
#include "f8.cuh"
#include "tc.cuh"

#include <algorithm>

namespace b200 {

namespace {

// A stable counting sort by one CTA, or by a cluster of eight where there are many pairs: every warp takes a run of the pairs, 32 at a time in their order.
// Lanes that hold the same expert find each other (ballots of its bits), so a warp's count of an expert is its own and no atomics decide an order.
//   1. counts[warp][e];  2. the sum in front of each: experts first, then CTAs, then warps;  3. the runs again, each pair to its place
// Bound by latencies and by the instructions of the SMs that it has: 8 192 pairs take 5.4 µs with eight, 12.6 with one.
constexpr int kOrderWarps = 32, kOrderThreads = 32 * kOrderWarps, kOrderCtas = 8;
constexpr int kOrderKept = 16384;   // choices of a CTA that are kept in shared memory, the others are read twice

__global__ void __launch_bounds__(kOrderThreads) expert_order_kernel(int32_t* __restrict__ starts, int32_t* __restrict__ source, int32_t* __restrict__ place,
                                                                     const int32_t* __restrict__ chosen, int pairs, int top, int experts, int run) {
  extern __shared__ int counts[];   // [warps][ld]
  const int ld = experts | 1;       // (a warp that takes one expert of all warps meets all banks)
  int* const total = counts + kOrderWarps * ld;   // [experts]: this CTA's rows of e, then where they begin
  int* const all_of = total + experts;            // [experts]: all CTAs' rows of e
  int* const kept = all_of + experts;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = (int)cluster_rank(), ctas = (int)gridDim.x;
  const int64_t cta_from = min((int64_t)rank * kOrderWarps * run, (int64_t)pairs);   // (a run is a warp's)
  const int mine_all = (int)min((int64_t)kOrderWarps * run, pairs - cta_from);
  const int32_t* const own_chosen = chosen + cta_from;
  pdl_wait();
  pdl_trigger();
#pragma unroll 4
  for (int i = threadIdx.x; i < min(mine_all, kOrderKept); i += kOrderThreads) kept[i] = own_chosen[i];
  for (int i = threadIdx.x; i < kOrderWarps * ld; i += kOrderThreads) counts[i] = 0;
  __syncthreads();
  const int from = min(warp * run, mine_all), to = min(from + run, mine_all);
  const int bits = 32 - __clz(experts - 1);   // of an expert's number
  int* const own = counts + warp * ld;
  // the pairs of this warp's run: where they lie, their expert (−1: none) and its count in front of them
  auto walk = [&](auto at) {
#pragma unroll 1
    for (int i = from + lane; i - lane < to; i += 32) {
      const bool is = i < to;
      const int e = !is ? -1 : i < kOrderKept ? kept[i] : own_chosen[i];
      const bool valid = e >= 0 && e < experts;
      unsigned same = __ballot_sync(0xffffffffu, valid);
      for (int b = 0; b < bits; ++b) {
        const unsigned ones = __ballot_sync(0xffffffffu, e >> b & 1);
        same &= e >> b & 1 ? ones : ~ones;
      }
      int before = 0;
      if (valid) before = own[e];
      __syncwarp();
      if (valid && lane == __ffs(same) - 1) own[e] = before + __popc(same);
      __syncwarp();
      if (is) at(i, valid ? e : -1, before + __popc(same & ((1u << lane) - 1)));
    }
  };
  walk([](int, int, int) {});
  __syncthreads();
  for (int e = warp; e < experts; e += kOrderWarps) {   // a lane has a warp's count
    const int c = counts[lane * ld + e];
    int upto = c;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    counts[lane * ld + e] = upto - c;
    if (lane == 31) total[e] = upto;
  }
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  int before_me[kMaxExperts / kOrderThreads];   // rows of an expert in the CTAs in front of this one
#pragma unroll
  for (int j = 0; j < kMaxExperts / kOrderThreads; ++j) {
    const int e = threadIdx.x + j * kOrderThreads;
    int sum = 0, mine = 0;
    if (e < experts) {
      for (int r = 0; r < ctas; ++r) {
        if (r == rank) mine = sum;
        sum += ctas > 1 ? ld_cluster_i32(mapa_u32(smem_u32(total + e), r)) : total[e];
      }
      all_of[e] = sum;
    }
    before_me[j] = mine;
  }
  if (ctas > 1) cluster_sync_all();   // (nobody reads the counts any more)
  else __syncthreads();
  if (warp == 0) {   // every lane a run of experts
    const int each = (experts + 31) / 32, e0 = min(lane * each, experts), e1 = min(e0 + each, experts);
    int mine = 0;
    for (int e = e0; e < e1; ++e) mine += all_of[e];
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto -= mine;
    for (int e = e0; e < e1; ++e) {
      total[e] = upto;
      if (rank == 0) starts[e] = upto;
      upto += all_of[e];
    }
    const int all = __shfl_sync(0xffffffffu, upto, 31);
    if (rank == 0 && lane == 0) starts[experts] = all;
    for (int i = all + rank * 32 + lane; i < pairs; i += ctas * 32) source[i] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMaxExperts / kOrderThreads; ++j)
    if ((int)threadIdx.x + j * kOrderThreads < experts) total[threadIdx.x + j * kOrderThreads] += before_me[j];
  __syncthreads();
  walk([&](int i, int e, int number) {
    const int pair = (int)cta_from + i, to_place = e < 0 ? -1 : total[e] + number;
    if (e >= 0) source[to_place] = pair / top;
    place[pair] = to_place;
  });
}

// out[r] = bf16( Σ_t weights[r, t]·y[place[r, t]] ), t in order, fp32.  Eight channels a thread (WIDE) or one.
// 2 048 × 2 048 of four each 10.7 µs, 3.9 TB/s: a place, then its row, two latencies to a CTA.
template <bool WIDE>
__global__ void __launch_bounds__(256) expert_combine_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ y, const int32_t* __restrict__ place,
                                                             const float* __restrict__ weights, int64_t rows, int top, int n) {
  pdl_wait();
  pdl_trigger();
  constexpr int EACH = WIDE ? 8 : 1;
  const int pieces = n / EACH;
  const int64_t all = rows * pieces, y_rows = rows * top;
  const bool small = all < 1ll << 31;   // (a division of 64 bits: a hundred instructions)
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
    const int64_t row = small ? (int64_t)((uint32_t)at / (uint32_t)pieces) : at / pieces;
    const int i = (int)(at - row * pieces) * EACH;
    float acc[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) acc[e] = 0.f;
    for (int t0 = 0; t0 < top; t0 += 4) {   // four rows on their way together
      float w[4];
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t from = t0 + j < top ? (int64_t)place[row * top + t0 + j] : -1;
        const bool is = from >= 0 && from < y_rows;
        w[j] = is ? weights[row * top + t0 + j] : 0.f;
        v[j] = make_uint4(0, 0, 0, 0);
        if constexpr (WIDE) {
          if (is) v[j] = *reinterpret_cast<const uint4*>(y + from * n + i);
        } else {
          if (is) v[j].x = *reinterpret_cast<const uint16_t*>(y + from * n + i);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (WIDE) {
          float u[8];
          unpack8(v[j], u);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = fmaf(w[j], u[e], acc[e]);
        } else {
          acc[0] = fmaf(w[j], bf16_lo(v[j].x), acc[0]);
        }
      }
    }
    if constexpr (WIDE) *reinterpret_cast<uint4*>(out + row * n + i) = make_uint4(pack2(acc[0], acc[1]), pack2(acc[2], acc[3]), pack2(acc[4], acc[5]), pack2(acc[6], acc[7]));
    else out[row * n + i] = f_to_bf16(acc[0]);
  }
}

constexpr int64_t up256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// where the parts of a layer's workspace lie
struct ExpertsSpace {
  int64_t starts, source, place, q, scale, gate_up, a, a_scale, y, bytes;
};
ExpertsSpace experts_space(int64_t rows, int64_t top, int64_t experts, int64_t width, int64_t ff) {
  ExpertsSpace s{};
  const int64_t pairs = rows * top;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += up256(bytes);
    return from;
  };
  s.starts = take((experts + 1) * 4);
  s.source = take(pairs * 4);
  s.place = take(pairs * 4);
  s.q = take(pairs * f8_ld(width));
  s.scale = take(pairs * f8_blocks(width) * 4);
  s.gate_up = take(pairs * 2 * ff * 2);
  s.a = take(pairs * f8_ld(ff));
  s.a_scale = take(pairs * f8_blocks(ff) * 4);
  s.y = take(pairs * width * 2);
  s.bytes = at;
  return s;
}

int check_pairs(const char* what, int64_t rows, int64_t top, int64_t experts) {
  B200_CHECK_ARG(rows >= 1 && top >= 1 && experts >= 1 && experts <= kMaxExperts && rows < 1 << 24 && top <= experts && rows * top < 1 << 24,
                 "%s: %lld rows with %lld of %lld experts out of range", what, (long long)rows, (long long)top, (long long)experts);
  return B200_OK;
}

}  // namespace

static int order_bytes(int64_t experts, int64_t kept) { return (int)(kOrderWarps * (experts | 1) + 2 * experts + std::min<int64_t>(kept, kOrderKept)) * 4; }

int launch_expert_order(int32_t* starts, int32_t* source, int32_t* place, const int32_t* chosen, int64_t rows, int64_t top, int64_t experts, cudaStream_t st) {
  const int64_t pairs = rows * top, ctas = pairs > 2 * kOrderThreads ? kOrderCtas : 1;
  const int64_t run = (pairs + ctas * kOrderThreads - 1) / (ctas * kOrderThreads) * 32;
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(expert_order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, order_bytes(kMaxExperts, kOrderKept)); }));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kOrderThreads);
  cfg.dynamicSmemBytes = (size_t)order_bytes(experts, run * kOrderWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = op_pdl(st) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  B200_CUDA(cudaLaunchKernelEx(&cfg, expert_order_kernel, starts, source, place, chosen, (int)pairs, (int)top, (int)experts, (int)run));
  return B200_OK;
}

int launch_expert_combine(void* out, const void* y, const int32_t* place, const float* weights, int64_t rows, int64_t top, int64_t n, cudaStream_t st) {
  const bool wide = n % 8 == 0 && aligned16(out, y);
  const int64_t threads = rows * (wide ? n / 8 : n);
  B200_CUDA(launch_pdl(wide ? expert_combine_kernel<true> : expert_combine_kernel<false>, dim3((unsigned)std::min<int64_t>((threads + 255) / 256, 148 * 32)), dim3(256),
                       0, st, op_pdl(st), (__nv_bfloat16*)out, (const __nv_bfloat16*)y, place, weights, rows, (int)top, (int)n));
  return B200_OK;
}

}  // namespace b200

extern "C" {

int b200_expert_order(int32_t* starts, int32_t* source, int32_t* place, const int32_t* chosen, int64_t rows, int64_t top, int64_t experts, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_pairs("expert_order", rows, top, experts)) != B200_OK) return rc;
  B200_CHECK_ARG(starts && source && place && chosen, "expert_order: null pointer");
  return launch_expert_order(starts, source, place, chosen, rows, top, experts, (cudaStream_t)stream);
}

int b200_expert_combine_bf16(void* out, const void* y, const int32_t* place, const float* weights, int64_t rows, int64_t top, int64_t n, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_pairs("expert_combine", rows, top, kMaxExperts)) != B200_OK) return rc;
  B200_CHECK_ARG(out && y && place && weights && n >= 1 && n <= 1 << 24, "expert_combine: rows of %lld out of range, or a null pointer", (long long)n);
  return launch_expert_combine(out, y, place, weights, rows, top, n, (cudaStream_t)stream);
}

int64_t b200_experts_f8_workspace_bytes(int64_t rows, int64_t top, int64_t experts, int64_t width, int64_t ff) {
  using namespace b200;
  if (rows < 1 || top < 1 || experts < 1 || width < 1 || ff < 1 || rows >= 1 << 24 || experts > kMaxExperts || top > experts || width > 1 << 20 || ff > 1 << 20) return -1;
  return experts_space(rows, top, experts, width, ff).bytes;
}

int b200_experts_f8_bf16(void* out, const void* x, const int32_t* chosen, const float* weights, const b200_f8_weight* w_in, const b200_f8_weight* w_out, int64_t rows,
                         int64_t top, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(out && x && chosen && weights && w_in && w_out && w_in->q && w_in->scale && w_out->q && w_out->scale, "experts_f8: null pointer");
  const int64_t experts = w_in->experts, width = w_in->k, ff = w_out->k;
  if ((rc = check_pairs("experts_f8", rows, top, experts)) != B200_OK) return rc;
  B200_CHECK_ARG(w_out->experts == experts && w_in->n == 2 * ff && w_out->n == width && width >= 1 && ff >= 1 && width <= 1 << 20 && ff <= 1 << 19 &&
                     experts * std::max(2 * ff, width) < 1ll << 31,
                 "experts_f8: %d matrices [%d, %d] and %d [%d, %d]", (int)w_in->experts, (int)w_in->n, (int)w_in->k, (int)w_out->experts, (int)w_out->n, (int)w_out->k);
  B200_CHECK_ARG(workspace && aligned16(workspace, w_in->q, w_out->q), "experts_f8: workspace and weights must be 16-byte aligned");
  const ExpertsSpace s = experts_space(rows, top, experts, width, ff);
  const int64_t pairs = rows * top;
  uint8_t* const ws = (uint8_t*)workspace;
  const cudaStream_t st = (cudaStream_t)stream;
  auto ints = [&](int64_t at) { return (int32_t*)(ws + at); };
  auto floats = [&](int64_t at) { return (float*)(ws + at); };
  if ((rc = launch_expert_order(ints(s.starts), ints(s.source), ints(s.place), chosen, rows, top, experts, st)) != B200_OK) return rc;
  if ((rc = launch_f8_rows_to(ws + s.q, floats(s.scale), x, ints(s.place), rows, top, pairs, width, st)) != B200_OK) return rc;
  if ((rc = launch_group_product({ws + s.gate_up, ws + s.q, floats(s.scale), w_in->q, w_in->scale, ints(s.starts), nullptr, pairs, experts, 2 * ff, width, true}, st)) != B200_OK)
    return rc;
  if ((rc = launch_silu_mul_f8(ws + s.a, floats(s.a_scale), ws + s.gate_up, pairs, ff, st)) != B200_OK) return rc;
  if ((rc = launch_group_product({ws + s.y, ws + s.a, floats(s.a_scale), w_out->q, w_out->scale, ints(s.starts), nullptr, pairs, experts, width, ff, true}, st)) != B200_OK)
    return rc;
  return launch_expert_combine(out, ws + s.y, ints(s.place), weights, rows, top, width, st);
}

}  // extern "C"
