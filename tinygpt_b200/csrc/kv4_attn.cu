// kv4_attn.cu — attention over the paged cache of 4-bit keys and values (kv4.cuh has the layout).
//
// Of a sequence's query rows, those of the query heads that share a key/value head are columns: column = token of the call · group + head of the
// group.  A warp holds 8·NT of them and goes over 16 tokens of the cache at a time:
//   scores   Sᵀ = K·qᵀ   values of the cache as exact bf16 integers, a group's sum scaled in fp32, + middle·Σq of the group
//   softmax  over the tokens, in fp32, with a running maximum and sum per column
//   output   Oᵀ += Vᵀ·P  a value's scale goes into its weight (rounded to bf16), Σ weight·middle is kept in fp32 beside the products
// Everything between memory and the products is in registers; a transposing move turns the weights of a score tile into the operand that Vᵀ meets.
//
// Work is cut evenly over the CTAs whatever the sequences' lengths: (sequence, column block, head, page) in this order is one line of units,
// of which every CTA takes an equal piece.  A CTA that holds all of an item's pages writes its rows; parts of an item go to the workspace and a
// second kernel joins them in their order.
#include "kv4.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;

struct Kv4Attn {
  b200_kv4_cache cache;
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  int64_t ld_q;
  const int32_t *seqs, *starts, *pos;
  float* parts;
  int layer, q_heads, group, n, rows, window;
  float scale_log2;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t o;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
  return o;
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A sequence of the call: its rows, the tokens they may see, its work.
struct Kv4Seq {
  int row0, count, pos, slot, last, page0, pages, blocks;   // tokens below `last`; pages page0 … page0 + pages − 1 (one at least)
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn& p, int i, int columns) {
  Kv4Seq s;
  s.row0 = min(max(p.starts[i], 0), p.rows);
  s.count = max(min(p.starts[i + 1], p.rows) - s.row0, 0);
  s.pos = min(p.pos[i], 1 << 30);
  s.slot = p.seqs[i];
  s.blocks = (int)(((int64_t)s.count * p.group + columns - 1) / columns);
  s.last = 0;
  s.page0 = 0;
  if (s.pos >= 0 && s.slot >= 0 && s.slot < p.cache.n_seqs)
    s.last = (int)min(min((int64_t)p.cache.length[s.slot], (int64_t)s.pos + s.count), min((int64_t)p.cache.max_pages * kPage, (int64_t)(1 << 30)));
  s.last = max(s.last, 0);
  if (p.window > 0 && s.pos >= p.window) s.page0 = min((s.pos - p.window + 1) / kPage, s.last / kPage);
  s.pages = max((s.last + kPage - 1) / kPage - s.page0, 1);
  return s;
}
// ends[i]: units of the sequences up to i; the longest item's pages come back.  All threads of the CTA.
__device__ int kv4_plan(const Kv4Attn& p, int columns, long long* ends) {
  __shared__ long long carry[kWarps];
  __shared__ int longest[kWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int kEach = kKvMaxSeqs / kThreads;
  long long mine[kEach], sum = 0;
  int most = 1;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x * kEach + e;
    if (i < p.n) {
      const Kv4Seq s = kv4_seq(p, i, columns);
      sum += (long long)s.blocks * p.cache.kv_heads * s.pages;
      if (s.blocks > 0) most = max(most, s.pages);
    }
    mine[e] = sum;
  }
  long long before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (lane == 31) {
    carry[warp] = before;
    longest[warp] = most;
  }
  __syncthreads();
  before -= sum;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += carry[w];
    most = max(most, longest[w]);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (threadIdx.x * kEach + e < p.n) ends[threadIdx.x * kEach + e] = before + mine[e];
  __syncthreads();
  return most;
}
// units of a CTA: an equal share, but at least a page to each warp where items have as many
__device__ __forceinline__ long long kv4_share(long long units, int ctas, int longest) { return max((units + ctas - 1) / ctas, (long long)min(longest, kWarps)); }
__device__ __forceinline__ int kv4_find(const long long* ends, int n, long long unit) {   // the first i with ends[i] > unit
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (ends[mid] > unit) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
__device__ __forceinline__ float* kv4_part(const Kv4Attn& p, int cta, int which, int columns) {
  return p.parts + ((int64_t)cta * 2 + which) * columns * (p.cache.dim + 2);
}

template <int NG, int NT>
struct Shape {
  static constexpr int kTile = kv4_tile_bytes(NG);
  static constexpr int kStageTiles = NG <= 2 ? 4 : 2;
  static constexpr int kStage = kStageTiles * kTile;
  static constexpr bool kQInRegs = NG * NT <= 4;
  static constexpr int kQBytes = kQInRegs ? 0 : NT * NG * 2 * 512;
  static constexpr int kSmem = kWarps * 2 * kStage + kQBytes + kKvMaxSeqs * 8;
  static_assert(8 * NT * (NG * 64 + 2) * 4 <= 2 * kStage, "a warp's output fits its ring");
};

template <int NG, int NT>
__global__ void __launch_bounds__(kThreads, 1) kv4_attn_kernel(const Kv4Attn p) {
  using S = Shape<NG, NT>;
  constexpr int kCols = 8 * NT, kDim = NG * 64, kPer = 4 / S::kStageTiles;   // stages of a page
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  uint8_t* const ring = smem + warp * 2 * S::kStage;
  uint4* const q_smem = reinterpret_cast<uint4*>(smem + kWarps * 2 * S::kStage);
  long long* const ends = reinterpret_cast<long long*>(smem + kWarps * 2 * S::kStage + S::kQBytes);
  pdl_wait();
  pdl_trigger();

  // rows of no sequence
  {
    const int head = min(max(p.starts[0], 0), p.rows), tail = min(max(p.starts[p.n], head), p.rows), width = p.q_heads * kDim;
    for (int64_t row = blockIdx.x; row < head + p.rows - tail; row += gridDim.x)
      for (int d = threadIdx.x; d < width; d += kThreads) p.out[(row < head ? row : row - head + tail) * width + d] = f_to_bf16(0.f);
  }
  const int longest = kv4_plan(p, kCols, ends);
  const long long units = ends[p.n - 1], share = kv4_share(units, gridDim.x, longest);
  long long unit = share * blockIdx.x;
  const long long stop = min(unit + share, units);
  int i = unit < stop ? kv4_find(ends, p.n, unit) : 0;
  while (unit < stop) {
    while (ends[i] <= unit) ++i;
    const Kv4Seq s = kv4_seq(p, i, kCols);
    const long long in_seq = unit - (i > 0 ? ends[i - 1] : 0);
    const int item = (int)(in_seq / s.pages), first = (int)(in_seq % s.pages), head = item % p.cache.kv_heads, block = item / p.cache.kv_heads;
    const int many = (int)min((long long)(s.pages - first), stop - unit);
    unit += many;

    // the block's queries, as the B operands of K·qᵀ, and their sums over each group
    const int col0 = block * kCols, n_cols = s.count * p.group;
    uint4 qf[S::kQInRegs ? NT : 1][NG][2];
    float qsum[NG][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = col0 + t * 8 + r;
      const __nv_bfloat16* src = p.q + (int64_t)(s.row0 + col / p.group) * p.ld_q + (int64_t)(head * p.group + col % p.group) * kDim + 8 * c;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = col < n_cols ? *reinterpret_cast<const uint4*>(src + g * 64 + h * 32) : make_uint4(0, 0, 0, 0);
          if constexpr (S::kQInRegs) qf[t][g][h] = v;
          else if (warp == 0) q_smem[((t * NG + g) * 2 + h) * 32 + lane] = v;
          mma16816(sum, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.x, v.y);
          mma16816(sum, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.z, v.w);
        }
        qsum[g][t][0] = sum[0];
        qsum[g][t][1] = sum[1];
      }
    }
    if constexpr (!S::kQInRegs) __syncthreads();
    int at[NT][2];   // positions of this lane's columns (2c, 2c + 1); −1: no column
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = col0 + t * 8 + 2 * c + e;
        at[t][e] = col < n_cols ? s.pos + col / p.group : -1;
      }
    const int at_low = s.pos + col0 / p.group, at_high = s.pos + (min(col0 + kCols, n_cols) - 1) / p.group;

    float o[NG * 4][NT][4] = {};
    float top[NT][2], sum[NT][2] = {}, mid[NG][NT][2] = {};
#pragma unroll
    for (int t = 0; t < NT; ++t) top[t][0] = top[t][1] = -INFINITY;

    const int32_t* table = p.cache.table + (int64_t)max(s.slot, 0) * p.cache.max_pages + s.page0 + first;
    const int n_stages = s.last > 0 ? many * kPer : 0;
    auto page_of = [&](int u) {
      if (u >= n_stages) return -1;
      const int page = table[u / kPer];
      return page < p.cache.n_pages ? page : -1;
    };
    auto fetch = [&](int u, int page, int slot) {
      if (page >= 0) {
        const uint8_t* src = kv4_head(p.cache, p.layer, page, head) + u % kPer * S::kStage;
#pragma unroll
        for (int b = 0; b < S::kStage; b += 512)
          if (S::kStage % 512 == 0 || b + lane * 16 < S::kStage) cp_async16(ring + slot * S::kStage + b + lane * 16, src + b + lane * 16);
      }
      cp_async_commit();
    };
    int page = page_of(warp), next = page_of(warp + kWarps), slot = 0;
    fetch(warp, page, 0);
    for (int u = warp; u < n_stages; u += kWarps, slot ^= 1) {
      fetch(u + kWarps, next, slot ^ 1);
      const int now = page;
      page = next;
      next = page_of(u + 2 * kWarps);
      cp_async_wait<1>();
      __syncwarp();
      if (now >= 0) {
        const uint8_t* stage = ring + slot * S::kStage;
        const int key0 = (s.page0 + first) * kPage + u * (S::kStageTiles * kKvTile);
        const bool whole = key0 + S::kStageTiles * kKvTile <= min(s.last, at_low + 1) && (p.window == 0 || at_high - key0 < p.window);
        float sc[S::kStageTiles][NT][4];
#pragma unroll
        for (int k = 0; k < S::kStageTiles; ++k) {
          const uint8_t* tile = stage + k * S::kTile;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[k][t][e] = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint4 w = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
            const uint2 small = *reinterpret_cast<const uint2*>(tile + NG * 512 + g * 64 + r * 8);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            float acc[NT][4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a[4];
              nibbles_bf16(words[j], a);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                uint4 b;
                if constexpr (S::kQInRegs) b = qf[t][g][j / 2];
                else b = q_smem[((t * NG + g) * 2 + j / 2) * 32 + lane];
                mma16816(acc[t], a[0], a[2], a[1], a[3], j % 2 ? b.z : b.x, j % 2 ? b.w : b.y);
              }
            }
            const float s0 = bf16_lo(small.x), m0 = bf16_hi(small.x), s1 = bf16_lo(small.y), m1 = bf16_hi(small.y);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              sc[k][t][0] = fmaf(s0, acc[t][0], fmaf(m0, qsum[g][t][0], sc[k][t][0]));
              sc[k][t][1] = fmaf(s0, acc[t][1], fmaf(m0, qsum[g][t][1], sc[k][t][1]));
              sc[k][t][2] = fmaf(s1, acc[t][2], fmaf(m1, qsum[g][t][0], sc[k][t][2]));
              sc[k][t][3] = fmaf(s1, acc[t][3], fmaf(m1, qsum[g][t][1], sc[k][t][3]));
            }
          }
        }
        if (!whole) {
#pragma unroll
          for (int k = 0; k < S::kStageTiles; ++k)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = key0 + k * kKvTile + r + 8 * (e / 2), from = at[t][e % 2];
                const bool seen = key <= from && key < s.last && (p.window == 0 || from - key < p.window);
                if (!seen) sc[k][t][e] = -INFINITY;
              }
        }
        float now_top[NT][2], shift[NT][2];
        bool moved = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < S::kStageTiles; ++k) m = fmaxf(m, fmaxf(sc[k][t][e], sc[k][t][e + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            m = fmaxf(top[t][e], m * p.scale_log2);
            now_top[t][e] = m;
            shift[t][e] = m == -INFINITY ? 0.f : m;
            moved |= m != top[t][e];
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = exp2_fast(top[t][e] - shift[t][e]);   // 0 where there was none
              top[t][e] = now_top[t][e];
              sum[t][e] *= f;
#pragma unroll
              for (int g = 0; g < NG; ++g) mid[g][t][e] *= f;
#pragma unroll
              for (int d = 0; d < NG * 4; ++d) {
                o[d][t][e] *= f;
                o[d][t][e + 2] *= f;
              }
            }
        }
#pragma unroll
        for (int k = 0; k < S::kStageTiles; ++k) {
          const uint8_t* tile = stage + k * S::kTile + NG * (512 + 64);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = exp2_fast(fmaf(sc[k][t][e], p.scale_log2, -shift[t][e % 2]));
              sum[t][e % 2] += v;
              sc[k][t][e] = v;
            }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint2 small = *reinterpret_cast<const uint2*>(tile + NG * 512 + g * 64 + r * 8);
            const float s0 = bf16_lo(small.x), m0 = bf16_hi(small.x), s1 = bf16_lo(small.y), m1 = bf16_hi(small.y);
            uint32_t b[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float w[4] = {sc[k][t][0] * s0, sc[k][t][1] * s0, sc[k][t][2] * s1, sc[k][t][3] * s1};
              float y[4] = {sc[k][t][0] * m0, sc[k][t][1] * m0, sc[k][t][2] * m1, sc[k][t][3] * m1};
              if (!whole) {   // what is not seen may hold anything
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (sc[k][t][e] == 0.f) w[e] = y[e] = 0.f;
              }
              mid[g][t][0] += y[0] + y[2];
              mid[g][t][1] += y[1] + y[3];
              b[t][0] = transpose8x8(pack2(w[0], w[1]));
              b[t][1] = transpose8x8(pack2(w[2], w[3]));
            }
            const uint4 v = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a[4];
              nibbles_bf16(words[j], a);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma16816(o[g * 4 + j][t], a[0], a[1], a[2], a[3], b[t][0], b[t][1]);
            }
          }
        }
      }
      __syncwarp();   // the stage is free
    }
    cp_async_wait<0>();
    __syncwarp();

    // the warps' parts meet in shared memory: [column][dim], then the maxima and the sums
    float* const own = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[t][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const int col = t * 8 + 2 * c + e;
        if (r == 0) {
          own[kCols * kDim + col] = top[t][e];
          own[kCols * kDim + kCols + col] = l;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float y = mid[g][t][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) y += __shfl_xor_sync(0xffffffffu, y, x);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            own[col * kDim + g * 64 + j * 16 + r] = o[g * 4 + j][t][e] + y;
            own[col * kDim + g * 64 + j * 16 + r + 8] = o[g * 4 + j][t][e + 2] + y;
          }
        }
      }
    __syncthreads();
    const bool all = many == s.pages;
    float* const part = all ? nullptr : kv4_part(p, blockIdx.x, first == 0, kCols);
    for (int x = threadIdx.x; x < kCols * kDim; x += kThreads) {
      const int col = x / kDim, d = x % kDim;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, reinterpret_cast<const float*>(smem + w * 2 * S::kStage)[kCols * kDim + col]);
      float l = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* from = reinterpret_cast<const float*>(smem + w * 2 * S::kStage);
        const float lw = from[kCols * kDim + kCols + col];
        if (lw != 0.f) {   // what has seen a token (one that is no number too)
          const float f = exp2_fast(from[kCols * kDim + col] - m);
          l = fmaf(f, lw, l);
          v = fmaf(f, from[x], v);
        }
      }
      if (all) {
        if (col0 + col < n_cols)
          p.out[((int64_t)(s.row0 + (col0 + col) / p.group) * p.q_heads + head * p.group + (col0 + col) % p.group) * kDim + d] =
              f_to_bf16(l == 0.f ? 0.f : v / l);
      } else {
        part[x] = v;
        if (d == 0) {
          part[kCols * kDim + col] = m;
          part[kCols * kDim + kCols + col] = l;
        }
      }
    }
    __syncthreads();
  }
}

// One CTA (of a row of the grid) for every border between two CTAs of the kernel above: it joins the item that lies across the border, if no border before
// lies in it too.  The item's parts are taken in their order.
__global__ void __launch_bounds__(kThreads) kv4_join_kernel(const Kv4Attn p, int columns, int ctas) {
  __shared__ long long ends[kKvMaxSeqs];
  pdl_wait();
  pdl_trigger();
  const int longest = kv4_plan(p, columns, ends);
  const long long units = ends[p.n - 1], share = kv4_share(units, ctas, longest), border = share * (blockIdx.x + 1);
  if (border >= units) return;
  const int i = kv4_find(ends, p.n, border);
  const Kv4Seq s = kv4_seq(p, i, columns);
  const long long base = i > 0 ? ends[i - 1] : 0;
  const int item = (int)((border - base) / s.pages);
  const long long begin = base + (long long)item * s.pages, end = begin + s.pages;
  if (begin == border || begin / share != blockIdx.x) return;
  const int head = item % p.cache.kv_heads, col0 = item / p.cache.kv_heads * columns, n_cols = s.count * p.group, dim = p.cache.dim;
  const int from = (int)(begin / share), to = (int)((end - 1) / share);
  for (int x = blockIdx.y * kThreads + threadIdx.x; x < columns * dim; x += gridDim.y * kThreads) {
    const int col = x / dim, d = x % dim;
    if (col0 + col >= n_cols) break;
    float m = -INFINITY, l = 0.f, v = 0.f;
    for (int c = from; c <= to; ++c) m = fmaxf(m, kv4_part(p, c, c == from, columns)[columns * dim + col]);
    for (int c = from; c <= to; ++c) {
      const float* part = kv4_part(p, c, c == from, columns);
      const float lw = part[columns * dim + columns + col];
      if (lw == 0.f) continue;
      const float f = exp2_fast(part[columns * dim + col] - m);
      l = fmaf(f, lw, l);
      v = fmaf(f, part[x], v);
    }
    p.out[((int64_t)(s.row0 + (col0 + col) / p.group) * p.q_heads + head * p.group + (col0 + col) % p.group) * dim + d] = f_to_bf16(l == 0.f ? 0.f : v / l);
  }
}

// Column tiles of a block: what an average sequence brings.
int column_tiles(int64_t group, int64_t n, int64_t rows) { return group * ((rows + n - 1) / n) <= 8 ? 1 : 2; }
int grid_of() { return 148; }

template <int NG, int NT>
int launch(const Kv4Attn& p, cudaStream_t st) {
  using S = Shape<NG, NT>;
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(kv4_attn_kernel<NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); }));
  const bool pdl = op_pdl(st);
  B200_CUDA(launch_pdl(kv4_attn_kernel<NG, NT>, dim3(grid_of()), dim3(kThreads), S::kSmem, st, pdl, p));
  B200_CUDA(launch_pdl(kv4_join_kernel, dim3(grid_of() - 1, 8 * NT * NG * 64 / kThreads), dim3(kThreads), 0, st, pdl, p, 8 * NT, grid_of()));
  return B200_OK;
}

}  // namespace

}  // namespace b200

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(const b200_kv4_cache* cache, int64_t q_heads, int64_t n, int64_t rows) {
  using namespace b200;
  if (cache == nullptr || cache->kv_heads < 1 || q_heads < 1 || q_heads % cache->kv_heads != 0 || n < 1 || rows < 1) return -1;
  const int tiles = column_tiles(q_heads / cache->kv_heads, n, rows);
  return (int64_t)grid_of() * 2 * 8 * tiles * (cache->dim + 2) * 4;
}

int b200_kv4_attention(void* out, const void* q, int64_t ld_q, const b200_kv4_cache* cache, int64_t layer, int64_t q_heads, const int32_t* seqs,
                       const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows, float scale, int64_t window, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_attention")) != B200_OK) return rc;
  B200_CHECK_ARG(out && q && workspace, "kv4_attention: null pointer");
  B200_CHECK_ARG(q_heads >= 1 && q_heads <= 1 << 16 && q_heads % cache->kv_heads == 0, "kv4_attention: %lld query heads over %d", (long long)q_heads,
                 cache->kv_heads);
  B200_CHECK_ARG(aligned16(q, workspace, out) && ld_q % 8 == 0 && ld_q >= q_heads * cache->dim, "kv4_attention: q's rows must be 16-byte aligned and apart");
  B200_CHECK_ARG(scale > 0.f && scale < 1e30f && window >= 0, "kv4_attention: scale %g, window %lld", (double)scale, (long long)window);
  B200_CHECK_ARG(rows * q_heads < 1ll << 31, "kv4_attention: %lld rows of %lld heads", (long long)rows, (long long)q_heads);
  Kv4Attn p{};
  p.cache = *cache;
  p.out = (__nv_bfloat16*)out;
  p.q = (const __nv_bfloat16*)q;
  p.ld_q = ld_q;
  p.seqs = seqs;
  p.starts = starts;
  p.pos = pos;
  p.parts = (float*)workspace;
  p.layer = (int)layer;
  p.q_heads = (int)q_heads;
  p.group = (int)(q_heads / cache->kv_heads);
  p.n = (int)n;
  p.rows = (int)rows;
  p.window = (int)std::min<int64_t>(window, INT32_MAX);
  p.scale_log2 = scale * 1.44269504f;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool two = column_tiles(p.group, n, rows) == 2;
  switch (cache->dim / kKvGroup) {
    case 1: return two ? launch<1, 2>(p, st) : launch<1, 1>(p, st);
    case 2: return two ? launch<2, 2>(p, st) : launch<2, 1>(p, st);
    case 3: return two ? launch<3, 2>(p, st) : launch<3, 1>(p, st);
    default: return two ? launch<4, 2>(p, st) : launch<4, 1>(p, st);
  }
}

}  // extern "C"
