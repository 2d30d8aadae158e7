// kv4_attn.cu — attention over the paged cache of 4-bit keys and values (kv4.cuh has the layout).
//
// Of a sequence's query rows, those of the query heads that share a key/value head are columns: column = token of the call · group + head of the
// group.  A warp holds 8·NT of them and goes over 16 tokens of the cache at a time:
//   scores   Sᵀ = K·qᵀ   values of the cache as exact bf16 integers, a group's sum scaled in fp32, + middle·Σq of the group
//   softmax  over the tokens, in fp32, with a running maximum and sum per column
//   output   Oᵀ += Vᵀ·P  a value's scale goes into its weight (rounded to bf16), Σ weight·middle is kept in fp32 beside the products
// Everything between memory and the products is in registers; a transposing move turns the weights of a score tile into the operand that Vᵀ meets.
//
// Work is cut evenly over the warps of the GPU whatever the sequences' lengths: the items (sequence, column block, head) form one line, each as
// long as its steps of 32 tokens and kAhead more for what an item costs before its first token, and every warp takes an equal piece of the line.  A warp
// that holds all of an item writes its rows; parts go to the workspace (one for a CTA whose warps are all inside an item) and a second
// kernel joins them in their order.
#include "kv4.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {

namespace {

constexpr int kStep = 32, kAhead = 2;
constexpr float kSlack = 8.f;
constexpr int kGrid = 148;

// Division by a number that the host knows (Granlund and Montgomery): a multiplication and two shifts
struct Divisor {
  uint32_t d, m;
  int s1, s2;
  Divisor(uint32_t d_ = 1) : d(d_) {
    int s = 0;
    while ((1ull << s) < d) ++s;
    m = (uint32_t)((((1ull << s) - d) << 32) / d + 1);
    s1 = std::min(s, 1);
    s2 = std::max(s - 1, 0);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int of(int n) const {
    const uint32_t t = __umulhi(m, (uint32_t)n);
    return (int)((t + (((uint32_t)n - t) >> s1)) >> s2);
  }
#endif
};

struct Kv4Attn {
  b200_kv4_cache cache;
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  int64_t ld_q;
  const int32_t *seqs, *starts, *pos;
  float* parts;
  struct Kv4Split* splits;   // of every warp
  Divisor group, kv_heads;   // query heads of a key/value head
  int layer, q_heads, n, rows, window;
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
__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long b = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += b;
  }
  return v;
}

// A sequence of the call: its rows, the tokens they may see, its items.
struct Kv4Seq {
  int row0, count, pos, slot, last, step0, steps, blocks;   // tokens below `last`; steps step0 … step0 + steps − 1 (one at least)
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn& p, int i, int columns) {
  Kv4Seq s;
  s.row0 = min(max(p.starts[i], 0), p.rows);
  s.count = max(min(p.starts[i + 1], p.rows) - s.row0, 0);
  s.pos = min(p.pos[i], 1 << 30);
  s.slot = p.seqs[i];
  s.blocks = (int)(((int64_t)s.count * p.group.d + columns - 1) / columns);
  s.last = 0;
  s.step0 = 0;
  if (s.pos >= 0 && s.slot >= 0 && s.slot < p.cache.n_seqs)
    s.last = (int)min(min((int64_t)p.cache.length[s.slot], (int64_t)s.pos + s.count), min((int64_t)p.cache.max_pages * kPage, (int64_t)(1 << 30)));
  s.last = max(s.last, 0);
  if (p.window > 0 && s.pos >= p.window) s.step0 = min((s.pos - p.window + 1) / kStep, s.last / kStep);
  s.steps = max((s.last + kStep - 1) / kStep - s.step0, 1);
  return s;
}
__device__ __forceinline__ long long kv4_line(const Kv4Attn& p, const Kv4Seq& s) { return (long long)s.blocks * p.cache.kv_heads * (s.steps + kAhead); }
__device__ __forceinline__ Kv4Seq kv4_from(const Kv4Seq& s, int lane) {   // another lane's
  Kv4Seq o;
  o.row0 = __shfl_sync(0xffffffffu, s.row0, lane);
  o.count = __shfl_sync(0xffffffffu, s.count, lane);
  o.pos = __shfl_sync(0xffffffffu, s.pos, lane);
  o.slot = __shfl_sync(0xffffffffu, s.slot, lane);
  o.last = __shfl_sync(0xffffffffu, s.last, lane);
  o.step0 = __shfl_sync(0xffffffffu, s.step0, lane);
  o.steps = __shfl_sync(0xffffffffu, s.steps, lane);
  o.blocks = __shfl_sync(0xffffffffu, s.blocks, lane);
  return o;
}
// ends[i]: the line up to the end of sequence i; all of it comes back.  The call has checked that it is below 2^31 for starts that do not fall; for others it may not
// be, and nothing is done.  All threads of a CTA of THREADS.
__device__ __forceinline__ int kv4_whole(long long line) { return line <= INT32_MAX ? (int)line : 0; }
template <int THREADS>
__device__ int kv4_plan(const Kv4Attn& p, int columns, int* ends) {
  __shared__ long long carry[THREADS / 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, each = (p.n + THREADS - 1) / THREADS, first = threadIdx.x * each;
  long long sum = 0;
  for (int i = first; i < min(first + each, p.n); ++i) sum += kv4_line(p, kv4_seq(p, i, columns));
  const long long upto = warp_scan(sum, lane);
  if (lane == 31) carry[warp] = upto;
  __syncthreads();
  long long before = upto - sum, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += carry[w];
    all += carry[w];
  }
  for (int i = first; i < min(first + each, p.n); ++i) ends[i] = (int)(before += kv4_line(p, kv4_seq(p, i, columns)));
  __syncthreads();
  return kv4_whole(all);
}
__device__ __forceinline__ int kv4_find(const int* ends, int n, int at) {   // the first i with ends[i] > at
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (ends[mid] > at) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// How the line is cut: `warps` pieces, `each` CTA having so many of them; piece w starts at about line·w / warps (as fp32 has it: the same for everyone).  A piece is no shorter than a step and what
// comes before it, and short lines are spread over the CTAs first.
struct Cut {
  int line, warps, each, whole, rest;   // line = whole·warps + rest
  float inverse;
  __device__ Cut(int line_, int most) : line(line_) {
    warps = min(max(line / (kAhead + 1), 1), kGrid * most);
    each = (warps + kGrid - 1) / kGrid;
    inverse = __frcp_rn((float)warps);
    whole = line / warps;
    rest = line - whole * warps;
  }
  __device__ __forceinline__ int start(int w) const { return w < warps ? w * whole + (int)((float)(w * rest) * inverse) : line; }
};
// a warp's parts: of an item that came before it (0) and of one that goes on behind it (1).  [column][dim], maxima, sums
__device__ __forceinline__ float* kv4_part(const Kv4Attn& p, int64_t warp, int which, int columns) {
  return p.parts + (warp * 2 + which) * columns * (p.cache.dim + 2);
}
// An item that its first warp does not finish, for the kernel that joins the parts: the warps that hold it, of those the ones that left one part for their CTA.
struct Kv4Split {
  int from, to, in0, in1;   // warps from … to; CTAs in0 … in1 − 1 (none: in0 >= in1)
  int row0, col0, n_cols, head, each;   // from < 0: none
};

template <int NG, int NT>
struct Shape {
  static constexpr int kTile = kv4_tile_bytes(NG);
  static constexpr int kTiles = kStep / kKvTile;                // of a step
  static constexpr int kStage = kTiles * kTile;
  static constexpr int kWarps = 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr bool kQInRegs = NG * NT <= 4;
  static constexpr int kQBytes = kQInRegs ? 0 : NT * NG * 2 * 512;
  static constexpr int kRoom = 232448 - 1024 - kKvMaxSeqs * 4;
  static constexpr int kStages = kWarps * (3 * kStage + kQBytes) <= kRoom ? 3 : 2;
  static constexpr int kRing = kStages * kStage > 8 * NT * (NG * 64 + 6) * 4 ? kStages * kStage : (8 * NT * (NG * 64 + 6) * 4 + 15) / 16 * 16;
  static constexpr int kOwn = kRing + kQBytes;                  // shared memory of a warp
  static constexpr int kSmem = kWarps * kOwn + kKvMaxSeqs * 4;
  static_assert(kWarps * kOwn <= kRoom, "shared memory of an SM");
};

template <int NG, int NT>
__global__ void __launch_bounds__(Shape<NG, NT>::kThreads, 1) kv4_attn_kernel(const Kv4Attn p) {
  using S = Shape<NG, NT>;
  constexpr int kCols = 8 * NT, kDim = NG * 64;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  uint8_t* const ring = smem + warp * S::kOwn;
  uint4* const q_smem = reinterpret_cast<uint4*>(ring + S::kRing);
  int* const ends = reinterpret_cast<int*>(smem + S::kWarps * S::kOwn);
  pdl_wait();
  pdl_trigger();

  // rows of no sequence
  {
    const int head = min(max(p.starts[0], 0), p.rows), tail = min(max(p.starts[p.n], head), p.rows), width = p.q_heads * kDim;
    for (int row = blockIdx.x; row < head + p.rows - tail; row += kGrid)
      for (int d = threadIdx.x; d < width; d += S::kThreads) p.out[(int64_t)(row < head ? row : row - head + tail) * width + d] = f_to_bf16(0.f);
  }
  // Up to 32 sequences: every warp has them all in its lanes, and nobody waits for anybody.
  const bool few = p.n <= 32;
  Kv4Seq mine{};
  int mine_end = 0, line;
  if (few) {
    if (lane < p.n) mine = kv4_seq(p, lane, kCols);
    const long long end = warp_scan(lane < p.n ? kv4_line(p, mine) : 0, lane);
    mine_end = (int)end;
    line = kv4_whole(__shfl_sync(0xffffffffu, end, 31));
  } else {
    line = kv4_plan<S::kThreads>(p, kCols, ends);
  }
  const Cut cut(line, S::kWarps);
  const int me = blockIdx.x * cut.each + warp;
  const int64_t own = (int64_t)blockIdx.x * S::kWarps + warp;   // of the workspace's places
  int at_line = cut.start(me);
  const int stop = warp < cut.each ? cut.start(me + 1) : at_line;
  if (lane == 0) p.splits[own].from = -1;
  int i = !few && at_line < stop ? kv4_find(ends, p.n, at_line) : 0;
  while (at_line < stop) {
    int base = 0;
    Kv4Seq s;
    if (few) {
      i = __popc(__ballot_sync(0xffffffffu, mine_end <= at_line));
      if (i > 0) base = __shfl_sync(0xffffffffu, mine_end, i - 1);
      s = kv4_from(mine, i);
    } else {
      while (ends[i] <= at_line) ++i;
      if (i > 0) base = ends[i - 1];
      s = kv4_seq(p, i, kCols);
    }
    const int length = s.steps + kAhead;
    int item = (int)((float)(at_line - base) * __frcp_rn((float)length));   // (a division costs more than these)
    while (item * length > at_line - base) --item;
    while ((item + 1) * length <= at_line - base) ++item;
    const int block = p.kv_heads.of(item), head = item - block * p.kv_heads.d;
    const int begin = base + item * length + kAhead, end = begin + s.steps;   // of its steps
    const int first = max(at_line - begin, 0), many = min(stop, end) - begin - first;
    at_line = min(stop, end);
    if (many <= 0) continue;

    const int col0 = block * kCols, n_cols = s.count * p.group.d;
    uint4 raw[NT][NG][2];   // the block's queries
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = col0 + t * 8 + r;
      const int token = p.group.of(col);
      const __nv_bfloat16* src = p.q + (int64_t)(s.row0 + token) * p.ld_q + (int64_t)(head * p.group.d + col - token * p.group.d) * kDim + 8 * c;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) raw[t][g][h] = col < n_cols ? *reinterpret_cast<const uint4*>(src + g * 64 + h * 32) : make_uint4(0, 0, 0, 0);
    }
    int at[NT][2];   // positions of this lane's columns (2c, 2c + 1); −1: no column
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = col0 + t * 8 + 2 * c + e;
        at[t][e] = col < n_cols ? s.pos + p.group.of(col) : -1;
      }
    const int at_low = s.pos + p.group.of(col0), at_high = s.pos + p.group.of(min(col0 + kCols, n_cols) - 1);

    float o[NG * 4][NT][4] = {};
    float top[NT][2], sum[NT][2] = {}, mid[NG][NT][2] = {};
#pragma unroll
    for (int t = 0; t < NT; ++t) top[t][0] = top[t][1] = -INFINITY;

    const int step0 = s.step0 + first, n_steps = s.last > 0 ? many : 0;
    const int32_t* table = p.cache.table + (int64_t)max(s.slot, 0) * p.cache.max_pages;
    auto page_of = [&](int u) {
      if (u >= n_steps) return -1;
      const int page = table[(step0 + u) / (kPage / kStep)];
      return page < p.cache.n_pages ? page : -1;
    };
    auto fetch = [&](int u, int page, int slot) {
      if (page >= 0) {
        const uint8_t* src = kv4_head(p.cache, p.layer, page, head) + (step0 + u) % (kPage / kStep) * S::kStage + lane * 16;
        uint8_t* dst = ring + slot * S::kStage + lane * 16;
#pragma unroll
        for (int b = 0; b < S::kStage; b += 512)
          if (S::kStage % 512 == 0 || b + lane * 16 < S::kStage) cp_async16(dst + b, src + b);
      }
      cp_async_commit();
    };
    uint32_t have = 0;   // bit u % 32: step u has a page
    int next;
#pragma unroll
    for (int u = 0; u < S::kStages - 1; ++u) {
      const int page = page_of(u);
      have |= (uint32_t)(page >= 0) << u;
      fetch(u, page, u);
    }
    next = page_of(S::kStages - 1);
    int slot = 0;

    // as the B operands of K·qᵀ, and their sums over each group
    uint4 qf[S::kQInRegs ? NT : 1][NG][2];
    float qsum[NG][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 u = raw[t][g][h];
          // entries {0, 2}, {1, 3}, {4, 6}, {5, 7}
          const uint4 v = make_uint4(__byte_perm(u.x, u.y, 0x5410), __byte_perm(u.x, u.y, 0x7632), __byte_perm(u.z, u.w, 0x5410), __byte_perm(u.z, u.w, 0x7632));
          if constexpr (S::kQInRegs) qf[t][g][h] = v;
          else q_smem[((t * NG + g) * 2 + h) * 32 + lane] = v;
          mma16816(sum, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.x, v.y);
          mma16816(sum, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, v.z, v.w);
        }
        qsum[g][t][0] = sum[0];
        qsum[g][t][1] = sum[1];
      }
    // scores of a step, as the products leave them
    auto scores = [&](const uint8_t* stage, float (&sc)[S::kTiles][NT][4]) {
#pragma unroll
      for (int k = 0; k < S::kTiles; ++k) {
        const uint8_t* tile = stage + k * S::kTile;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint4 w = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
          const uint2 small = *reinterpret_cast<const uint2*>(tile + NG * 512 + g * 64 + r * 8);
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
          float acc[NT][4] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a[4];
            nibbles_128(words[j], a);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              uint4 b;
              if constexpr (S::kQInRegs) b = qf[t][g][j / 2];
              else b = q_smem[((t * NG + g) * 2 + j / 2) * 32 + lane];
              mma16816(acc[t], a[0], a[2], a[1], a[3], j % 2 ? b.z : b.x, j % 2 ? b.w : b.y);
            }
          }
          const float s0 = bf16_lo(small.x), m0 = fmaf(-kNibbleOff, s0, bf16_hi(small.x)), s1 = bf16_lo(small.y), m1 = fmaf(-kNibbleOff, s1, bf16_hi(small.y));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sc[k][t][0] = fmaf(s0, acc[t][0], fmaf(m0, qsum[g][t][0], g ? sc[k][t][0] : 0.f));
            sc[k][t][1] = fmaf(s0, acc[t][1], fmaf(m0, qsum[g][t][1], g ? sc[k][t][1] : 0.f));
            sc[k][t][2] = fmaf(s1, acc[t][2], fmaf(m1, qsum[g][t][0], g ? sc[k][t][2] : 0.f));
            sc[k][t][3] = fmaf(s1, acc[t][3], fmaf(m1, qsum[g][t][1], g ? sc[k][t][3] : 0.f));
          }
        }
      }
    };
    // weights and values of a step; `whole`: every column sees all of it
    auto values = [&](const uint8_t* stage, const float (&sc)[S::kTiles][NT][4], auto whole) {
      float shift[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) shift[t][e] = whole || top[t][e] != -INFINITY ? -top[t][e] : 0.f;
#pragma unroll
      for (int k = 0; k < S::kTiles; ++k) {
        const uint8_t* tile = stage + k * S::kTile + NG * (512 + 64);
        float weight[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            weight[t][e] = exp2_fast(fmaf(sc[k][t][e], p.scale_log2, shift[t][e % 2]));
            sum[t][e % 2] += weight[t][e];
          }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint2 small = *reinterpret_cast<const uint2*>(tile + NG * 512 + g * 64 + r * 8);
          const float s0 = bf16_lo(small.x), m0 = bf16_hi(small.x), s1 = bf16_lo(small.y), m1 = bf16_hi(small.y);
          uint32_t b[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float w[4] = {weight[t][0] * s0, weight[t][1] * s0, weight[t][2] * s1, weight[t][3] * s1};
            float y[4] = {m0, m0, m1, m1};
            if constexpr (!whole) {   // what is not seen may hold anything
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (weight[t][e] == 0.f) w[e] = y[e] = 0.f;
            }
            mid[g][t][0] = fmaf(weight[t][2], y[2], fmaf(weight[t][0], y[0], mid[g][t][0]));
            mid[g][t][1] = fmaf(weight[t][3], y[3], fmaf(weight[t][1], y[1], mid[g][t][1]));
            b[t][0] = transpose8x8(pack2(w[0], w[1]));
            b[t][1] = transpose8x8(pack2(w[2], w[3]));
          }
          const uint4 v = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
          const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a[4];
            nibbles_bf16(words[j], a);   // exact: what is taken off afterwards would be rounded off the sums over all tokens
#pragma unroll
            for (int t = 0; t < NT; ++t) mma16816(o[g * 4 + j][t], a[0], a[1], a[2], a[3], b[t][0], b[t][1]);
          }
        }
      }
    };
    for (int u = 0; u < n_steps; ++u) {
      const int ahead = u + S::kStages - 1, into = slot == 0 ? S::kStages - 1 : slot - 1;
      have = (have & ~(1u << (ahead % 32))) | (uint32_t)(next >= 0) << (ahead % 32);
      fetch(ahead, next, into);
      next = page_of(ahead + 1);
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const uint8_t* stage = ring + slot * S::kStage;
      float sc[S::kTiles][NT][4];
      scores(stage, sc);
      // a page that is not there counts as not seen, whatever the stage holds
      const int key0 = (step0 + u) * kStep, last = have >> (u % 32) & 1 ? s.last : 0;
      const bool whole = key0 + kStep <= min(last, at_low + 1) && (p.window == 0 || at_high - key0 < p.window);
      if (!whole) {
#pragma unroll
        for (int k = 0; k < S::kTiles; ++k)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + k * kKvTile + r + 8 * (e / 2), from = at[t][e % 2];
              const bool seen = key <= from && key < last && (p.window == 0 || from - key < p.window);
              if (!seen) sc[k][t][e] = -INFINITY;
            }
      }
      float m[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[t][e] = -INFINITY;
#pragma unroll
          for (int k = 0; k < S::kTiles; ++k) m[t][e] = fmaxf(m[t][e], fmaxf(sc[k][t][e], sc[k][t][e + 2]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) m[t][e] = fmaxf(m[t][e], __shfl_xor_sync(0xffffffffu, m[t][e], x));
        }
      // The running maximum moves only where it would be passed by more than 2^8: up to there weights and sums are as exact with the old one
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[t][e] *= p.scale_log2;
          moved |= m[t][e] > top[t][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float now = fmaxf(top[t][e], m[t][e]), f = now == -INFINITY ? 1.f : exp2_fast(top[t][e] - now);   // 0 where there was none
            top[t][e] = now;
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
      if (whole) values(stage, sc, std::true_type());
      else values(stage, sc, std::false_type());
      __syncwarp();   // the stage is free
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncwarp();

    // Σ over the tokens is whole but for what the lanes of a column keep apart
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[t][e] += __shfl_xor_sync(0xffffffffu, sum[t][e], x);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float y = mid[g][t][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) y += __shfl_xor_sync(0xffffffffu, y, x);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[g * 4 + j][t][e] += y;
            o[g * 4 + j][t][e + 2] += y;
          }
        }
      }
    if (many == s.steps) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = col0 + t * 8 + 2 * c + e;
          if (col >= n_cols) continue;
          const float f = sum[t][e] == 0.f ? 0.f : 1.f / sum[t][e];
          const int token = p.group.of(col);
          __nv_bfloat16* dst = p.out + ((int64_t)(s.row0 + token) * p.q_heads + head * p.group.d + col - token * p.group.d) * kDim + 2 * r;
#pragma unroll
          for (int d = 0; d < NG * 4; ++d) *reinterpret_cast<uint32_t*>(dst + 16 * d) = pack2(o[d][t][e] * f, o[d][t][e + 2] * f);
        }
    } else {
      // all the CTA's warps have a piece, and of this item alone
      const int cta = cut.start(blockIdx.x * cut.each), cta_end = cut.start((blockIdx.x + 1) * cut.each);
      const bool inside = cut.each > 1 && cta >= begin && cta_end <= end && ((int)blockIdx.x + 1) * cut.each <= cut.warps;
      const int wide = inside ? kDim + 4 : kDim;   // (shared memory: columns on other banks)
      float* const part = inside ? reinterpret_cast<float*>(ring) : kv4_part(p, own, first == 0, kCols);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = t * 8 + 2 * c + e;
#pragma unroll
          for (int d = 0; d < NG * 4; ++d) *reinterpret_cast<float2*>(part + col * wide + 16 * d + 2 * r) = make_float2(o[d][t][e], o[d][t][e + 2]);
          if (r == 0) {
            part[kCols * wide + col] = top[t][e];
            part[kCols * wide + kCols + col] = sum[t][e];
          }
        }
      if (first == 0 && lane == 0) {
        Kv4Split split;
        auto warp_at = [&](int x) {   // whose piece of the line x is
          int w = min(x / cut.whole, cut.warps - 1);
          while (cut.start(w) > x) --w;
          while (cut.start(w + 1) <= x) ++w;
          return w;
        };
        split.from = me;
        split.to = warp_at(end - 1);
        split.in0 = cta == begin ? blockIdx.x : blockIdx.x + 1;
        split.in1 = cut.start(split.to + 1) == end && (split.to + 1) % cut.each == 0 ? (split.to + 1) / cut.each : split.to / cut.each;
        if (cut.each == 1) split.in1 = split.in0;
        split.row0 = s.row0;
        split.col0 = col0;
        split.n_cols = n_cols;
        split.head = head;
        split.each = cut.each;
        p.splits[own] = split;
      }
      if (inside) {   // every warp of the CTA that has a piece comes here, once
        named_bar_sync(1, cut.each * 32);
        float* const joined = kv4_part(p, (int64_t)blockIdx.x * S::kWarps, 0, kCols);
        for (int col = warp; col < kCols; col += cut.each) {   // a warp takes a column, a lane a warp's maximum and sum
          const float* of = reinterpret_cast<const float*>(smem + min(lane, cut.each - 1) * S::kOwn) + kCols * (kDim + 4) + col;
          float l = lane < cut.each ? of[kCols] : 0.f, m = l != 0.f ? of[0] : -INFINITY;   // (a sum that is no number has seen a token)
          float all = m;
#pragma unroll
          for (int x = 1; x < 32; x <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, x));
          const float f = l != 0.f ? exp2_fast(m - all) : 0.f;
          l *= f;
#pragma unroll
          for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
          float2 v[NG];
#pragma unroll
          for (int g = 0; g < NG; ++g) v[g] = make_float2(0.f, 0.f);
#pragma unroll 4
          for (int w = 0; w < cut.each; ++w) {
            const float fw = __shfl_sync(0xffffffffu, f, w);
            if (fw == 0.f) continue;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float2 o2 = *reinterpret_cast<const float2*>(smem + w * S::kOwn + (col * (kDim + 4) + g * 64 + 2 * lane) * 4);
              v[g].x = fmaf(fw, o2.x, v[g].x);
              v[g].y = fmaf(fw, o2.y, v[g].y);
            }
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) *reinterpret_cast<float2*>(joined + col * kDim + g * 64 + 2 * lane) = v[g];
          if (lane == 0) {
            joined[kCols * kDim + col] = all;
            joined[kCols * kDim + kCols + col] = l;
          }
        }
      }
    }
  }
}

// The items that lie in more than one warp's piece of the line.  CTA (c, column) takes those that begin in CTA c's pieces: a warp each while their parts are few,
// else all warps, every eighth part in order, and then the warps meet.
constexpr int kJoinWarps = 8;
template <int NG>
struct Joined {
  float m = -INFINITY, l = 0.f;
  float2 v[NG];
  __device__ Joined() {
#pragma unroll
    for (int g = 0; g < NG; ++g) v[g] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void take(float mw, float lw, const float2 (&x)[NG]) {
    if (lw == 0.f) return;   // has seen no token
    const float top = fmaxf(m, mw), f = exp2_fast(mw - top), keep = l == 0.f ? 0.f : exp2_fast(m - top);
    m = top;
    l = fmaf(f, lw, l * keep);
#pragma unroll
    for (int g = 0; g < NG; ++g) v[g] = make_float2(fmaf(f, x[g].x, v[g].x * keep), fmaf(f, x[g].y, v[g].y * keep));
  }
};
template <int NG>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(const Kv4Attn p, int columns, int warps) {
  __shared__ float part_m[kJoinWarps], part_l[kJoinWarps];
  __shared__ float2 part_v[kJoinWarps][NG * 32];
  constexpr int kDim = NG * 64, kAtOnce = 4;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, col = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const Kv4Split* splits = p.splits + blockIdx.x * warps;
  const Kv4Split mine = lane < warps ? splits[lane] : Kv4Split{-1};
  auto of = [&](int v, int from) { return __shfl_sync(0xffffffffu, v, from); };
  int number = 0;
  for (uint32_t left = __ballot_sync(0xffffffffu, mine.from >= 0 && mine.col0 + col < mine.n_cols); left != 0; left &= left - 1) {
    const int i = __ffs(left) - 1, from = of(mine.from, i), to = of(mine.to, i), in0 = of(mine.in0, i), in1 = of(mine.in1, i), each = of(mine.each, i);
    const bool some = in0 < in1;
    const int before = some ? in0 * each - from : to - from + 1, whole = some ? in1 - in0 : 0, parts = before + whole + (some ? to - in1 * each + 1 : 0);
    const bool alone = parts <= 2 * kAtOnce;
    if (alone && number++ % kJoinWarps != warp) continue;
    const int first = alone ? 0 : warp, step = alone ? 1 : kJoinWarps;
    Joined<NG> o;
    for (int k0 = first; k0 < parts; k0 += kAtOnce * step) {
      float m[kAtOnce], l[kAtOnce];
      float2 x[kAtOnce][NG];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const int k = min(k0 + e * step, parts - 1);
        const int w = k < before ? from + k : k < before + whole ? (in0 + k - before) * each : in1 * each + k - before - whole;
        const float* part = kv4_part(p, (int64_t)(w / each) * warps + w % each, k < before && k == 0, columns);
        m[e] = part[columns * kDim + col];
        l[e] = k0 + e * step < parts ? part[columns * kDim + columns + col] : 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) x[e][g] = *reinterpret_cast<const float2*>(part + col * kDim + g * 64 + 2 * lane);
      }
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) o.take(m[e], l[e], x[e]);
    }
    const int at = of(mine.col0, i) + col;
    const int token = p.group.of(at);
    __nv_bfloat16* out = p.out + ((int64_t)(of(mine.row0, i) + token) * p.q_heads + of(mine.head, i) * p.group.d + at - token * p.group.d) * kDim;
    if (!alone) {
      if (lane == 0) {
        part_m[warp] = o.m;
        part_l[warp] = o.l;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) part_v[warp][g * 32 + lane] = o.v[g];
      __syncthreads();
      if (warp == 0) {
        o = Joined<NG>();
        for (int w = 0; w < kJoinWarps; ++w) {
          float2 x[NG];
#pragma unroll
          for (int g = 0; g < NG; ++g) x[g] = part_v[w][g * 32 + lane];
          o.take(part_m[w], part_l[w], x);
        }
      }
      __syncthreads();
    }
    if (alone || warp == 0) {
      const float f = o.l == 0.f ? 0.f : 1.f / o.l;
#pragma unroll
      for (int g = 0; g < NG; ++g) *reinterpret_cast<uint32_t*>(out + g * 64 + 2 * lane) = pack2(o.v[g].x * f, o.v[g].y * f);
    }
  }
}

// Column tiles of a block: what an average sequence brings.
int column_tiles(int64_t group, int64_t n, int64_t rows) { return group * ((rows + n - 1) / n) <= 8 ? 1 : 2; }

template <int NG, int NT>
int launch(const Kv4Attn& p, cudaStream_t st) {
  using S = Shape<NG, NT>;
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(kv4_attn_kernel<NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); }));
  const bool pdl = op_pdl(st);
  B200_CUDA(launch_pdl(kv4_attn_kernel<NG, NT>, dim3(kGrid), dim3(S::kThreads), S::kSmem, st, pdl, p));
  B200_CUDA(launch_pdl(kv4_join_kernel<NG>, dim3(kGrid, 8 * NT), dim3(kJoinWarps * 32), 0, st, pdl, p, 8 * NT, S::kWarps));
  return B200_OK;
}
int warps_of(int groups, int tiles) {
  switch (groups * 2 + tiles - 3) {
    case 0: return Shape<1, 1>::kWarps;
    case 1: return Shape<1, 2>::kWarps;
    case 2: return Shape<2, 1>::kWarps;
    case 3: return Shape<2, 2>::kWarps;
    case 4: return Shape<3, 1>::kWarps;
    case 5: return Shape<3, 2>::kWarps;
    case 6: return Shape<4, 1>::kWarps;
    default: return Shape<4, 2>::kWarps;
  }
}

}  // namespace

}  // namespace b200

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(const b200_kv4_cache* cache, int64_t q_heads, int64_t n, int64_t rows) {
  using namespace b200;
  if (cache == nullptr || cache->kv_heads < 1 || q_heads < 1 || q_heads % cache->kv_heads != 0 || n < 1 || rows < 1) return -1;
  if (cache->dim % kKvGroup != 0 || cache->dim < 64 || cache->dim > 256) return -1;
  const int tiles = column_tiles(q_heads / cache->kv_heads, n, rows);
  return (int64_t)kGrid * warps_of(cache->dim / kKvGroup, tiles) * (2 * 8 * tiles * (cache->dim + 2) * 4 + (int64_t)sizeof(Kv4Split));
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
  // the line of all work is counted in 32 bits: 1 M rows of 32 heads over 64 K tokens, or 64 K over 1 M
  const int64_t group = q_heads / cache->kv_heads, columns = 8 * column_tiles(group, n, rows);
  const int64_t items = cache->kv_heads * std::min(rows * ((group + columns - 1) / columns), rows * group / columns + n);
  B200_CHECK_ARG(items * ((int64_t)cache->max_pages * (kPage / kStep) + kAhead) < 1ll << 31 && rows * q_heads < 1ll << 31,
                 "kv4_attention: %lld rows of %lld heads over %d pages are too many for one call", (long long)rows, (long long)q_heads, cache->max_pages);
  Kv4Attn p{};
  p.cache = *cache;
  p.out = (__nv_bfloat16*)out;
  p.q = (const __nv_bfloat16*)q;
  p.ld_q = ld_q;
  p.seqs = seqs;
  p.starts = starts;
  p.pos = pos;
  p.parts = (float*)workspace;
  const int tiles = column_tiles(q_heads / cache->kv_heads, n, rows);
  p.splits = (Kv4Split*)(p.parts + (int64_t)kGrid * warps_of(cache->dim / kKvGroup, tiles) * 2 * 8 * tiles * (cache->dim + 2));
  p.layer = (int)layer;
  p.q_heads = (int)q_heads;
  p.group = Divisor((uint32_t)(q_heads / cache->kv_heads));
  p.kv_heads = Divisor((uint32_t)cache->kv_heads);
  p.n = (int)n;
  p.rows = (int)rows;
  p.window = (int)std::min<int64_t>(window, INT32_MAX);
  p.scale_log2 = scale * 1.44269504f;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool two = tiles == 2;
  switch (cache->dim / kKvGroup) {
    case 1: return two ? launch<1, 2>(p, st) : launch<1, 1>(p, st);
    case 2: return two ? launch<2, 2>(p, st) : launch<2, 1>(p, st);
    case 3: return two ? launch<3, 2>(p, st) : launch<3, 1>(p, st);
    default: return two ? launch<4, 2>(p, st) : launch<4, 1>(p, st);
  }
}

}  // extern "C"
