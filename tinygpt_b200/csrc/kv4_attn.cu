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
#include "kv4_steps.cuh"
#include "tc.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr float kSlack = 8.f;

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

// A sequence of the call: its rows and the tokens below `last` that they may see.  Nothing else reads the call's lists and the lengths; who writes to them meanwhile
// spoils results, but no two threads that meet at a barrier may go by different ones.
struct Kv4Rows {
  int row0, count, pos, slot, last;
};
__device__ __forceinline__ Kv4Rows kv4_read(const Kv4Attn& p, int i) {
  Kv4Rows s;
  s.row0 = min(max(p.starts[i], 0), p.rows);
  s.count = max(min(p.starts[i + 1], p.rows) - s.row0, 0);
  s.pos = min(p.pos[i], INT32_MAX - 64 - s.count);   // (so that positions, and a step behind them, stay in 32 bits)
  s.slot = p.seqs[i];
  s.last = 0;
  if (s.pos >= 0 && s.slot >= 0 && s.slot < p.cache.n_seqs)
    s.last = (int)min(min((int64_t)p.cache.length[s.slot], (int64_t)s.pos + s.count), min((int64_t)p.cache.max_pages * kPage, (int64_t)(1 << 30)));
  s.last = max(s.last, 0);
  return s;
}
__device__ __forceinline__ Kv4Rows kv4_read_warp(const Kv4Attn& p, int i) {   // lane 0's reading, for a warp
  const Kv4Rows s = kv4_read(p, i);
  Kv4Rows o;
  o.row0 = __shfl_sync(0xffffffffu, s.row0, 0);
  o.count = __shfl_sync(0xffffffffu, s.count, 0);
  o.pos = __shfl_sync(0xffffffffu, s.pos, 0);
  o.slot = __shfl_sync(0xffffffffu, s.slot, 0);
  o.last = __shfl_sync(0xffffffffu, s.last, 0);
  return o;
}
// The same with its items: steps step0 … step0 + steps − 1 (one at least), blocks of columns.
struct Kv4Seq : Kv4Rows {
  int step0, steps, blocks;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn& p, const Kv4Rows& rows, int columns) {
  Kv4Seq s;
  static_cast<Kv4Rows&>(s) = rows;
  s.blocks = (int)(((int64_t)s.count * p.group.d + columns - 1) / columns);
  const Kv4Steps steps = kv4_seq_steps(s.pos, s.last, p.window);
  s.step0 = steps.first;
  s.steps = steps.n;
  return s;
}
// The steps that a block of columns sees, from s.step0 on: the first of them, and how many (one at least).
__device__ __forceinline__ Kv4Steps kv4_block_steps(const Kv4Attn& p, const Kv4Seq& s, int block, int columns) {
  const int low = s.pos + p.group.of(block * columns), high = s.pos + p.group.of(min((block + 1) * columns, s.count * (int)p.group.d) - 1);
  return kv4_rows_steps(low, high, s.last, p.window, {s.step0, s.steps});
}
// What a sequence takes of the line.  EXACT: every block what its own columns see (a prompt's first rows see little of it, and under a window none sees all: 2 048
// rows of 16 / 8 heads of 128 from the first token on 194 → 114 µs); else all that the sequence's rows see.
template <bool EXACT>
__device__ __forceinline__ long long kv4_line(const Kv4Attn& p, const Kv4Seq& s, int columns) {
  if constexpr (!EXACT) return (long long)s.blocks * p.cache.kv_heads * (s.steps + kAhead);
  long long sum = 0;
  for (int b = 0; b < s.blocks; ++b) sum += kv4_block_steps(p, s, b, columns).n + kAhead;
  return sum * p.cache.kv_heads;
}
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
// be, and nothing is done.  `rows`: the sequences, where they have been read (EXACT).  All threads of a CTA of THREADS.
__device__ __forceinline__ int kv4_whole(long long line) { return line <= INT32_MAX ? (int)line : 0; }
template <int THREADS, bool EXACT>
__device__ int kv4_plan(const Kv4Attn& p, int columns, int* ends, const Kv4Rows* rows) {
  __shared__ long long carry[THREADS / 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, each = (p.n + THREADS - 1) / THREADS, first = threadIdx.x * each;
  long long sum = 0;
  for (int i = first; i < min(first + each, p.n); ++i) {
    const long long length = kv4_line<EXACT>(p, kv4_seq(p, EXACT ? rows[i] : kv4_read(p, i), columns), columns);
    ends[i] = (int)min(length, (long long)INT32_MAX);
    sum += length;
  }
  const long long upto = warp_scan(sum, lane);
  if (lane == 31) carry[warp] = upto;
  __syncthreads();
  long long before = upto - sum, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += carry[w];
    all += carry[w];
  }
  for (int i = first; i < min(first + each, p.n); ++i) ends[i] = (int)(before += ends[i]);
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
// a warp's parts: of an item that came before it (0) and of one that goes on behind it (1).  [column][dim], maxima, sums
__device__ __forceinline__ float* kv4_part(const Kv4Attn& p, int64_t warp, int which, int columns) {
  return p.parts + (warp * 2 + which) * columns * (p.cache.dim + 2);
}
// An item that its first warp does not finish, for the kernel that joins the parts: the pieces that hold it, its columns.
struct Kv4Split : Kv4Pieces {
  int row0, col0, n_cols, head;
};

// What a warp keeps of its 8·NT columns while it goes over the tokens: lane 4r + c has columns 2c, 2c + 1 of every tile.
template <int NG, int NT>
struct Columns {
  static constexpr int kDim = NG * 64, kTiles = kStep / kKvTile;
  float o[NG * 4][NT][4], mid[NG][NT][2], top[NT][2], sum[NT][2], qsum[NG][NT][2];
  int at[NT][2];          // positions; −1: no column
  int at_low, at_high;    // of the block

  __device__ __forceinline__ void start(const Kv4Attn& p, const Kv4Seq& s, int col0, int n_cols, int c) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = col0 + t * 8 + 2 * c + e;
        at[t][e] = col < n_cols ? s.pos + p.group.of(col) : -1;
        top[t][e] = -INFINITY;
        sum[t][e] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) mid[g][t][e] = 0.f;
#pragma unroll
        for (int d = 0; d < NG * 4; ++d) o[d][t][e] = o[d][t][e + 2] = 0.f;
      }
    at_low = s.pos + p.group.of(col0);
    at_high = s.pos + p.group.of(min(col0 + 8 * NT, n_cols) - 1);
  }
  // q's rows of the columns → the B operands of K·qᵀ (entries {0, 2}, {1, 3}, {4, 6}, {5, 7} of eight) and their sums over each group
  __device__ __forceinline__ void take(int g, int t, uint4 (&q)[2]) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = q[h];
      q[h] = make_uint4(__byte_perm(u.x, u.y, 0x5410), __byte_perm(u.x, u.y, 0x7632), __byte_perm(u.z, u.w, 0x5410), __byte_perm(u.z, u.w, 0x7632));
      mma16816(s, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, q[h].x, q[h].y);
      mma16816(s, kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones, q[h].z, q[h].w);
    }
    qsum[g][t][0] = s[0];
    qsum[g][t][1] = s[1];
  }
  // scores of a step, as the products leave them: `words` gives the A operands of a tile and group, `small` its scales and middles, `query` the B operands
  template <typename Words, typename Small, typename Query>
  __device__ __forceinline__ void scores(float (&sc)[kTiles][NT][4], const Words& words, const Small& small, const Query& query) const {
#pragma unroll
    for (int k = 0; k < kTiles; ++k)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const auto w = words(k, g);
        const uint2 two = small(k, g);
        float acc[NT][4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
          w.keys(j, a);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4 b = query(t, g, j / 2);
            mma16816(acc[t], a[0], a[2], a[1], a[3], j % 2 ? b.z : b.x, j % 2 ? b.w : b.y);
          }
        }
        const float s0 = bf16_lo(two.x), m0 = fmaf(-w.kOff, s0, bf16_hi(two.x)), s1 = bf16_lo(two.y), m1 = fmaf(-w.kOff, s1, bf16_hi(two.y));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          sc[k][t][0] = fmaf(s0, acc[t][0], fmaf(m0, qsum[g][t][0], g ? sc[k][t][0] : 0.f));
          sc[k][t][1] = fmaf(s0, acc[t][1], fmaf(m0, qsum[g][t][1], g ? sc[k][t][1] : 0.f));
          sc[k][t][2] = fmaf(s1, acc[t][2], fmaf(m1, qsum[g][t][0], g ? sc[k][t][2] : 0.f));
          sc[k][t][3] = fmaf(s1, acc[t][3], fmaf(m1, qsum[g][t][1], g ? sc[k][t][3] : 0.f));
        }
      }
  }
  // whether every column sees all tokens of the step at key0; where not, the scores of the others are −∞
  __device__ __forceinline__ bool mask(float (&sc)[kTiles][NT][4], int key0, int last, int window, int r) const {
    const bool whole = key0 + kStep <= min(last, at_low + 1) && (window == 0 || at_high - key0 < window);
    if (!whole) {
#pragma unroll
      for (int k = 0; k < kTiles; ++k)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + k * kKvTile + r + 8 * (e / 2), from = at[t][e % 2];
            const bool seen = key <= from && key < last && (window == 0 || from - key < window);
            if (!seen) sc[k][t][e] = -INFINITY;
          }
    }
    return whole;
  }
  // The running maximum moves only where it would be passed by more than 2^8: up to there weights and sums are as exact with the old one.
  __device__ __forceinline__ void settle(const float (&sc)[kTiles][NT][4], float scale_log2) {
    float m[NT][2];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[t][e] = -INFINITY;
#pragma unroll
        for (int k = 0; k < kTiles; ++k) m[t][e] = fmaxf(m[t][e], fmaxf(sc[k][t][e], sc[k][t][e + 2]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) m[t][e] = fmaxf(m[t][e], __shfl_xor_sync(0xffffffffu, m[t][e], x));
        m[t][e] *= scale_log2;
        moved |= m[t][e] > top[t][e] + kSlack;
      }
    if (!__any_sync(0xffffffffu, moved)) return;
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
  // weights and values of a step
  template <bool WHOLE, typename Words, typename Small>
  __device__ __forceinline__ void values(const float (&sc)[kTiles][NT][4], float scale_log2, const Words& words, const Small& small) {
    float shift[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) shift[t][e] = WHOLE || top[t][e] != -INFINITY ? -top[t][e] : 0.f;
#pragma unroll
    for (int k = 0; k < kTiles; ++k) {
      float weight[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          weight[t][e] = exp2_fast(fmaf(sc[k][t][e], scale_log2, shift[t][e % 2]));
          sum[t][e % 2] += weight[t][e];
        }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 two = small(k, g);
        const float s0 = bf16_lo(two.x), m0 = bf16_hi(two.x), s1 = bf16_lo(two.y), m1 = bf16_hi(two.y);
        uint32_t b[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float w[4] = {weight[t][0] * s0, weight[t][1] * s0, weight[t][2] * s1, weight[t][3] * s1};
          float y[4] = {m0, m0, m1, m1};
          if constexpr (!WHOLE) {   // what is not seen may hold anything (and what is seen counts, however small its weight)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sc[k][t][e] == -INFINITY) w[e] = y[e] = 0.f;
          }
          mid[g][t][0] = fmaf(weight[t][2], y[2], fmaf(weight[t][0], y[0], mid[g][t][0]));
          mid[g][t][1] = fmaf(weight[t][3], y[3], fmaf(weight[t][1], y[1], mid[g][t][1]));
          b[t][0] = transpose8x8(pack2(w[0], w[1]));
          b[t][1] = transpose8x8(pack2(w[2], w[3]));
        }
        const auto v = words(k, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
          v.values(j, a);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma16816(o[g * 4 + j][t], a[0], a[1], a[2], a[3], b[t][0], b[t][1]);
        }
      }
    }
  }
  // Σ over the tokens is whole then, but for what the lanes of a column have kept apart
  __device__ __forceinline__ void finish() {
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
  }
  __device__ __forceinline__ void write(const Kv4Attn& p, const Kv4Seq& s, int head, int col0, int n_cols, int r, int c) const {
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
  }
  // as a part: columns first … of `columns`, `wide` floats from one to the next, behind them all maxima and all sums
  __device__ __forceinline__ void leave(float* part, int first, int columns, int wide, int r, int c) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = first + t * 8 + 2 * c + e;
#pragma unroll
        for (int d = 0; d < NG * 4; ++d) *reinterpret_cast<float2*>(part + col * wide + 16 * d + 2 * r) = make_float2(o[d][t][e], o[d][t][e + 2]);
        if (r == 0) {
          part[columns * wide + col] = top[t][e];
          part[columns * wide + columns + col] = sum[t][e];
        }
      }
  }
};
// the query that column `col` of the block belongs to, eight entries from 8c on
template <int NG>
__device__ __forceinline__ const __nv_bfloat16* kv4_query(const Kv4Attn& p, const Kv4Seq& s, int head, int col, int c) {
  const int token = p.group.of(col);
  return p.q + (int64_t)(s.row0 + token) * p.ld_q + (int64_t)(head * p.group.d + col - token * p.group.d) * (NG * 64) + 8 * c;
}
// A operands from a tile's nibbles
struct Nibbles {
  static constexpr float kOff = kNibbleOff;
  uint4 w;
  __device__ __forceinline__ uint32_t word(int j) const { return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w; }
  __device__ __forceinline__ void keys(int j, uint32_t (&a)[4]) const { nibbles_128(word(j), a); }
  __device__ __forceinline__ void values(int j, uint32_t (&a)[4]) const { nibbles_bf16(word(j), a); }   // exact: 136 taken off later would be rounded off the sums over all tokens
};
// the same, unpacked in shared memory
struct Unpacked {
  static constexpr float kOff = 0.f;
  const uint4* of;   // this lane's, of word 0
  __device__ __forceinline__ void keys(int j, uint32_t (&a)[4]) const {
    const uint4 v = of[j * 32];
    a[0] = v.x;
    a[1] = v.y;
    a[2] = v.z;
    a[3] = v.w;
  }
  __device__ __forceinline__ void values(int j, uint32_t (&a)[4]) const { keys(j, a); }
};

// A CTA's (EXACT) or a warp's way along the line: the sequences' ends, and one item after the other.  Warps that go their way together have the sequences from one
// reading in shared memory; those that go alone read them for themselves, and meet at no barrier that depends on what they read.
constexpr int walk_room(bool exact) { return kKvMaxSeqs * (4 + (exact ? (int)sizeof(Kv4Rows) : 0)); }   // bytes of shared memory
template <bool EXACT>
struct Walk {
  Kv4Seq mine;      // up to 32 sequences: every warp has them all in its lanes
  int mine_end, line, i;
  const int* ends;  // more: in shared memory
  const Kv4Rows* rows;
  bool few;
  template <int THREADS>
  __device__ __forceinline__ void plan(const Kv4Attn& p, int columns, int* room) {
    const int lane = threadIdx.x % 32;
    few = p.n <= 32;
    ends = room;
    rows = reinterpret_cast<const Kv4Rows*>(room + kKvMaxSeqs);
    mine = Kv4Seq{};
    mine_end = 0;
    if constexpr (EXACT) {
      for (int k = threadIdx.x; k < p.n; k += THREADS) reinterpret_cast<Kv4Rows*>(room + kKvMaxSeqs)[k] = kv4_read(p, k);
      __syncthreads();
    }
    if (few) {
      if (lane < p.n) mine = kv4_seq(p, EXACT ? rows[lane] : kv4_read(p, lane), columns);
      constexpr int kAlone = EXACT ? 2 : INT32_MAX;   // blocks that a lane goes through by itself
      long long length = lane < p.n && mine.blocks <= kAlone ? kv4_line<EXACT>(p, mine, columns) : 0;
      for (uint32_t left = __ballot_sync(0xffffffffu, mine.blocks > kAlone); left != 0; left &= left - 1) {
        const int of = __ffs(left) - 1;
        const Kv4Seq s = kv4_from(mine, of);
        long long sum = 0;
        for (int b = lane; b < s.blocks; b += 32) sum += kv4_block_steps(p, s, b, columns).n + kAhead;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == of) length = sum * p.cache.kv_heads;
      }
      const long long end = warp_scan(length, lane);
      mine_end = (int)end;
      line = kv4_whole(__shfl_sync(0xffffffffu, end, 31));
    } else {
      line = kv4_plan<THREADS, EXACT>(p, columns, room, rows);
    }
  }
  __device__ __forceinline__ void seek(int n, int at, int stop) { i = !few && at < stop ? kv4_find(ends, n, at) : 0; }
  // the item at this place of the line: its sequence, key/value head, block of columns; its steps lie at begin … end − 1
  Kv4Seq s;
  int head, block, begin, end;
  __device__ __forceinline__ void item(const Kv4Attn& p, int columns, int at) {
    int base = 0, limit;
    if (few) {
      i = __popc(__ballot_sync(0xffffffffu, mine_end <= at));
      if (i > 0) base = __shfl_sync(0xffffffffu, mine_end, i - 1);
      limit = __shfl_sync(0xffffffffu, mine_end, i);
      s = kv4_from(mine, i);
    } else {
      while (ends[i] <= at) ++i;
      if (i > 0) base = ends[i - 1];
      limit = ends[i];
      s = kv4_seq(p, EXACT ? rows[i] : kv4_read_warp(p, i), columns);
    }
    if constexpr (EXACT) {
      const int lane = threadIdx.x % 32;
      block = 0;
      for (int first = 0; first < s.blocks; first += 32) {   // (`at` lies in a block of the sequence)
        const Kv4Steps steps = first + lane < s.blocks ? kv4_block_steps(p, s, first + lane, columns) : Kv4Steps{0, -kAhead};
        const int upto = (int)warp_scan((long long)(steps.n + kAhead) * (int)p.kv_heads.d, lane);
        const uint32_t before = __ballot_sync(0xffffffffu, base + upto <= at);
        if (before == 0xffffffffu) {
          base += __shfl_sync(0xffffffffu, upto, 31);
          continue;
        }
        const int k = __popc(before);
        if (k > 0) base += __shfl_sync(0xffffffffu, upto, k - 1);
        block = first + k;
        s.step0 += __shfl_sync(0xffffffffu, steps.first, k);
        s.steps = __shfl_sync(0xffffffffu, steps.n, k);
        break;
      }
    }
    const Kv4Item item = kv4_item(at, base, limit, s.steps);
    if constexpr (EXACT) {
      head = min(item.number, (int)p.kv_heads.d - 1);
    } else {
      block = p.kv_heads.of(item.number);
      head = item.number - block * p.kv_heads.d;
    }
    begin = item.begin;
    end = item.end;
  }
};
template <bool EXACT>
__device__ __forceinline__ void kv4_split(const Kv4Attn& p, const Walk<EXACT>& w, const Kv4Cut& cut, int64_t own, int me, int col0, int n_cols) {
  Kv4Split split;
  static_cast<Kv4Pieces&>(split) = kv4_pieces(cut, blockIdx.x, me, w.begin, w.end);
  split.row0 = w.s.row0;
  split.col0 = col0;
  split.n_cols = n_cols;
  split.head = w.head;
  p.splits[own] = split;
}
// rows of no sequence are zero
__device__ __forceinline__ void kv4_others(const Kv4Attn& p) {
  const int head = min(max(p.starts[0], 0), p.rows), tail = min(max(p.starts[p.n], head), p.rows), width = p.q_heads * p.cache.dim;
  for (int row = blockIdx.x; row < head + p.rows - tail; row += gridDim.x)
    for (int d = threadIdx.x; d < width; d += blockDim.x) p.out[(int64_t)(row < head ? row : row - head + tail) * width + d] = f_to_bf16(0.f);
}

// ---- few columns to a sequence: every warp for itself.  Two tiles of columns of heads of 192 and 256 take more than 255 registers (some 70 and 450 bytes of spills): 2 × 8 rows of 8 / 4
// heads of 256 over 8 000 and 3 000 tokens 22.6 µs.
// (the workspace is sized by this)
constexpr int kPieceWarps = 8;
template <int NG, int NT>
struct Shape {
  static constexpr int kTile = kv4_tile_bytes(NG);
  static constexpr int kTiles = kStep / kKvTile;                // of a step
  static constexpr int kStage = kTiles * kTile;
  static constexpr int kWarps = kPieceWarps, kPieces = kWarps, kCols = 8 * NT;   // pieces of the line to a CTA, columns of a block
  static constexpr int kThreads = kWarps * 32;
  static constexpr bool kQInRegs = NG * NT <= 4;
  static constexpr int kQBytes = kQInRegs ? 0 : NT * NG * 2 * 512;
  static constexpr int kRoom = 232448 - 1024 - walk_room(false);
  static constexpr int kStages = kWarps * (3 * kStage + kQBytes) <= kRoom ? 3 : 2;
  static constexpr int kRing = kStages * kStage > 8 * NT * (NG * 64 + 6) * 4 ? kStages * kStage : (8 * NT * (NG * 64 + 6) * 4 + 15) / 16 * 16;
  static constexpr int kOwn = kRing + kQBytes;                  // shared memory of a warp
  static constexpr int kSmem = kWarps * kOwn + walk_room(false);
  static_assert(kWarps * kOwn <= kRoom, "shared memory of an SM");
};

// A warp goes over steps first … first + many − 1 of a sequence's with the columns of a block.
template <int NG, int NT>
__device__ __forceinline__ void kv4_run(const Kv4Attn& p, const Kv4Seq& s, int head, int col0, int n_cols, int first, int many, uint8_t* own, Columns<NG, NT>& cols) {
  using S = Shape<NG, NT>;
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  uint8_t* const ring = own;
  uint4* const q_smem = reinterpret_cast<uint4*>(own + S::kRing);
  uint4 q[NT][NG][2];   // the block's queries
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = col0 + t * 8 + r;
    const __nv_bfloat16* src = kv4_query<NG>(p, s, head, col, c);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) q[t][g][h] = col < n_cols ? *reinterpret_cast<const uint4*>(src + g * 64 + h * 32) : make_uint4(0, 0, 0, 0);
  }
  cols.start(p, s, col0, n_cols, c);

  // (steps that no column sees, in a block whose columns stand far apart from the sequence's others, are not gone over)
  const int step0 = s.step0 + first, n_steps = col0 < n_cols ? kv4_steps_end(cols.at_high, s.last, step0, many) : 0;
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
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      cols.take(g, t, q[t][g]);
      if constexpr (!S::kQInRegs) {
        q_smem[((t * NG + g) * 2) * 32 + lane] = q[t][g][0];
        q_smem[((t * NG + g) * 2 + 1) * 32 + lane] = q[t][g][1];
      }
    }
  for (int u = 0; u < n_steps; ++u) {
    const int ahead = u + S::kStages - 1, into = slot == 0 ? S::kStages - 1 : slot - 1;
    have = (have & ~(1u << (ahead % 32))) | (uint32_t)(next >= 0) << (ahead % 32);
    fetch(ahead, next, into);
    next = page_of(ahead + 1);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    const uint8_t* stage = ring + slot * S::kStage;
    auto keys = [&](int k, int g) { return Nibbles{*reinterpret_cast<const uint4*>(stage + k * S::kTile + g * 512 + lane * 16)}; };
    auto key_small = [&](int k, int g) { return *reinterpret_cast<const uint2*>(stage + k * S::kTile + NG * 512 + g * 64 + r * 8); };
    auto values = [&](int k, int g) { return Nibbles{*reinterpret_cast<const uint4*>(stage + k * S::kTile + NG * (512 + 64) + g * 512 + lane * 16)}; };
    auto value_small = [&](int k, int g) { return *reinterpret_cast<const uint2*>(stage + k * S::kTile + NG * (512 + 64 + 512) + g * 64 + r * 8); };
    auto query = [&](int t, int g, int h) {
      if constexpr (S::kQInRegs) return q[t][g][h];
      else return q_smem[((t * NG + g) * 2 + h) * 32 + lane];
    };
    float sc[S::kTiles][NT][4];
    cols.scores(sc, keys, key_small, query);
    // a page that is not there counts as not seen, whatever the stage holds
    const bool whole = cols.mask(sc, (step0 + u) * kStep, have >> (u % 32) & 1 ? s.last : 0, p.window, r);
    cols.settle(sc, p.scale_log2);
    if (whole) cols.template values<true>(sc, p.scale_log2, values, value_small);
    else cols.template values<false>(sc, p.scale_log2, values, value_small);
    __syncwarp();   // the stage is free
    slot = slot + 1 == S::kStages ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  __syncwarp();
  cols.finish();
}

// The parts of a CTA's first `each` warps, left in their shared memory, become one at `joined`, `wide` floats from a column to the next: a warp takes a column, a lane a
// warp's maximum and sum.
template <int NG>
constexpr int kMeetWide = NG * 64 + 4;   // floats of a column there (columns on other banks)
template <int NG, int NT>
__device__ __forceinline__ void kv4_meet(const uint8_t* smem, int each, float* joined, int wide) {
  using S = Shape<NG, NT>;
  constexpr int kCols = S::kCols, kWide = kMeetWide<NG>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int col = warp; col < kCols; col += each) {
    const float* of = reinterpret_cast<const float*>(smem + min(lane, each - 1) * S::kOwn) + kCols * kWide + col;
    float l = lane < each ? of[kCols] : 0.f, m = l != 0.f ? of[0] : -INFINITY;   // (a sum that is no number has seen a token)
    float all = m;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, x));
    const float f = l != 0.f ? exp2_fast(m - all) : 0.f;
    const uint32_t some = __ballot_sync(0xffffffffu, l != 0.f);   // warps that have seen a token
    l *= f;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    float2 v[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) v[g] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < each; ++k) {
      const float fk = __shfl_sync(0xffffffffu, f, k);
      if (!(some >> k & 1)) continue;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float2 o2 = *reinterpret_cast<const float2*>(smem + k * S::kOwn + (col * kWide + g * 64 + 2 * lane) * 4);
        v[g].x = fmaf(fk, o2.x, v[g].x);
        v[g].y = fmaf(fk, o2.y, v[g].y);
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) *reinterpret_cast<float2*>(joined + col * wide + g * 64 + 2 * lane) = v[g];
    if (lane == 0) {
      joined[kCols * wide + col] = all;
      joined[kCols * wide + kCols + col] = l;
    }
  }
}

template <int NG, int NT>
__global__ void __launch_bounds__(Shape<NG, NT>::kThreads, 1) kv4_attn_kernel(const Kv4Attn p) {
  using S = Shape<NG, NT>;
  constexpr int kCols = 8 * NT, kDim = NG * 64;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  uint8_t* const ring = smem + warp * S::kOwn;
  pdl_wait();
  pdl_trigger();

  Walk<false> w{};
  w.template plan<S::kThreads>(p, kCols, reinterpret_cast<int*>(smem + S::kWarps * S::kOwn));
  const Kv4Cut cut(w.line, S::kWarps);
  const int me = blockIdx.x * cut.each + warp;
  const int64_t own = (int64_t)blockIdx.x * S::kWarps + warp;   // of the workspace's places
  int at_line = cut.start(me);
  const int stop = warp < cut.each ? cut.start(me + 1) : at_line;
  if (lane == 0) p.splits[own].from = -1;
  w.seek(p.n, at_line, stop);
  bool left_here = false;   // all the CTA's warps that have a piece leave their part here, of one item, or none does
  while (at_line < stop) {
    w.item(p, kCols, at_line);
    const Kv4Seq& s = w.s;
    const int first = max(at_line - w.begin, 0), many = min(stop, w.end) - w.begin - first;
    at_line = min(stop, w.end);
    if (many <= 0) continue;

    const int col0 = w.block * kCols, n_cols = s.count * p.group.d;
    Columns<NG, NT> cols;
    kv4_run(p, s, w.head, col0, n_cols, first, many, ring, cols);
    if (many == s.steps) {
      cols.write(p, s, w.head, col0, n_cols, r, c);
      continue;
    }
    if (first == 0 && lane == 0) kv4_split(p, w, cut, own, me, col0, n_cols);
    // all the CTA's warps have a piece, and of this item alone
    if (!kv4_inside(cut, blockIdx.x, w.begin, w.end)) {
      cols.leave(kv4_part(p, own, first == 0, kCols), 0, kCols, kDim, r, c);
      continue;
    }
    cols.leave(reinterpret_cast<float*>(ring), 0, kCols, kMeetWide<NG>, r, c);
    left_here = true;   // (its last item)
  }
  if (__syncthreads_and(left_here || warp >= cut.each) && warp < cut.each) kv4_meet<NG, NT>(smem, cut.each, kv4_part(p, (int64_t)blockIdx.x * S::kWarps, 0, kCols), kDim);
  kv4_others(p);
}

// ---- few columns to a sequence of a small cache: a cluster takes a sequence's head, its warps equal pieces of the steps; the parts meet in shared memory, first the
// CTA's, then over the cluster's.  One launch, no workspace.
template <int NG, int NT>
struct Cluster : Shape<NG, NT> {
  using S = Shape<NG, NT>;
  static constexpr int kWide = kMeetWide<NG>, kJoined = S::kWarps * S::kOwn;      // the CTA's part, behind the warps' rings
  static constexpr int kSmem = kJoined + S::kCols * (kWide + 2) * 4;
};
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
template <int NG, int NT>
__global__ void __launch_bounds__(Shape<NG, NT>::kThreads, 1) kv4_cluster_kernel(const Kv4Attn p, int ctas) {
  using S = Cluster<NG, NT>;
  constexpr int kCols = S::kCols, kDim = NG * 64;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, rank = (int)cluster_rank();
  uint8_t* const ring = smem + warp * S::kOwn;
  float* const joined = reinterpret_cast<float*>(smem + S::kJoined);
  pdl_wait();
  pdl_trigger();
  const int number = blockIdx.x / ctas, i = p.kv_heads.of(number), head = number - i * p.kv_heads.d;
  const Kv4Seq s = kv4_seq(p, kv4_read_warp(p, i), kCols);
  const int n_cols = s.count * p.group.d, piece = rank * S::kWarps + warp, pieces = ctas * S::kWarps;
  const int first = (int)((int64_t)s.steps * piece / pieces), many = (int)((int64_t)s.steps * (piece + 1) / pieces) - first;
  __shared__ int blocks_here;   // of the first CTA: all of the cluster go over so many
  int blocks = 1;
  if (threadIdx.x == 0) blocks_here = s.blocks;
  for (int col0 = 0, block = 0; block < blocks; ++block, col0 += kCols) {
    Columns<NG, NT> cols;
    kv4_run(p, s, head, col0, n_cols, first, many, ring, cols);
    cols.leave(reinterpret_cast<float*>(ring), 0, kCols, S::kWide, r, c);
    __syncthreads();
    kv4_meet<NG, NT>(smem, S::kWarps, joined, S::kWide);
    cluster_sync_all();
    if (block == 0) blocks = ld_cluster_i32(mapa_u32(smem_u32(&blocks_here), 0));
    for (int col = rank + ctas * warp; col < kCols; col += ctas * S::kWarps) {
      if (col0 + col >= n_cols) break;
      const uint32_t at = smem_u32(joined + S::kCols * S::kWide + col);
      const uint32_t from = mapa_u32(at, min(lane, ctas - 1));
      float l = lane < ctas ? ld_cluster_f1(from + kCols * 4) : 0.f, m = l != 0.f ? ld_cluster_f1(from) : -INFINITY, all = m;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, x));
      const float f = l != 0.f ? exp2_fast(m - all) : 0.f;
      const uint32_t some = __ballot_sync(0xffffffffu, l != 0.f);
      l *= f;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      float2 v[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) v[g] = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int k = 0; k < ctas; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        if (!(some >> k & 1)) continue;
        const uint32_t part = mapa_u32(smem_u32(joined + col * S::kWide + 2 * lane), k);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float2 o2 = ld_cluster_f2(part + g * 256);
          v[g].x = fmaf(fk, o2.x, v[g].x);
          v[g].y = fmaf(fk, o2.y, v[g].y);
        }
      }
      const float inverse = l == 0.f ? 0.f : 1.f / l;
      const int token = p.group.of(col0 + col);
      __nv_bfloat16* out = p.out + ((int64_t)(s.row0 + token) * p.q_heads + head * p.group.d + col0 + col - token * p.group.d) * kDim;
#pragma unroll
      for (int g = 0; g < NG; ++g) *reinterpret_cast<uint32_t*>(out + g * 64 + 2 * lane) = pack2(v[g].x * inverse, v[g].y * inverse);
    }
    cluster_sync_all();   // nobody reads this CTA's part any more
  }
  kv4_others(p);
}

// ---- many columns to a sequence: a CTA takes 8·NT of them to a warp, all warps unpack a step's tokens once for all
template <int NG>
struct Prompt {
  static constexpr int kTile = kv4_tile_bytes(NG);
  static constexpr int kTiles = kStep / kKvTile;
  static constexpr int kStage = kTiles * kTile;
  static constexpr int kStages = 4;
  static constexpr int kNT = NG <= 2 ? 2 : 1;
  static constexpr int kWarps = 8, kPieces = 1;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCols = kWarps * 8 * kNT;
  static constexpr int kUnpacked = kTiles * 2 * NG * 4 * 512;   // of a step
  static constexpr bool kQInRegs = NG * kNT <= 4;
  static constexpr int kSmem = kStages * kStage + 2 * kUnpacked + walk_room(true);
};
template <int NG>
__global__ void __launch_bounds__(Prompt<NG>::kThreads, 1) kv4_prompt_kernel(const Kv4Attn p) {
  using S = Prompt<NG>;
  constexpr int NT = S::kNT, kDim = NG * 64;
  static_assert(S::kQInRegs, "queries in registers");
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  uint8_t* const ring = smem;
  uint4* const unpacked = reinterpret_cast<uint4*>(smem + S::kStages * S::kStage);
  pdl_wait();
  pdl_trigger();

  Walk<true> w{};
  w.template plan<S::kThreads>(p, S::kCols, reinterpret_cast<int*>(smem + S::kStages * S::kStage + 2 * S::kUnpacked));
  const Kv4Cut cut(w.line, 1);
  int at_line = cut.start(blockIdx.x);
  const int stop = cut.start(blockIdx.x + 1);
  if (threadIdx.x == 0) p.splits[blockIdx.x].from = -1;
  w.seek(p.n, at_line, stop);
  while (at_line < stop) {
    w.item(p, S::kCols, at_line);
    const Kv4Seq& s = w.s;
    const int first = max(at_line - w.begin, 0), many = min(stop, w.end) - w.begin - first;
    at_line = min(stop, w.end);
    if (many <= 0) continue;

    const int block0 = w.block * S::kCols, col0 = block0 + warp * 8 * NT, n_cols = s.count * p.group.d;
    uint4 q[NT][NG][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = col0 + t * 8 + r;
      const __nv_bfloat16* src = kv4_query<NG>(p, s, w.head, col, c);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) q[t][g][h] = col < n_cols ? *reinterpret_cast<const uint4*>(src + g * 64 + h * 32) : make_uint4(0, 0, 0, 0);
    }
    Columns<NG, NT> cols;
    cols.start(p, s, col0, n_cols, c);
    const bool some = col0 < n_cols;

    // steps that a column of the block sees
    const int step0 = s.step0 + first, high = s.pos + p.group.of(min(block0 + S::kCols, n_cols) - 1), low = s.pos + p.group.of(block0);
    const int begin = kv4_steps_begin(low, p.window, step0), end = kv4_steps_end(high, s.last, step0, many);
    const int32_t* table = p.cache.table + (int64_t)max(s.slot, 0) * p.cache.max_pages;
    auto page_of = [&](int u) {
      if (u >= end) return -1;
      const int page = table[(step0 + u) / (kPage / kStep)];
      return page < p.cache.n_pages ? page : -1;
    };
    auto fetch = [&](int u, int page) {
      if (page >= 0) {
        const uint8_t* src = kv4_head(p.cache, p.layer, page, w.head) + (step0 + u) % (kPage / kStep) * S::kStage;
        uint8_t* dst = ring + u % S::kStages * S::kStage;
        for (int b = threadIdx.x * 16; b < S::kStage; b += S::kThreads * 16) cp_async16(dst + b, src + b);
      }
      cp_async_commit();
    };
    // a warp unpacks whole groups of a tile's keys or values: the operands in the order in which a product takes them
    auto unpack = [&](int u) {
      const uint8_t* stage = ring + u % S::kStages * S::kStage;
      uint4* to = unpacked + u % 2 * (S::kUnpacked / 16);
      for (int e = warp; e < S::kTiles * 2 * NG; e += S::kWarps) {   // (tile, keys | values, group)
        const int k = e / (2 * NG), v = e / NG % 2, g = e % NG;
        const Nibbles n{*reinterpret_cast<const uint4*>(stage + k * S::kTile + v * NG * (512 + 64) + g * 512 + lane * 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
          n.values(j, a);
          to[(e * 4 + j) * 32 + lane] = make_uint4(a[0], a[1], a[2], a[3]);
        }
      }
    };
    uint32_t have = 0;   // bit u % 32: step u has a page
    for (int u = begin; u < begin + S::kStages - 2; ++u) {
      const int page = page_of(u);
      have |= (uint32_t)(page >= 0) << (u % 32);
      fetch(u, page);
    }
    int next = page_of(begin + S::kStages - 2);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int g = 0; g < NG; ++g) cols.take(g, t, q[t][g]);
    // Step u is unpacked one turn of the loop before its products, so that one barrier a turn does: behind it step u's raw bytes are there, the products of
    // u − 2 are done and the operands of u − 1 lie ready.
    for (int u = begin; u <= end; ++u) {
      const int ahead = u + S::kStages - 2;
      have = (have & ~(1u << (ahead % 32))) | (uint32_t)(next >= 0) << (ahead % 32);
      cp_async_wait<S::kStages - 3>();
      __syncthreads();
      fetch(ahead, next);
      next = page_of(ahead + 1);
      if (u < end) unpack(u);
      if (u == begin || !some) continue;
      const int v = u - 1, key0 = (step0 + v) * kStep;
      if (key0 > cols.at_high || (p.window > 0 && cols.at_low - key0 >= p.window + kStep - 1)) continue;   // nothing that this warp's columns see
      const uint8_t* stage = ring + v % S::kStages * S::kStage;
      const uint4* from = unpacked + v % 2 * (S::kUnpacked / 16) + lane;
      auto keys = [&](int k, int g) { return Unpacked{from + (k * 2 * NG + g) * 4 * 32}; };
      auto key_small = [&](int k, int g) { return *reinterpret_cast<const uint2*>(stage + k * S::kTile + NG * 512 + g * 64 + r * 8); };
      auto values = [&](int k, int g) { return Unpacked{from + (k * 2 * NG + NG + g) * 4 * 32}; };
      auto value_small = [&](int k, int g) { return *reinterpret_cast<const uint2*>(stage + k * S::kTile + NG * (512 + 64 + 512) + g * 64 + r * 8); };
      auto query = [&](int t, int g, int h) { return q[t][g][h]; };
      float sc[S::kTiles][NT][4];
      cols.scores(sc, keys, key_small, query);
      const bool whole = cols.mask(sc, key0, have >> (v % 32) & 1 ? s.last : 0, p.window, r);
      cols.settle(sc, p.scale_log2);
      if (whole) cols.template values<true>(sc, p.scale_log2, values, value_small);
      else cols.template values<false>(sc, p.scale_log2, values, value_small);
    }
    cp_async_wait<0>();
    __syncthreads();   // the ring and the operands are free
    cols.finish();
    if (many == s.steps) {
      cols.write(p, s, w.head, col0, n_cols, r, c);
    } else {
      if (first == 0 && threadIdx.x == 0) kv4_split(p, w, cut, blockIdx.x, blockIdx.x, block0, n_cols);
      if (some) cols.leave(kv4_part(p, blockIdx.x, first == 0, S::kCols), warp * 8 * NT, S::kCols, kDim, r, c);
    }
  }
  kv4_others(p);
}

// The items that lie in more than one piece of the line.  CTA (c, y) joins parts of those that begin in CTA c's pieces: a column to a warp while an item's parts are
// few, else a column to the CTA, its warps every eighth part in order, and then the warps meet.
constexpr int kJoinWarps = 8, kJoinRows = 16;
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
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, turns = gridDim.y * kJoinWarps;
  pdl_wait();
  pdl_trigger();
  const Kv4Split* splits = p.splits + blockIdx.x * warps;
  Kv4Split mine{};
  mine.from = -1;
  if (lane < warps) mine = splits[lane];
  auto of = [&](int v, int from) { return __shfl_sync(0xffffffffu, v, from); };
  int number = 0;   // of items that are joined a column to a warp
  for (uint32_t left = __ballot_sync(0xffffffffu, mine.from >= 0); left != 0; left &= left - 1) {
    const int i = __ffs(left) - 1;
    const Kv4Pieces pieces{of(mine.from, i), 0, of(mine.in0, i), of(mine.in1, i), of(mine.each, i), of(mine.before, i), of(mine.whole, i), 0};
    const int many = min(of(mine.n_cols, i) - of(mine.col0, i), columns);
    const int parts = of(mine.parts, i);
    const bool alone = parts <= 2 * kAtOnce;
    const int first = alone ? 0 : warp, step = alone ? 1 : kJoinWarps;
    // columns are dealt out in turn, over the items that a warp joins alone
    const int start = alone ? (blockIdx.y * kJoinWarps + warp + turns - number * columns % turns) % turns : blockIdx.y;
    if (alone) ++number;
    for (int col = start; col < many; col += alone ? turns : gridDim.y) {
    Joined<NG> o;
    for (int k0 = first; k0 < parts; k0 += kAtOnce * step) {
      float m[kAtOnce], l[kAtOnce];
      float2 x[kAtOnce][NG];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const int k = min(k0 + e * step, parts - 1), w = pieces.piece(k);
        const float* part = kv4_part(p, (int64_t)(w / pieces.each) * warps + w % pieces.each, k < pieces.before && k == 0, columns);
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
}

// How a call's rows are taken: by the columns that an average sequence brings.  Up to 8: a tile of columns to a warp; up to 32: two; more: a CTA for 128 (64 of heads
// of 192 and 256), which unpacks for all of them (257 rows of 16 / 8 heads of 128 under a window of 1 024: 32.0 µs, two tiles to a warp 36.7).
// Few columns over a small cache go to clusters: they save the second launch, and are worth it while a warp's share of the longest sequence that the cache can
// hold is no more than some three steps above what the even cut would give it (µs, clusters / even cut, one sequence of 24 / 8 heads of 128: 1 000 tokens
// 7.5 / 10.2, 4 000 9.0 / 10.9, 12 000 14.1 / 12.2; 14 / 2 heads of 64: 1 000 6.4 / 9.3, 4 000 7.0 / 10.2, 16 000 9.6 / 11.4; 32 / 4 heads of 128: 8 000 9.5 / 12.0,
// 32 768 17.2 / 15.0).  As large a cluster as the SMs hold all of at once: of 16 CTAs 7, of 8 15, of 4 33 (36 / 6 heads of 128, 12 000
// tokens: clusters of 16 11.0, of 10 13.0; 24 / 8 heads, 4 000 tokens, where eight clusters of 16 are two rounds: 15.9).  A cluster goes over its sequence's blocks of columns
// in turn, so both shares count once for every block of the sequence that may bring most rows, the others bringing one each (32 tokens beside a piece of 800 rows, 4 / 4 heads
// of 128 over 832 tokens: clusters 434, even cut 31).
// One way is taken for a whole call, by its average: a prompt's piece beside many single tokens is faster as two calls (µs, 32 / 8 heads of 128 over 4 000 tokens each: 512 rows beside 63
// tokens 850, apart 184 + 81).
struct Way {
  int tiles, columns, warps, cluster;   // tiles of a warp (0: the CTA's way), columns of a block, pieces of the line to a CTA; CTAs of a cluster (0: none)
};
Way kv4_way(int64_t group, int64_t n, int64_t rows, const b200_kv4_cache& cache) {
  const int64_t columns = group * ((rows + n - 1) / n), items = n * cache.kv_heads;
  if (columns > 32) return {0, cache.dim <= 128 ? 128 : 64, 1, 0};
  const int tiles = columns > 8 ? 2 : 1;
  int ctas = items <= 6 ? 16 : items <= 15 ? 8 : items <= 33 ? 4 : items <= 74 ? 2 : items <= kGrid ? 1 : 0;   // (that the SMs hold at once)
  const double steps = (double)cache.max_pages * (kPage / kStep);
  while (ctas > 1 && ctas / 2 * kPieceWarps >= steps) ctas /= 2;   // no more than a warp for every step
  const int64_t blocks = (group * std::max<int64_t>(rows - n + 1, 1) + 8 * tiles - 1) / (8 * tiles);
  if (ctas > 0 && (double)blocks * steps * (1.0 / (ctas * kPieceWarps) - (double)cache.kv_heads / (kGrid * kPieceWarps)) <= 3.2) return {tiles, 8 * tiles, 0, ctas};
  return {tiles, 8 * tiles, kPieceWarps, 0};
}

template <typename Shape, void (*kKernel)(Kv4Attn, int)>
int launch_cluster(const Kv4Attn& p, const Way& way, cudaStream_t st) {
  static PerDevice attrs;
  B200_CUDA(attrs([] {
    const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.n * p.kv_heads.d * way.cluster));
  cfg.blockDim = dim3(Shape::kThreads);
  cfg.dynamicSmemBytes = Shape::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)way.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = op_pdl(st) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  B200_CUDA(cudaLaunchKernelEx(&cfg, kKernel, p, way.cluster));
  return B200_OK;
}
template <typename Shape, void (*kKernel)(Kv4Attn), void (*kJoin)(Kv4Attn, int, int)>
int launch(const Kv4Attn& p, const Way& way, cudaStream_t st) {
  B200_CHECK_ARG(way.warps == Shape::kPieces && way.columns == Shape::kCols, "kv4_attention: the workspace is not this kernel's");
  static PerDevice attrs;
  B200_CUDA(attrs([] { return cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem); }));
  const bool pdl = op_pdl(st);
  B200_CUDA(launch_pdl(kKernel, dim3(kGrid), dim3(Shape::kThreads), Shape::kSmem, st, pdl, p));
  B200_CUDA(launch_pdl(kJoin, dim3(kGrid, std::min(way.columns, kJoinRows)), dim3(kJoinWarps * 32), 0, st, pdl, p, way.columns, way.warps));
  return B200_OK;
}
template <int NG>
int launch_groups(const Kv4Attn& p, const Way& way, cudaStream_t st) {
  if (way.cluster > 0)
    return way.tiles == 1 ? launch_cluster<Cluster<NG, 1>, kv4_cluster_kernel<NG, 1>>(p, way, st) : launch_cluster<Cluster<NG, 2>, kv4_cluster_kernel<NG, 2>>(p, way, st);
  if (way.tiles == 1) return launch<Shape<NG, 1>, kv4_attn_kernel<NG, 1>, kv4_join_kernel<NG>>(p, way, st);
  if (way.tiles == 2) return launch<Shape<NG, 2>, kv4_attn_kernel<NG, 2>, kv4_join_kernel<NG>>(p, way, st);
  return launch<Prompt<NG>, kv4_prompt_kernel<NG>, kv4_join_kernel<NG>>(p, way, st);
}
int64_t part_floats(const Way& way, int dim) { return (int64_t)kGrid * way.warps * 2 * way.columns * (dim + 2); }

}  // namespace

}  // namespace b200

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(const b200_kv4_cache* cache, int64_t q_heads, int64_t n, int64_t rows) {
  using namespace b200;
  if (cache == nullptr || cache->kv_heads < 1 || q_heads < 1 || q_heads % cache->kv_heads != 0 || n < 1 || rows < 1) return -1;
  if (cache->dim % kKvGroup != 0 || cache->dim < 64 || cache->dim > 256) return -1;
  const Way way = kv4_way(q_heads / cache->kv_heads, n, rows, *cache);
  return part_floats(way, cache->dim) * 4 + (int64_t)kGrid * way.warps * sizeof(Kv4Split);
}

int b200_kv4_attention(void* out, const void* q, int64_t ld_q, const b200_kv4_cache* cache, int64_t layer, int64_t q_heads, const int32_t* seqs,
                       const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows, float scale, int64_t window, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_attention")) != B200_OK) return rc;
  B200_CHECK_ARG(out && q, "kv4_attention: null pointer");
  B200_CHECK_ARG(q_heads >= 1 && q_heads <= 1 << 16 && q_heads % cache->kv_heads == 0, "kv4_attention: %lld query heads over %d", (long long)q_heads,
                 cache->kv_heads);
  B200_CHECK_ARG(aligned16(q, workspace, out) && ld_q % 8 == 0 && ld_q >= q_heads * cache->dim, "kv4_attention: q's rows must be 16-byte aligned and apart");
  B200_CHECK_ARG(scale > 0.f && scale < 1e30f && window >= 0, "kv4_attention: scale %g, window %lld", (double)scale, (long long)window);
  // the line of all work is counted in 32 bits: 1 M rows of 32 heads over 64 K tokens, or 64 K over 1 M
  const int64_t group = q_heads / cache->kv_heads;
  const Way way = kv4_way(group, n, rows, *cache);
  const int64_t columns = way.columns;
  const int64_t items = cache->kv_heads * std::min(rows * ((group + columns - 1) / columns), rows * group / columns + n);
  B200_CHECK_ARG(items * ((int64_t)cache->max_pages * (kPage / kStep) + kAhead) < 1ll << 31 && rows * q_heads < 1ll << 31,
                 "kv4_attention: %lld rows of %lld heads over %d pages are too many for one call", (long long)rows, (long long)q_heads, cache->max_pages);
  B200_CHECK_ARG(workspace || way.warps == 0, "kv4_attention: null workspace");
  Kv4Attn p{};
  p.cache = *cache;
  p.out = (__nv_bfloat16*)out;
  p.q = (const __nv_bfloat16*)q;
  p.ld_q = ld_q;
  p.seqs = seqs;
  p.starts = starts;
  p.pos = pos;
  p.parts = (float*)workspace;
  p.splits = (Kv4Split*)(p.parts + part_floats(way, cache->dim));
  p.layer = (int)layer;
  p.q_heads = (int)q_heads;
  p.group = Divisor((uint32_t)(q_heads / cache->kv_heads));
  p.kv_heads = Divisor((uint32_t)cache->kv_heads);
  p.n = (int)n;
  p.rows = (int)rows;
  p.window = window > INT32_MAX - 64 ? 0 : (int)window;   // positions end before that, so such a window masks nothing; and a step added to it stays in 32 bits
  p.scale_log2 = scale * 1.44269504f;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (cache->dim / kKvGroup) {
    case 1: return launch_groups<1>(p, way, st);
    case 2: return launch_groups<2>(p, way, st);
    case 3: return launch_groups<3>(p, way, st);
    default: return launch_groups<4>(p, way, st);
  }
}

}  // extern "C"
