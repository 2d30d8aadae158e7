// kv4.cu — rows into the paged cache of 4-bit keys and values and back (kv4.cuh has the layout).
#include "kv4.cuh"

namespace b200 {

namespace {

// A warp takes the keys or the values of a group of a head, of kRows rows; a CTA has eight such.  The rows that go to one tile of 16 tokens are a run, which the
// warp with its first row deals with: it has the whole tile in registers in the layout of the cache, and where all 16 tokens come stores it with 16
// bytes a lane.  kRows is 16 for prompts, and 1 where most sequences bring few rows, whose warps then wait for memory side by side.
constexpr int kStoreWarps = 8;

struct Job {
  int row, head, group, values;
  Kv4Place place;     // of row row + lane
  uint32_t leads, nowhere;
};
// Up to 32 sequences: a lane has each, so that all a row needs is there after one wait for memory.  More: starts go through shared memory, where the search is.
template <int ROWS>
__device__ Job find_job(const b200_kv4_cache& cache, const int32_t* seqs, const int32_t* starts, const int32_t* pos, int n, int rows, int32_t* shared) {
  const int groups = cache.dim / kKvGroup, lane = threadIdx.x % 32, job = blockIdx.y * kStoreWarps + threadIdx.x / 32;
  Job j{};
  j.row = blockIdx.x * ROWS;
  j.values = job % 2;
  j.group = job / 2 % groups;
  j.head = job / (2 * groups);
  j.place = {-1, 0, 0};
  const int row = j.row + lane;
  const bool in = j.head < cache.kv_heads && lane < ROWS && row < rows;
  int i = 0, slot, at, first, end;   // the last i with starts[i] <= row
  if (n <= 32) {
    const int my_start = lane < n ? starts[lane] : INT32_MAX, my_slot = lane < n ? seqs[lane] : -1, my_pos = lane < n ? pos[lane] : -1, last = starts[n];
    for (int s = 1; s < n; ++s) i = __shfl_sync(0xffffffffu, my_start, s) <= row ? s : i;
    slot = __shfl_sync(0xffffffffu, my_slot, i);
    at = __shfl_sync(0xffffffffu, my_pos, i);
    first = __shfl_sync(0xffffffffu, my_start, i);
    end = __shfl_sync(0xffffffffu, my_start, min(i + 1, 31));
    if (i + 1 == n) end = last;
  } else {
    for (int s = threadIdx.x; s <= n; s += kStoreWarps * 32) shared[s] = starts[s];
    __syncthreads();
    int hi = n;
    while (hi - i > 1) {
      const int mid = (i + hi) / 2;
      if (shared[mid] <= row) i = mid;
      else hi = mid;
    }
    slot = seqs[i];
    at = pos[i];
    first = shared[i];
    end = shared[i + 1];
  }
  if (in) j.place = kv4_place(cache, slot, at, first, min(end, rows), row);
  j.leads = __ballot_sync(0xffffffffu, j.place.slot >= 0 && j.place.run > 0);
  j.nowhere = __ballot_sync(0xffffffffu, in && j.place.slot < 0);
  return j;
}

// The greatest of a token's entries and of their negatives, two bf16 side by side: lanes' words first, then the lanes' halves.  NaN stays.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
constexpr uint32_t kNegate = 0x80008000u;
template <int N>
__device__ __forceinline__ uint32_t extremes(const uint32_t* two) {   // {greatest, greatest negative} of N words
  uint32_t top = two[0], low = two[0] ^ kNegate;
#pragma unroll
  for (int i = 1; i < N; ++i) {
    top = max2(top, two[i]);
    low = max2(low, two[i] ^ kNegate);
  }
  return max2(__byte_perm(top, low, 0x5410), __byte_perm(top, low, 0x7632));
}

// Scale and middle of a group with these extremes.
struct Scale {
  float s, m, inverse;
  uint32_t both;
};
__device__ __forceinline__ Scale make_scale(uint32_t ends) {
  const float hi = bf16_lo(ends), lo = -bf16_hi(ends);
  const __nv_bfloat16 s = f_to_bf16(hi / 15.f - lo / 15.f), m = f_to_bf16(fmaf(8.f, bf16_to_f(s), lo));
  if (!isfinite(hi) || !isfinite(lo)) return {0.f, 0.f, 0.f, 0x7fff7fffu};   // reads as NaN
  return {bf16_to_f(s), bf16_to_f(m), bf16_to_f(s) > 0.f ? 1.f / bf16_to_f(s) : 0.f, (uint32_t)__bfloat16_as_ushort(s) | (uint32_t)__bfloat16_as_ushort(m) << 16};
}

// N words of two entries → 2N nibbles (value + 8), each in the low bits of a whole number whose next bits up to 16 are zero.  The quotient by the scale decides,
// rounded as a division rounds it: the product with the (rounded) inverse and one step of Markstein's correction by the exact remainder give just that
// as long as nothing underflows, in three instructions; ties are common, since entries, middles and scales have eight bits each.  Scales that are next to
// nothing are divided by.
constexpr float kRound = 12582912.f + 8.f;   // 1.5·2^23: a sum with it is rounded to a whole number
__device__ __noinline__ float exact_value(float d, float scale) { return fminf(fmaxf(d / scale, -8.f), 7.f); }
template <int N>
__device__ __forceinline__ void to_nibbles(uint32_t (&out)[2 * N], const uint32_t* two, const Scale& sc) {
  const bool tiny = sc.s > 0.f && sc.s < 0x1p-100f;
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) {
    const float d = (i % 2 ? bf16_hi(two[i / 2]) : bf16_lo(two[i / 2])) - sc.m, q = d * sc.inverse;
    out[i] = __float_as_uint(fminf(fmaxf(fmaf(fmaf(-q, sc.s, d), sc.inverse, q), -8.f), 7.f) + kRound);
  }
  if (tiny)
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) out[i] = __float_as_uint(exact_value((i % 2 ? bf16_hi(two[i / 2]) : bf16_lo(two[i / 2])) - sc.m, sc.s) + kRound);
}

// Five CTAs to an SM, in 48 registers, which spills 132 bytes: 3 049 rows of 8 heads of 128 are stored in 10.7 µs and stored and read back in 18.8; four (64 registers, 56 bytes) take 11.1
// and 19.7, six (40, 264) 12.0 and 20.4.  There the issue slots are busy for 64 % of the cycles and the ALU for 47; 32 768 rows take 73 µs (79 and 60 %): instructions, then.
template <int ROWS>
__global__ void __launch_bounds__(kStoreWarps * 32, 5) kv4_store_kernel(const b200_kv4_cache cache, int layer, const __nv_bfloat16* k, int64_t ld_k,
                                                                     const __nv_bfloat16* v, int64_t ld_v, const int32_t* seqs, const int32_t* starts,
                                                                     const int32_t* pos, int n, int rows) {
  __shared__ int32_t shared[kKvMaxSeqs + 1];
  pdl_wait();
  pdl_trigger();
  const Job job = find_job<ROWS>(cache, seqs, starts, pos, n, rows, shared);
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, g = job.group, head = job.head, groups = cache.dim / kKvGroup;
  for (uint32_t left = job.leads; left != 0; left &= left - 1) {
    const int lead = __ffs(left) - 1, row = job.row + lead;
    const Kv4Place to{__shfl_sync(0xffffffffu, job.place.slot, lead), __shfl_sync(0xffffffffu, job.place.at, lead), __shfl_sync(0xffffffffu, job.place.run, lead)};
    const int first = to.at % kKvTile;
    auto here = [&](int token) { return token >= first && token < first + to.run; };
    // the rows, while the page is looked up
    uint32_t x[16];
    if (job.values == 0) {   // keys: of tokens r and r + 8 the entries {0 … 7, 32 … 39} + 8c
      const __nv_bfloat16* src = k + (int64_t)(row - first) * ld_k + head * cache.dim + g * kKvGroup + 8 * c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int token = r + e / 2 * 8;
        const uint4 w = here(token) ? *reinterpret_cast<const uint4*>(src + token * ld_k + e % 2 * 32) : make_uint4(0, 0, 0, 0);
        x[4 * e] = w.x;
        x[4 * e + 1] = w.y;
        x[4 * e + 2] = w.z;
        x[4 * e + 3] = w.w;
      }
    } else {                 // values: of tokens 2c + {0, 8, 1, 9} the entries 16j + 2r + {0, 1}
      const __nv_bfloat16* src = v + (int64_t)(row - first) * ld_v + head * cache.dim + g * kKvGroup + 2 * r;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int token = 2 * c + b % 2 * 8 + b / 2;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * b + j] = here(token) ? *reinterpret_cast<const uint32_t*>(src + token * ld_v + 16 * j) : 0;
      }
    }
    const int page = kv4_page(cache, to.slot, to.at);
    const int owners = page >= 0 ? cache.refs[page] : 0;   // (asked for here, looked at when there is something to store)
    uint8_t* tile = kv4_head(cache, layer, max(page, 0), head) + to.at % kPage / kKvTile * kv4_tile_bytes(groups) + job.values * groups * (512 + 64);
    uint32_t* small = reinterpret_cast<uint32_t*>(tile + groups * 512) + g * 16;
    uint8_t* mine = tile + g * 512 + lane * 16;
    uint32_t half[8], both[4];   // the lane's four words, 16 bits each; its tokens' scales and middles
    if (job.values == 0) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        uint32_t ends = extremes<8>(x + 8 * hi), q[16];
        ends = max2(ends, __shfl_xor_sync(0xffffffffu, ends, 1));
        ends = max2(ends, __shfl_xor_sync(0xffffffffu, ends, 2));
        const Scale sc = make_scale(ends);
        to_nibbles<8>(q, x + 8 * hi, sc);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t byte = q[2 * e] + 16 * q[2 * e + 1];
          half[e] = hi == 0 ? byte : half[e] + 256 * byte;
        }
        both[hi] = sc.both;
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {   // byte 2e + p of every word
        const int e = b / 2, p = b % 2, token = 2 * c + 8 * p + e;
        uint32_t ends = extremes<4>(x + 4 * b), q[8];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) ends = max2(ends, __shfl_xor_sync(0xffffffffu, ends, o));
        const Scale sc = make_scale(ends);
        to_nibbles<4>(q, x + 4 * b, sc);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t byte = q[2 * j] + 16 * q[2 * j + 1];
          half[2 * j + e] = p == 0 ? byte : half[2 * j + e] + 256 * byte;
        }
        both[b] = sc.both;
      }
    }
    if (owners != 1) continue;
    if (job.values == 0) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
        if (here(r + 8 * hi) && c == 0) small[r * 2 + hi] = both[hi];
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int token = 2 * c + 8 * (b % 2) + b / 2;
        if (here(token) && r == 0) small[token % 8 * 2 + token / 8] = both[b];
      }
    }
    uint32_t words[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) words[j] = __byte_perm(half[2 * j], half[2 * j + 1], 0x5410);
    if (to.run == kKvTile) {
      *reinterpret_cast<uint4*>(mine) = make_uint4(words[0], words[1], words[2], words[3]);
    } else {   // the bytes of the tokens that come
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (here(job.values == 0 ? r + 8 * (b % 2) : 2 * c + 8 * (b % 2) + b / 2))
#pragma unroll
          for (int j = 0; j < 4; ++j) mine[4 * j + b] = (uint8_t)(words[j] >> (8 * b));
    }
  }
}

template <int ROWS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_load_kernel(float* k, float* v, const b200_kv4_cache cache, int layer, const int32_t* seqs,
                                                                    const int32_t* starts, const int32_t* pos, int n, int rows) {
  __shared__ int32_t shared[kKvMaxSeqs + 1];
  pdl_wait();
  pdl_trigger();
  const Job job = find_job<ROWS>(cache, seqs, starts, pos, n, rows, shared);
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, g = job.group, head = job.head, groups = cache.dim / kKvGroup;
  const int64_t ld = (int64_t)cache.kv_heads * cache.dim;
  float* const out = (job.values ? v : k) + head * cache.dim + g * kKvGroup;
  for (uint32_t left = job.nowhere; left != 0; left &= left - 1)
    *reinterpret_cast<float2*>(out + (job.row + __ffs(left) - 1) * ld + 2 * lane) = make_float2(0.f, 0.f);
  for (uint32_t left = job.leads; left != 0; left &= left - 1) {
    const int lead = __ffs(left) - 1, row = job.row + lead;
    const Kv4Place from{__shfl_sync(0xffffffffu, job.place.slot, lead), __shfl_sync(0xffffffffu, job.place.at, lead), __shfl_sync(0xffffffffu, job.place.run, lead)};
    const int first = from.at % kKvTile, page = kv4_page(cache, from.slot, from.at);
    if (page < 0) {
      for (int t = 0; t < from.run; ++t) *reinterpret_cast<float2*>(out + (row + t) * ld + 2 * lane) = make_float2(0.f, 0.f);
      continue;
    }
    float* const dst = out + (int64_t)(row - first) * ld;
    const uint8_t* tile = kv4_head(cache, layer, page, head) + from.at % kPage / kKvTile * kv4_tile_bytes(groups) + job.values * groups * (512 + 64);
    const uint32_t* small = reinterpret_cast<const uint32_t*>(tile + groups * 512) + g * 16;
    const uint4 w = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    if (job.values == 0) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int token = r + 8 * hi;
        if (token < first || token >= first + from.run) continue;
        const float s = bf16_lo(small[r * 2 + hi]), m = bf16_hi(small[r * 2 + hi]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // word 2h + t: four entries
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = fmaf(s, (float)(int)(words[j] >> (16 * (e / 2) + 8 * hi + 4 * (e % 2)) & 15) - 8.f, m);
          *reinterpret_cast<float4*>(dst + token * ld + j / 2 * 32 + 8 * c + j % 2 * 4) = make_float4(o[0], o[1], o[2], o[3]);
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int token = 2 * c + b % 2 * 8 + b / 2;
        if (token < first || token >= first + from.run) continue;
        const uint32_t both = small[token % 8 * 2 + token / 8];
        const float s = bf16_lo(both), m = bf16_hi(both);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t byte = words[j] >> (8 * b);
          *reinterpret_cast<float2*>(dst + token * ld + 16 * j + 2 * r) =
              make_float2(fmaf(s, (float)(int)(byte & 15) - 8.f, m), fmaf(s, (float)(int)(byte >> 4 & 15) - 8.f, m));
        }
      }
    }
  }
}

int rows_of_a_warp(int64_t n, int64_t rows) { return rows <= 4 * n ? 1 : 16; }
dim3 store_grid(const b200_kv4_cache& c, int64_t rows, int per) {
  return dim3((unsigned)((rows + per - 1) / per), (unsigned)((c.kv_heads * (c.dim / kKvGroup) * 2 + kStoreWarps - 1) / kStoreWarps));
}

}  // namespace

int check_kv4(const b200_kv4_cache* c, const char* what) {
  B200_CHECK_ARG(c && c->pages && c->table && c->length && c->refs, "%s: null pointer in the cache", what);
  B200_CHECK_ARG(c->layers >= 1 && c->n_pages >= 1 && c->n_seqs >= 1 && c->max_pages >= 1 && c->max_pages <= 1 << 24 && c->kv_heads >= 1 &&
                     c->kv_heads <= 65535,
                 "%s: cache of %d layers, %d pages, %d sequences of %d pages, %d heads", what, c->layers, c->n_pages, c->n_seqs, c->max_pages, c->kv_heads);
  B200_CHECK_ARG(c->dim % kKvGroup == 0 && c->dim >= 64 && c->dim <= 256, "%s: heads of %d (64, 128, 192 or 256)", what, c->dim);
  B200_CHECK_ARG(aligned16(c->pages), "%s: pages must be 16-byte aligned", what);
  return B200_OK;
}

int check_kv4_rows(const b200_kv4_cache* c, int64_t layer, const int32_t* seqs, const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows,
                   const char* what) {
  const int rc = check_kv4(c, what);
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(layer >= 0 && layer < c->layers, "%s: layer %lld of %d", what, (long long)layer, c->layers);
  B200_CHECK_ARG(seqs && starts && pos && n >= 1 && n <= kKvMaxSeqs, "%s: %lld sequences (1 … %d), or a null pointer", what, (long long)n, kKvMaxSeqs);
  B200_CHECK_ARG(rows >= 1 && rows <= 1 << 24, "%s: %lld rows", what, (long long)rows);
  return B200_OK;
}

}  // namespace b200

extern "C" {

int64_t b200_kv4_page_bytes(int64_t kv_heads, int64_t dim) {
  if (kv_heads < 1 || kv_heads > 65535 || dim < 64 || dim > 256 || dim % 64 != 0) return -1;
  return kv_heads * 4 * b200::kv4_tile_bytes((int)dim / b200::kKvGroup);
}

int b200_kv4_store(const b200_kv4_cache* cache, int64_t layer, const void* k, int64_t ld_k, const void* v, int64_t ld_v, const int32_t* seqs,
                   const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_store")) != B200_OK) return rc;
  B200_CHECK_ARG(k && v && ld_k >= (int64_t)cache->kv_heads * cache->dim && ld_v >= (int64_t)cache->kv_heads * cache->dim, "kv4_store: k / v rows overlap");
  B200_CHECK_ARG(aligned16(k, v) && ld_k % 8 == 0 && ld_v % 8 == 0, "kv4_store: k's and v's rows must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const int per = rows_of_a_warp(n, rows);
  B200_CUDA(launch_pdl(per == 1 ? kv4_store_kernel<1> : kv4_store_kernel<16>, store_grid(*cache, rows, per), dim3(kStoreWarps * 32), 0, st, op_pdl(st), *cache, (int)layer, (const __nv_bfloat16*)k, ld_k,
                       (const __nv_bfloat16*)v, ld_v, seqs, starts, pos, (int)n, (int)rows));
  return B200_OK;
}

int b200_kv4_load(float* k, float* v, const b200_kv4_cache* cache, int64_t layer, const int32_t* seqs, const int32_t* starts, const int32_t* pos,
                  int64_t n, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_load")) != B200_OK) return rc;
  B200_CHECK_ARG(k && v && aligned16(k, v), "kv4_load: k and v must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const int per = rows_of_a_warp(n, rows);
  B200_CUDA(launch_pdl(per == 1 ? kv4_load_kernel<1> : kv4_load_kernel<16>, store_grid(*cache, rows, per), dim3(kStoreWarps * 32), 0, st, op_pdl(st), k, v, *cache, (int)layer, seqs, starts, pos, (int)n, (int)rows));
  return B200_OK;
}

}  // extern "C"
