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
  Kv4Place at;        // of lane's row row + lane
  uint32_t leads, nowhere;
};
// starts go through shared memory: the search would wait for memory with every step
template <int ROWS>
__device__ Job find_job(const b200_kv4_cache& cache, const int32_t* seqs, const int32_t* starts, const int32_t* pos, int n, int rows, int32_t* shared, bool owned) {
  for (int i = threadIdx.x; i <= n; i += kStoreWarps * 32) shared[i] = starts[i];
  __syncthreads();
  const int groups = cache.dim / kKvGroup, lane = threadIdx.x % 32;
  int job = blockIdx.y * kStoreWarps + threadIdx.x / 32;
  Job j{};
  j.row = blockIdx.x * ROWS;
  j.values = job % 2;
  j.group = job / 2 % groups;
  j.head = job / (2 * groups);
  j.at = {-1, 0, 0};
  const bool in = j.head < cache.kv_heads && lane < ROWS && j.row + lane < rows;
  if (in) j.at = kv4_place(cache, seqs, shared, pos, n, rows, j.row + lane);
  if (owned && j.at.page >= 0 && cache.refs[j.at.page] != 1) j.at.page = -1;
  j.leads = __ballot_sync(0xffffffffu, j.at.page >= 0 && j.at.run > 0);
  j.nowhere = __ballot_sync(0xffffffffu, in && j.at.page < 0);
  return j;
}

// Scale and middle of what `lo`, `hi` bound, and a value's nibble.
struct Scale {
  float s, m, inverse;
  uint32_t both;
};
__device__ __forceinline__ Scale make_scale(float lo, float hi, bool finite) {
  const __nv_bfloat16 s = f_to_bf16(hi / 15.f - lo / 15.f), m = f_to_bf16(fmaf(8.f, bf16_to_f(s), lo));
  if (!finite) return {0.f, 0.f, __uint_as_float(0x7fffffffu), 0x7fff7fffu};   // reads as NaN
  return {bf16_to_f(s), bf16_to_f(m), 1.f / bf16_to_f(s), (uint32_t)__bfloat16_as_ushort(s) | (uint32_t)__bfloat16_as_ushort(m) << 16};
}
// Eight values of a token in fp32, −8 … 7.  The quotient decides, rounded as a division rounds it; a product with the inverse is within 2^-20 of it, so that only
// what comes nearer than that to the middle between two values (or has an inverse that is none) is divided.
__device__ __noinline__ float exact_value(float d, float scale) { return scale > 0.f ? rintf(fminf(fmaxf(d / scale, -8.f), 7.f)) : 0.f; }
template <int N>
__device__ __forceinline__ void to_values(float (&x)[N], const Scale& sc) {
  constexpr float kMagic = 12582912.f;   // 1.5·2^23: a sum with it is rounded to a whole number
  bool close = !(sc.inverse < INFINITY);
  float d[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    d[i] = x[i] - sc.m;
    const float q = fminf(fmaxf(d[i] * sc.inverse, -8.f), 7.f);
    x[i] = (q + kMagic) - kMagic;
    close |= !(fabsf(q - x[i]) < 0.499998f);
  }
  if (close)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = exact_value(d[i], sc.s);
}
// a byte's two values, and a whole number below 65 536 from fp32
__device__ __forceinline__ float two_values(float first, float second) { return fmaf(16.f, second, first); }
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  constexpr float kMagic = 8388608.f + 8 * 4369;   // 2^23, and 8 for each of four values
  return __byte_perm(__float_as_uint(lo + kMagic), __float_as_uint(hi + kMagic), 0x5410);
}
__device__ __forceinline__ bool is_finite(uint32_t two) { return (two & 0x7f80u) != 0x7f80u && (two & 0x7f800000u) != 0x7f800000u; }

template <int ROWS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_store_kernel(const b200_kv4_cache cache, int layer, const __nv_bfloat16* k, int64_t ld_k,
                                                                     const __nv_bfloat16* v, int64_t ld_v, const int32_t* seqs, const int32_t* starts,
                                                                     const int32_t* pos, int n, int rows) {
  __shared__ int32_t shared[kKvMaxSeqs + 1];
  pdl_wait();
  pdl_trigger();
  const Job job = find_job<ROWS>(cache, seqs, starts, pos, n, rows, shared, true);
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, g = job.group, head = job.head, groups = cache.dim / kKvGroup;
  for (uint32_t left = job.leads; left != 0; left &= left - 1) {
    const int lead = __ffs(left) - 1, row = job.row + lead;
    const Kv4Place at{__shfl_sync(0xffffffffu, job.at.page, lead), __shfl_sync(0xffffffffu, job.at.token, lead), __shfl_sync(0xffffffffu, job.at.run, lead)};
    const int first = at.token % kKvTile;
    uint8_t* tile = kv4_head(cache, layer, at.page, head) + at.token / kKvTile * kv4_tile_bytes(groups) + job.values * groups * (512 + 64);
    uint32_t* small = reinterpret_cast<uint32_t*>(tile + groups * 512) + g * 16;
    uint8_t* mine = tile + g * 512 + lane * 16;
    float half[8];   // of the lane's four words
    if (job.values == 0) {   // keys: tokens r and r + 8, 16 entries of each
      const __nv_bfloat16* src = k + (int64_t)(row - first) * ld_k + head * cache.dim + g * kKvGroup + 8 * c;
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int token = r + 8 * hi;
        const bool here = token >= first && token < first + at.run;
        uint4 x[2];
        x[0] = x[1] = make_uint4(0, 0, 0, 0);
        if (here) {
          x[0] = *reinterpret_cast<const uint4*>(src + token * ld_k);
          x[1] = *reinterpret_cast<const uint4*>(src + token * ld_k + 32);
        }
        float f[16], lo, top;
        bool finite = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t two[4] = {x[h].x, x[h].y, x[h].z, x[h].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[8 * h + 2 * e] = bf16_lo(two[e]);
            f[8 * h + 2 * e + 1] = bf16_hi(two[e]);
            finite &= is_finite(two[e]);
          }
        }
        lo = top = f[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) {
          lo = fminf(lo, f[e]);
          top = fmaxf(top, f[e]);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          finite &= __shfl_xor_sync(0xffffffffu, (int)finite, o) != 0;
        }
        const Scale sc = make_scale(lo, top, finite);
        to_values(f, sc);
#pragma unroll
        for (int e = 0; e < 8; ++e) half[e] = hi == 0 ? two_values(f[2 * e], f[2 * e + 1]) : fmaf(256.f, two_values(f[2 * e], f[2 * e + 1]), half[e]);
        if (here && c == 0) small[r * 2 + hi] = sc.both;
      }
    } else {              // values: four tokens, eight entries of each
      const __nv_bfloat16* src = v + (int64_t)(row - first) * ld_v + head * cache.dim + g * kKvGroup + 2 * r;
#pragma unroll
      for (int b = 0; b < 4; ++b) {   // byte 2e + p of every word
        const int e = b / 2, p = b % 2, token = 2 * c + 8 * p + e;
        const bool here = token >= first && token < first + at.run;
        uint32_t two[4];
        bool finite = true;
        float lo = INFINITY, top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          two[j] = here ? *reinterpret_cast<const uint32_t*>(src + token * ld_v + 16 * j) : 0;
          finite &= is_finite(two[j]);
          lo = fminf(lo, fminf(bf16_lo(two[j]), bf16_hi(two[j])));
          top = fmaxf(top, fmaxf(bf16_lo(two[j]), bf16_hi(two[j])));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          finite &= __shfl_xor_sync(0xffffffffu, (int)finite, o) != 0;
        }
        const Scale sc = make_scale(lo, top, finite);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] = bf16_lo(two[j]);
          f[2 * j + 1] = bf16_hi(two[j]);
        }
        to_values(f, sc);
#pragma unroll
        for (int j = 0; j < 4; ++j) half[2 * j + e] = p == 0 ? two_values(f[2 * j], f[2 * j + 1]) : fmaf(256.f, two_values(f[2 * j], f[2 * j + 1]), half[2 * j + e]);
        if (here && r == 0) small[token % 8 * 2 + token / 8] = sc.both;
      }
    }
    const uint32_t words[4] = {halves(half[0], half[1]), halves(half[2], half[3]), halves(half[4], half[5]), halves(half[6], half[7])};
    if (at.run == kKvTile) {
      *reinterpret_cast<uint4*>(mine) = make_uint4(words[0], words[1], words[2], words[3]);
    } else {   // the bytes of the tokens that come
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int token = job.values == 0 ? r + 8 * (b % 2) : 2 * c + 8 * (b % 2) + b / 2;
        if (token >= first && token < first + at.run)
#pragma unroll
          for (int j = 0; j < 4; ++j) mine[4 * j + b] = (uint8_t)(words[j] >> (8 * b));
      }
    }
  }
}

template <int ROWS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_load_kernel(float* k, float* v, const b200_kv4_cache cache, int layer, const int32_t* seqs,
                                                                    const int32_t* starts, const int32_t* pos, int n, int rows) {
  __shared__ int32_t shared[kKvMaxSeqs + 1];
  pdl_wait();
  pdl_trigger();
  const Job job = find_job<ROWS>(cache, seqs, starts, pos, n, rows, shared, false);
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, g = job.group, head = job.head, groups = cache.dim / kKvGroup;
  const int64_t ld = (int64_t)cache.kv_heads * cache.dim;
  for (uint32_t left = job.nowhere; left != 0; left &= left - 1)
    *reinterpret_cast<float2*>((job.values ? v : k) + (job.row + __ffs(left) - 1) * ld + head * cache.dim + g * kKvGroup + 2 * lane) = make_float2(0.f, 0.f);
  for (uint32_t left = job.leads; left != 0; left &= left - 1) {
    const int lead = __ffs(left) - 1, row = job.row + lead;
    const Kv4Place at{__shfl_sync(0xffffffffu, job.at.page, lead), __shfl_sync(0xffffffffu, job.at.token, lead), __shfl_sync(0xffffffffu, job.at.run, lead)};
    const int first = at.token % kKvTile;
    const uint8_t* tile = kv4_head(cache, layer, at.page, head) + at.token / kKvTile * kv4_tile_bytes(groups) + job.values * groups * (512 + 64);
    const uint32_t* small = reinterpret_cast<const uint32_t*>(tile + groups * 512) + g * 16;
    const uint4 w = *reinterpret_cast<const uint4*>(tile + g * 512 + lane * 16);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    const int64_t from = (int64_t)(row - first) * ld + head * cache.dim + g * kKvGroup;
    if (job.values == 0) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int token = r + 8 * hi;
        if (token < first || token >= first + at.run) continue;
        const float s = bf16_lo(small[r * 2 + hi]), m = bf16_hi(small[r * 2 + hi]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // word 2h + t: four entries
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = fmaf(s, (float)(int)(words[j] >> (16 * (e / 2) + 8 * hi + 4 * (e % 2)) & 15) - 8.f, m);
          *reinterpret_cast<float4*>(k + from + token * ld + j / 2 * 32 + 8 * c + j % 2 * 4) = make_float4(o[0], o[1], o[2], o[3]);
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int token = 2 * c + b % 2 * 8 + b / 2;
        if (token < first || token >= first + at.run) continue;
        const uint32_t both = small[token % 8 * 2 + token / 8];
        const float s = bf16_lo(both), m = bf16_hi(both);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t byte = words[j] >> (8 * b);
          *reinterpret_cast<float2*>(v + from + token * ld + 16 * j + 2 * r) =
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
