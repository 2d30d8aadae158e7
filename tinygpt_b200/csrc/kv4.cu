// kv4.cu — rows into the paged cache of 4-bit keys and values and back (kv4.cuh has the layout).
#include "kv4.cuh"

namespace b200 {

namespace {

// A warp takes a head of a row, its keys and its values; a lane two entries of every group.
__global__ void __launch_bounds__(256) kv4_store_kernel(const b200_kv4_cache cache, int layer, const __nv_bfloat16* k, int64_t ld_k, const __nv_bfloat16* v,
                                                        int64_t ld_v, const int32_t* seqs, const int32_t* starts, const int32_t* pos, int n, int rows) {
  pdl_wait();
  pdl_trigger();
  const int64_t job = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32, head = (int)(job % cache.kv_heads);
  const int64_t row = job / cache.kv_heads;
  if (row >= rows) return;
  const Kv4Place at = kv4_place(cache, seqs, starts, pos, n, (int)row);
  if (at.page < 0 || cache.refs[at.page] != 1) return;
  const int groups = cache.dim / kKvGroup, in_tile = at.token % kKvTile;
  uint8_t* tile = kv4_head(cache, layer, at.page, head) + at.token / kKvTile * kv4_tile_bytes(groups);
  for (int kv = 0; kv < 2; ++kv) {
    const __nv_bfloat16* src = (kv ? v + row * ld_v : k + row * ld_k) + head * cache.dim;
    uint8_t* values = tile + kv * groups * (512 + 64);
    uint32_t* small = reinterpret_cast<uint32_t*>(values + groups * 512);
    for (int g = 0; g < groups; ++g) {
      const float x0 = bf16_to_f(src[g * kKvGroup + 2 * lane]), x1 = bf16_to_f(src[g * kKvGroup + 2 * lane + 1]);
      float lo = fminf(x0, x1), hi = fmaxf(x0, x1);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const bool finite = !__any_sync(0xffffffffu, !isfinite(x0) || !isfinite(x1));
      const __nv_bfloat16 sb = f_to_bf16(hi / 15.f - lo / 15.f);
      const float s = bf16_to_f(sb);
      const __nv_bfloat16 mb = f_to_bf16(fmaf(8.f, s, lo));
      const float m = bf16_to_f(mb);
      const bool some = finite && s > 0.f;
      const uint32_t q0 = some ? 8 + (int)fminf(fmaxf(rintf((x0 - m) / s), -8.f), 7.f) : 8;
      const uint32_t q1 = some ? 8 + (int)fminf(fmaxf(rintf((x1 - m) / s), -8.f), 7.f) : 8;
      if (kv == 0) {   // entries d and d + 2 share a byte: this lane's and its neighbour's
        const bool odd = lane & 1;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? q0 : q1, 1);
        const int h = lane / 16, c = lane / 4 % 4, t = lane / 2 % 2;
        values[g * 512 + (in_tile % 8 * 4 + c) * 16 + (2 * h + t) * 4 + 2 * odd + in_tile / 8] = (uint8_t)(odd ? other | q1 << 4 : q0 | other << 4);
      } else {         // entries d and d + 8
        const bool upper = lane & 4;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, upper ? q0 : q1, 4);
        const int d = 2 * (lane & ~4) + upper, c = in_tile % 8 / 2;
        values[g * 512 + (d % 8 * 4 + c) * 16 + d / 16 * 4 + 2 * (in_tile % 2) + in_tile / 8] = (uint8_t)(upper ? other | q1 << 4 : q0 | other << 4);
      }
      if (lane == 0) {
        const uint32_t both = (uint32_t)__bfloat16_as_ushort(sb) | (uint32_t)__bfloat16_as_ushort(mb) << 16;
        small[g * 16 + in_tile % 8 * 2 + in_tile / 8] = finite ? both : 0x7fff7fffu;
      }
    }
  }
}

__global__ void __launch_bounds__(256) kv4_load_kernel(float* k, float* v, const b200_kv4_cache cache, int layer, const int32_t* seqs,
                                                       const int32_t* starts, const int32_t* pos, int n, int rows) {
  pdl_wait();
  pdl_trigger();
  const int64_t job = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32, head = (int)(job % cache.kv_heads);
  const int64_t row = job / cache.kv_heads;
  if (row >= rows) return;
  const Kv4Place at = kv4_place(cache, seqs, starts, pos, n, (int)row);
  const int groups = cache.dim / kKvGroup, in_tile = at.token % kKvTile;
  const uint8_t* tile = at.page < 0 ? nullptr : kv4_head(cache, layer, at.page, head) + at.token / kKvTile * kv4_tile_bytes(groups);
  for (int kv = 0; kv < 2; ++kv) {
    float* dst = (kv ? v : k) + job * cache.dim;
    const uint8_t* values = tile + kv * groups * (512 + 64);
    const uint32_t* small = reinterpret_cast<const uint32_t*>(values + groups * 512);
    for (int g = 0; g < groups; ++g) {
      float2 o = make_float2(0.f, 0.f);
      if (tile != nullptr) {
        const uint32_t both = small[g * 16 + in_tile % 8 * 2 + in_tile / 8];
        const float s = bf16_lo(both), m = bf16_hi(both);
        uint32_t q[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = 2 * lane + e;
          const uint8_t* b = kv == 0 ? values + g * 512 + (in_tile % 8 * 4 + d / 8 % 4) * 16 + (2 * (d / 32) + d / 4 % 2) * 4 + 2 * (d % 2) + in_tile / 8
                                     : values + g * 512 + (d % 8 * 4 + in_tile % 8 / 2) * 16 + d / 16 * 4 + 2 * (in_tile % 2) + in_tile / 8;
          q[e] = (kv == 0 ? d / 2 % 2 : d / 8 % 2) ? *b >> 4 : *b & 15;
        }
        o = make_float2(fmaf(s, (float)((int)q[0] - 8), m), fmaf(s, (float)((int)q[1] - 8), m));
      }
      *reinterpret_cast<float2*>(dst + g * kKvGroup + 2 * lane) = o;
    }
  }
}

}  // namespace

int check_kv4(const b200_kv4_cache* c, const char* what) {
  B200_CHECK_ARG(c && c->pages && c->table && c->length && c->refs, "%s: null pointer in the cache", what);
  B200_CHECK_ARG(c->layers >= 1 && c->n_pages >= 1 && c->n_seqs >= 1 && c->max_pages >= 1 && c->max_pages <= 1 << 24 && c->kv_heads >= 1 &&
                     c->kv_heads <= 1 << 16,
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
  if (kv_heads < 1 || kv_heads > 1 << 16 || dim < 64 || dim > 256 || dim % 64 != 0) return -1;
  return kv_heads * 4 * b200::kv4_tile_bytes((int)dim / b200::kKvGroup);
}

int b200_kv4_store(const b200_kv4_cache* cache, int64_t layer, const void* k, int64_t ld_k, const void* v, int64_t ld_v, const int32_t* seqs,
                   const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_store")) != B200_OK) return rc;
  B200_CHECK_ARG(k && v && ld_k >= (int64_t)cache->kv_heads * cache->dim && ld_v >= (int64_t)cache->kv_heads * cache->dim, "kv4_store: k / v rows overlap");
  const unsigned grid = (unsigned)((rows * cache->kv_heads + 7) / 8);
  const cudaStream_t st = (cudaStream_t)stream;
  B200_CUDA(launch_pdl(kv4_store_kernel, dim3(grid), dim3(256), 0, st, op_pdl(st), *cache, (int)layer, (const __nv_bfloat16*)k, ld_k,
                       (const __nv_bfloat16*)v, ld_v, seqs, starts, pos, (int)n, (int)rows));
  return B200_OK;
}

int b200_kv4_load(float* k, float* v, const b200_kv4_cache* cache, int64_t layer, const int32_t* seqs, const int32_t* starts, const int32_t* pos,
                  int64_t n, int64_t rows, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4_rows(cache, layer, seqs, starts, pos, n, rows, "kv4_load")) != B200_OK) return rc;
  B200_CHECK_ARG(k && v && aligned16(k, v), "kv4_load: k and v must be 16-byte aligned");
  const unsigned grid = (unsigned)((rows * cache->kv_heads + 7) / 8);
  const cudaStream_t st = (cudaStream_t)stream;
  B200_CUDA(launch_pdl(kv4_load_kernel, dim3(grid), dim3(256), 0, st, op_pdl(st), k, v, *cache, (int)layer, seqs, starts, pos, (int)n, (int)rows));
  return B200_OK;
}

}  // extern "C"
