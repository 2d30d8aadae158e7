// kv4_pages.cu — who owns the pages of the cache: growing, forking, freeing and compacting sequences, all on the device.
//
// A call is one CTA that plans (checks, prefix sums, the lowest free pages in order) and, where pages are copied, a second kernel over all SMs.  Nothing
// depends on the order in which threads run: page k of a call is the k-th free page, references are counted with integer atomics.
#include "kv4.cuh"

#include <algorithm>

namespace b200 {

namespace {

// Threads of a planning CTA: a sequence of the call each, and kEach pages at a time.  Small calls over small pools take the small one, whose barriers and
// launch cost less (µs, 1 024 / 256 threads, 8 sequences over 384 pages: fork 7.3 / 5.8, extend 4.4 / 3.3).
constexpr int kMany = kKvMaxSeqs, kFew = 256, kEach = 8;
inline bool few(int64_t n, int n_pages) { return n <= kFew && n_pages <= 2 * kFew * kEach; }
constexpr int kCopy = 4 * 256 * 16;   // bytes of a page that a CTA copies at a time

// Sums up to and with every thread's; `total` of all.  All threads of a planning CTA.
template <int THREADS>
__device__ __forceinline__ long long scan_block(long long v, long long* total) {
  __shared__ long long warps[THREADS / 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long b = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += b;
  }
  __syncthreads();   // what an earlier scan left has been read
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  long long w = lane < THREADS / 32 ? warps[lane] : 0, mine = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long b = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += b;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  return v + __shfl_sync(0xffffffffu, w - mine, warp);
}

// The first pages that `pick` takes, in order, until there are `want` or no more: list[k]; how many.  All threads of a planning CTA.
template <int THREADS, typename Pick>
__device__ __forceinline__ int list_pages(int n_pages, long long want, int32_t* list, Pick pick) {
  long long found = 0;
  for (int64_t base = 0; base < n_pages && found < want; base += kEach * THREADS) {
    const int64_t first = base + kEach * threadIdx.x;
    bool is[kEach];
    int mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      is[e] = first + e < n_pages && pick((int)(first + e));
      mine += is[e];
    }
    long long total;
    long long at = found + scan_block<THREADS>(mine, &total) - mine;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (is[e]) list[at++] = (int32_t)(first + e);
    found += total;
  }
  __syncthreads();
  return (int)found;
}

// whether seqs[i] names a sequence and has not stood before i
__device__ bool first_mention(const int32_t* seqs, int i, int n_seqs) {
  const int s = seqs[i];
  if (s < 0 || s >= n_seqs) return false;
  for (int j = 0; j < i; ++j)
    if (seqs[j] == s) return false;
  return true;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv4_extend_kernel(const b200_kv4_cache c, const int32_t* seqs_in, const int32_t* counts, int32_t* pos, int n,
                                                           int32_t* list) {
  __shared__ int32_t seqs[THREADS];
  __shared__ int have[THREADS], granted[THREADS];
  __shared__ long long start[THREADS];
  pdl_wait();
  pdl_trigger();
  const int i = threadIdx.x;
  if (i < n) seqs[i] = seqs_in[i];
  __syncthreads();
  bool ok = i < n && first_mention(seqs, i, c.n_seqs);
  const int count = ok ? counts[i] : 0, length = ok ? c.length[seqs[i]] : 0;
  const long long want = ((long long)length + count + kPage - 1) / kPage;
  ok = ok && count >= 0 && want <= c.max_pages;
  have[i] = (length + kPage - 1) / kPage;
  const long long need = ok ? want - have[i] : 0;
  long long total;
  const long long end = scan_block<THREADS>(need, &total);
  const int free_pages = list_pages<THREADS>(c.n_pages, total, list, [&](int p) { return c.refs[p] == 0; });
  ok = ok && (need == 0 || end <= free_pages);
  granted[i] = ok ? (int)need : 0;
  start[i] = end - need;
  if (i < n) {
    pos[i] = ok ? length : -1;
    if (ok) c.length[seqs[i]] = length + count;
  }
  __syncthreads();
  for (int j = threadIdx.x / 32; j < n; j += THREADS / 32)
    for (int e = threadIdx.x % 32; e < granted[j]; e += 32) {
      const int page = list[start[j] + e];
      c.table[(int64_t)seqs[j] * c.max_pages + have[j] + e] = page;
      c.refs[page] = 1;
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv4_fork_kernel(const b200_kv4_cache c, const int32_t* src_in, const int32_t* dst_in, int32_t* done, int n,
                                                         int32_t* list, int2* copies) {
  __shared__ int32_t src[THREADS], dst[THREADS];
  __shared__ int whole[THREADS], own[THREADS];
  pdl_wait();
  pdl_trigger();
  const int i = threadIdx.x;
  if (i < n) {
    src[i] = src_in[i];
    dst[i] = dst_in[i];
  }
  __syncthreads();
  bool ok = i < n && src[i] >= 0 && src[i] < c.n_seqs && src[i] != dst[i] && first_mention(dst, i, c.n_seqs) && c.length[dst[i]] == 0;
  const int length = ok ? c.length[src[i]] : 0;
  ok = ok && (length + kPage - 1) / kPage <= c.max_pages;
  const int need = ok && length % kPage != 0;
  long long total;
  const long long end = scan_block<THREADS>(need, &total);
  const int free_pages = list_pages<THREADS>(c.n_pages, total, list, [&](int p) { return c.refs[p] == 0; });
  ok = ok && (need == 0 || end <= free_pages);
  whole[i] = ok ? length / kPage : -1;
  own[i] = ok && need ? list[end - 1] : -1;
  __syncthreads();   // every length and every free page has been read
  if (i < n) {
    done[i] = ok;
    int2 copy = make_int2(-1, -1);
    if (ok) c.length[dst[i]] = length;
    if (own[i] >= 0) {
      copy = make_int2(c.table[(int64_t)src[i] * c.max_pages + whole[i]], own[i]);
      if (copy.x < 0 || copy.x >= c.n_pages) copy = make_int2(-1, -1);
      c.table[(int64_t)dst[i] * c.max_pages + whole[i]] = own[i];
      c.refs[own[i]] = 1;
    }
    copies[i] = copy;
  }
  for (int j = threadIdx.x / 32; j < n; j += THREADS / 32)
    for (int e = threadIdx.x % 32; e < whole[j]; e += 32) {
      const int page = c.table[(int64_t)src[j] * c.max_pages + e];
      c.table[(int64_t)dst[j] * c.max_pages + e] = page;
      if (page >= 0 && page < c.n_pages) atomicAdd(c.refs + page, 1);
    }
}

__device__ __forceinline__ void copy_part(const b200_kv4_cache& c, int64_t page_bytes, int layer, int from, int to, int part) {
  const uint4* src = reinterpret_cast<const uint4*>((const uint8_t*)c.pages + ((int64_t)layer * c.n_pages + from) * page_bytes);
  uint4* dst = reinterpret_cast<uint4*>((uint8_t*)c.pages + ((int64_t)layer * c.n_pages + to) * page_bytes);
  const int64_t first = (int64_t)part * (kCopy / 16) + threadIdx.x, all = page_bytes / 16;
  uint4 v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (first + e * 256 < all) v[e] = src[first + e * 256];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (first + e * 256 < all) dst[first + e * 256] = v[e];
}

__global__ void __launch_bounds__(256) kv4_copy_kernel(const b200_kv4_cache c, int64_t page_bytes, const int2* copies) {
  pdl_wait();
  pdl_trigger();
  const int2 copy = copies[blockIdx.y];
  if (copy.x >= 0) copy_part(c, page_bytes, blockIdx.z, copy.x, copy.y, blockIdx.x);
}

// A CTA takes a sequence.
__global__ void __launch_bounds__(128) kv4_free_kernel(const b200_kv4_cache c, const int32_t* seqs) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x, s = seqs[i];
  if (s < 0 || s >= c.n_seqs) return;
  int before = 0;
  for (int j = threadIdx.x; j < i; j += 128) before |= seqs[j] == s;
  if (__syncthreads_or(before)) return;
  const int n = min((c.length[s] + kPage - 1) / kPage, c.max_pages);
  for (int e = threadIdx.x; e < n; e += 128) {
    int32_t* const entry = c.table + (int64_t)s * c.max_pages + e;
    const int page = *entry;
    *entry = -1;
    if (page >= 0 && page < c.n_pages) atomicSub(c.refs + page, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) c.length[s] = 0;
}

// The pages in use behind their number, in order, go to the free ones below it, in order.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv4_compact_kernel(const b200_kv4_cache c, int32_t* live_out, int32_t* moved, int32_t* map, int32_t* from, int32_t* to) {
  pdl_wait();
  pdl_trigger();
  long long mine = 0, live;
  for (int p = threadIdx.x; p < c.n_pages; p += THREADS) {
    mine += c.refs[p] > 0;
    map[p] = p;
  }
  scan_block<THREADS>(mine, &live);
  const int holes = list_pages<THREADS>((int)live, live, to, [&](int p) { return c.refs[p] <= 0; });
  const int behind = c.n_pages - (int)live;
  const int sources = list_pages<THREADS>(behind, holes, from, [&](int p) { return c.refs[(int)live + p] > 0; });
  const int n = min(holes, sources);   // the same number
  for (int k = threadIdx.x; k < n; k += THREADS) {
    const int src = from[k] + (int)live, dst = to[k];
    map[src] = dst;
    from[k] = src;
    c.refs[dst] = c.refs[src];
    c.refs[src] = 0;
  }
  if (threadIdx.x == 0) {
    *live_out = (int)live;
    *moved = n;
  }
}

__global__ void __launch_bounds__(256) kv4_move_kernel(const b200_kv4_cache c, int64_t page_bytes, const int32_t* moved, const int32_t* map, const int32_t* from,
                                                       const int32_t* to) {
  pdl_wait();
  pdl_trigger();
  const int n = *moved;
  if (n == 0) return;
  const int parts = (int)((page_bytes + kCopy - 1) / kCopy);
  for (int64_t job = blockIdx.x; job < (int64_t)n * c.layers * parts; job += gridDim.x) {
    const int k = (int)(job / parts % n);
    copy_part(c, page_bytes, (int)(job / parts / n), from[k], to[k], (int)(job % parts));
  }
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < (int64_t)c.n_seqs * c.max_pages; e += (int64_t)gridDim.x * 256) {
    const int page = c.table[e];
    if (page >= 0 && page < c.n_pages) c.table[e] = map[page];
  }
}

// the workspace: three lists of pages, a pair for every sequence of a call, a word
struct Ws {
  int32_t *a, *b, *c, *word;
  int2* pairs;
  Ws(void* ws, int64_t n_pages) {
    pairs = (int2*)ws;
    a = (int32_t*)(pairs + kKvMaxSeqs);
    b = a + n_pages;
    c = b + n_pages;
    word = c + n_pages;
  }
};

int check_seqs(const b200_kv4_cache* cache, const void* a, const void* b, const void* c, int64_t n, const char* what) {
  const int rc = check_kv4(cache, what);
  if (rc != B200_OK) return rc;
  B200_CHECK_ARG(a && b && c && n >= 1 && n <= kKvMaxSeqs, "%s: %lld sequences (1 … %d), or a null pointer", what, (long long)n, kKvMaxSeqs);
  return B200_OK;
}

}  // namespace

}  // namespace b200

extern "C" {

int64_t b200_kv4_workspace_bytes(const b200_kv4_cache* cache) {
  return cache == nullptr || cache->n_pages < 1 ? -1 : (int64_t)b200::kKvMaxSeqs * 8 + (3 * (int64_t)cache->n_pages + 4) * 4;
}

int b200_kv4_extend(const b200_kv4_cache* cache, const int32_t* seqs, const int32_t* counts, int32_t* pos, int64_t n, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_seqs(cache, seqs, counts, pos, n, "kv4_extend")) != B200_OK) return rc;
  B200_CHECK_ARG(workspace && aligned16(workspace), "kv4_extend: workspace must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const bool small = few(n, cache->n_pages);
  B200_CUDA(launch_pdl(small ? kv4_extend_kernel<kFew> : kv4_extend_kernel<kMany>, dim3(1), dim3(small ? kFew : kMany), 0, st, op_pdl(st), *cache, seqs, counts, pos, (int)n, Ws(workspace, cache->n_pages).a));
  return B200_OK;
}

int b200_kv4_fork(const b200_kv4_cache* cache, const int32_t* src, const int32_t* dst, int32_t* done, int64_t n, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_seqs(cache, src, dst, done, n, "kv4_fork")) != B200_OK) return rc;
  B200_CHECK_ARG(workspace && aligned16(workspace), "kv4_fork: workspace must be 16-byte aligned");
  B200_CHECK_ARG(cache->layers <= 65535, "kv4_fork: %d layers", cache->layers);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pdl = op_pdl(st);
  const Ws ws(workspace, cache->n_pages);
  const int64_t bytes = b200_kv4_page_bytes(cache->kv_heads, cache->dim);
  const bool small = few(n, cache->n_pages);
  B200_CUDA(launch_pdl(small ? kv4_fork_kernel<kFew> : kv4_fork_kernel<kMany>, dim3(1), dim3(small ? kFew : kMany), 0, st, pdl, *cache, src, dst, done, (int)n, ws.a, ws.pairs));
  B200_CUDA(launch_pdl(kv4_copy_kernel, dim3((unsigned)((bytes + kCopy - 1) / kCopy), (unsigned)n, (unsigned)cache->layers), dim3(256), 0, st, pdl, *cache, bytes,
                       ws.pairs));
  return B200_OK;
}

int b200_kv4_free(const b200_kv4_cache* cache, const int32_t* seqs, int64_t n, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_seqs(cache, seqs, seqs, seqs, n, "kv4_free")) != B200_OK) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  B200_CUDA(launch_pdl(kv4_free_kernel, dim3((unsigned)n), dim3(128), 0, st, op_pdl(st), *cache, seqs));
  return B200_OK;
}

int b200_kv4_compact(const b200_kv4_cache* cache, int32_t* live, void* workspace, void* stream) {
  using namespace b200;
  int rc = op_check();
  if (rc != B200_OK || (rc = check_kv4(cache, "kv4_compact")) != B200_OK) return rc;
  B200_CHECK_ARG(live && workspace && aligned16(workspace), "kv4_compact: null pointer, or a workspace that is not 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pdl = op_pdl(st);
  const Ws ws(workspace, cache->n_pages);
  const int64_t bytes = b200_kv4_page_bytes(cache->kv_heads, cache->dim);
  const bool small = few(1, cache->n_pages);
  B200_CUDA(launch_pdl(small ? kv4_compact_kernel<kFew> : kv4_compact_kernel<kMany>, dim3(1), dim3(small ? kFew : kMany), 0, st, pdl, *cache, live, ws.word, ws.a, ws.b, ws.c));
  B200_CUDA(launch_pdl(kv4_move_kernel, dim3(148 * 4), dim3(256), 0, st, pdl, *cache, bytes, ws.word, ws.a, ws.b, ws.c));
  return B200_OK;
}

}  // extern "C"
