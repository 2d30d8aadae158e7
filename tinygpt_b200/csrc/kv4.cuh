// kv4.cuh — the paged cache of keys and values in 4 bits: its layout, and what its kernels share.
//
// A page holds kPage tokens of every key/value head; of a head, four tiles of 16 tokens lie one behind the other, each
//   keys    [group of 64 entries][512 bytes]     lane 4r + c, word 2h + t, byte 2e + hi:  token r + 8·hi, entries 32h + 8c + 4t + 2e + {0, 1}
//   their scale | middle << 16                    [group][r][hi]
//   values  [group][512 bytes]                    lane 4r + c, word j, byte 2e + p:        token 2c + 8p + e, entries 16j + 2r + {0, 1}
//   their scale | middle << 16                    [group][token % 8][token / 8]
// so that a lane's 16 bytes are its A operands of four m16n8k16 products (tokens × entries of K, entries × tokens of Vᵀ), no two tokens share a byte, and
// a byte holds two neighbouring entries.
#pragma once
#include "lowbit.cuh"

namespace b200 {

constexpr int kPage = 64, kKvGroup = 64, kKvTile = 16;
constexpr int kKvMaxSeqs = 1024;                                     // of one call
__host__ __device__ constexpr int kv4_tile_bytes(int groups) { return groups * 2 * (512 + 64); }

// the checks of arguments that the entry points share
int check_kv4(const b200_kv4_cache* c, const char* what);
int check_kv4_rows(const b200_kv4_cache* c, int64_t layer, const int32_t* seqs, const int32_t* starts, const int32_t* pos, int64_t n, int64_t rows,
                   const char* what);

#ifdef __CUDACC__
// Where a row goes: its slot and position (slot < 0: nowhere), and how many rows from it on lie in its tile of 16 (0: an earlier row's run has it).
struct Kv4Place {
  int slot, at, run;
};
__device__ __forceinline__ Kv4Place kv4_place(const b200_kv4_cache& c, int slot, int pos, int first, int end, int row) {   // of a sequence with rows first … end − 1
  const int64_t at = (int64_t)pos + row - first;
  if (first > row || row >= end || pos < 0 || slot < 0 || slot >= c.n_seqs || at >= (int64_t)c.max_pages * kPage) return {-1, 0, 0};
  const int in_tile = (int)(at % kKvTile);
  return {slot, (int)at, in_tile == 0 || row == max(first, 0) ? min(kKvTile - in_tile, end - row) : 0};
}
__device__ __forceinline__ int kv4_page(const b200_kv4_cache& c, int slot, int at) {   // −1: none
  const int page = c.table[(int64_t)slot * c.max_pages + at / kPage];
  return page < c.n_pages ? page : -1;
}
__device__ __forceinline__ uint8_t* kv4_head(const b200_kv4_cache& c, int layer, int page, int head) {
  const int64_t block = 4 * kv4_tile_bytes(c.dim / kKvGroup);
  return (uint8_t*)c.pages + (((int64_t)layer * c.n_pages + page) * c.kv_heads + head) * block;
}
#endif

}  // namespace b200
