// lr_pieces.h - padded caches of different lengths cut into pieces of one size, in a list
// that every wave works out from the lengths by itself: the lengths stay on the device.
#pragma once

#include "lr_attention.h"

namespace lr {
namespace {

constexpr int kListed = 512;   // caches of a list at most: eight lengths per lane

__device__ __forceinline__ int ceil_div(int a, int b) { return (int)((uint32_t)(a + b - 1) / (uint32_t)b); }
__device__ __forceinline__ int keys_of(const int32_t* lengths, int i, int k_rows) {
  return lengths ? (int)clamp64(lengths[i], 0, k_rows) : k_rows;
}

struct Pieces {
  int tiles[kListed / 64];   // of caches lane, lane + 64, ..
  int groups;
  __device__ __forceinline__ void load(const int32_t* lengths, int n, int k_rows, int tile) {
    const int lane = threadIdx.x & 63;
    groups = (n + 63) >> 6;
#pragma unroll
    for (int g = 0; g < kListed / 64; ++g) {
      const int i = 64 * g + lane;
      tiles[g] = i < n ? (int)((uint32_t)(keys_of(lengths, i, k_rows) + tile - 1) / (uint32_t)tile) : 0;
    }
  }
  // How many pieces of `size` tiles there are. In fp32: what has to be exact is below 2^24.
  __device__ __forceinline__ float count(int size) const {
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < kListed / 64; ++g)
      if (g < groups) sum += (float)ceil_div(tiles[g], size);
    // The same in every lane; said so, since what depends on it addresses memory.
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_tree_sum(sum))));
  }
  // The cache (-1: none) that has piece `place`, and its first piece.
  __device__ __forceinline__ void find(int n, int size, int place, int& seq, int& first) const {
    const int lane = threadIdx.x & 63;
    int before = 0;
    seq = -1;
#pragma unroll
    for (int g = 0; g < kListed / 64; ++g) {
      if (g >= groups || seq >= 0) continue;
      const int mine = ceil_div(tiles[g], size), upto = wave_prefix_sum(mine);
      const uint64_t hit = __ballot(before + upto > place && 64 * g + lane < n);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        seq = 64 * g + l;
        first = before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  // Tiles of a piece where `all` are cut into `count`: even ones, the last at most smaller.
  static __device__ __forceinline__ int even(int all, int count) { return count > 1 ? ceil_div(all, count) : all; }
};

}  // namespace
}  // namespace lr
