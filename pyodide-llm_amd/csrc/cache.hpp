// cache.hpp — the cache held in 8 bits (include/pyodide_llm_hip.h hk_cache): its layout, what its kernels share, and
// their launchers. One layer's cache:
//   keys   int8  [n_kv][blocks][hs / 16][32][16]   channel 16 c + i of the block's position t at [c][t][i]
//   values uint8 [n_kv][blocks][hs][32]            value + 128 of position t at byte value_byte(t) of its channel's 32
//   scales float [n_kv][blocks][2]                 the block's key and value scales
//   recent float [128 + 32][n_kv][hs]              position p's row at p % 128 (the latest 128), then the rows of the
//                                                  first block of a call that displaced them
// A block of 32 positions is one MFMA tile of keys: a lane's 16 bytes of a key row are contiguous, a load instruction of a
// wave reads 1 KiB in order; a lane's 16 bytes of a value column are the positions whose probabilities it holds after the
// product of keys and queries, so that the probabilities go from one product's output registers to the other's input.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

constexpr int CACHE_BLOCK = 32;    // positions a scale (HK_CACHE_BLOCK)
constexpr int CACHE_RECENT = 128;  // positions whose float32 rows are kept (HK_CACHE_RECENT)

// the byte of a channel's 32 that holds position t of a block: half (t >> 2 & 1), then its positions in order
__device__ __forceinline__ int value_byte(int t) {
  return ((t >> 2 & 1) << 4) | ((t >> 4) << 3) | ((t >> 3 & 1) << 2) | (t & 3);
}

}  // namespace ple
