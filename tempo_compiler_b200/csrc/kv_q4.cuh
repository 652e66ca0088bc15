// The 4-bit key/value cache's layout. A cache is [seqs][kv_heads][capacity / 16] tiles of 16 positions; a tile holds
// one 1152-byte block per group of 64 head dimensions:
//   [0, 512)      key codes, 32 bytes per position: dimension d in byte d / 2, the even one in the low half
//   [512, 1024)   value codes, alike
//   [1024, 1152)  per position four BF16 words: key scale, key low, value scale, value low
// A tile is contiguous, so the positions of one (sequence, head) are one stream and a run of tiles is one bulk copy.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tempo {

constexpr uint32_t kQ4Group = 64;
constexpr uint32_t kQ4Tile = 16;
constexpr uint32_t kQ4Codes = kQ4Tile * kQ4Group / 2;              // 512 bytes of codes per tile, group and K or V
constexpr uint32_t kQ4Block = 2 * kQ4Codes + kQ4Tile * 4 * 2;      // 1152

// The block of group `group` holding position `pos` of (seq, head) in a cache of `kv_heads` heads, `tiles` tiles per
// sequence and `groups` groups per head.
__device__ __forceinline__ size_t q4_block(uint32_t seq, uint32_t head, uint32_t pos, uint32_t group,
                                           uint32_t kv_heads, uint32_t tiles, uint32_t groups) {
  return (((size_t(seq) * kv_heads + head) * tiles + pos / kQ4Tile) * groups + group) * kQ4Block;
}

}  // namespace tempo
