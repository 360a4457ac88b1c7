// Byte layout of 4-bit KV pages, shared by the kernels that write, read and
// attend over them.
//
// A page of one kv-head is a run of blocks of 16 tokens; a block is one
// contiguous record of 20 * D bytes (5 bits per stored value):
//   key codes    8 D bytes   word (token, group g, j) = dims 32 g + 8 j .. + 7
//   key (s, z)   2 D bytes   half2 per (token, group)
//   value codes  8 D bytes   word (token, x) = dims 8 x .. 8 x + 7
//   value (s, z) 2 D bytes   half2 per (token, group)
// A group is 32 dims of one token; value = code * s + z; nibble n of a word
// is its n-th dim. The words are ordered for warp MMAs (m16n8k16): lane
// 4 i + j of a warp finds its key words (tokens i and i + 8, one word per
// group) and its value words (tokens 2j, 2j+1, 2j+8, 2j+9; dims 8 w i ..) in
// 16-byte pieces, and the pieces of a warp are contiguous, so that one warp
// load reads 512 contiguous bytes without shared-memory bank conflicts.
#pragma once

#include "common.cuh"

namespace ss {

constexpr int kBlkTokens = 16;
constexpr int kGroup = 32;
constexpr float kInt4Max = 32768.f;  // larger magnitudes saturate (code * s + z stays finite in fp16)

template <int D>
struct Int4Blk {
  static_assert(D % 64 == 0, "head_dim");
  static constexpr int G = D / kGroup;         // groups of a row
  static constexpr int W = D / 64;             // value words of a lane per token
  static constexpr int N = G < 4 ? G : 4;      // key words in one piece
  static constexpr int kBytes = 20 * D;
  static constexpr int kKs = 8 * D, kV = 10 * D, kVs = 18 * D;  // section offsets (keys at 0)

  static __host__ __device__ constexpr int key_word(int tok, int g, int j) {
    return (((g / N) * 16 + tok) * 4 + j) * (N * 4) + (g % N) * 4;
  }
  static __host__ __device__ constexpr int key_sz(int tok, int g) { return kKs + (tok * G + g) * 4; }
  static __host__ __device__ constexpr int value_word(int tok, int x) {
    return kV + ((((tok >> 3) * 2 + (tok & 1)) * W + x % W) >> 2) * 512 +
           ((x / W) * 4 + ((tok & 7) >> 1)) * 16 + ((((tok >> 3) * 2 + (tok & 1)) * W + x % W) & 3) * 4;
  }
  static __host__ __device__ constexpr int value_sz(int tok, int g) {
    return kVs + (((g * 4 + ((tok & 7) >> 1)) * 2 + (tok >> 3)) * 2 + (tok & 1)) * 4;
  }
};

inline bool int4_head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

}  // namespace ss
