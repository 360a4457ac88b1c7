// What the two kernels of int4_attention share: the call's parameters, which
// requests go to which kernel, and fp16 pair arithmetic on 4-bit codes.
#pragma once

#include "int4_pages.cuh"

namespace ss {

struct AttnParams {
  const void* q;
  int dtype, q_vec;  // q_vec: rows of q are 16-byte aligned
  int64_t q_st, q_sh;
  int64_t n_tokens;
  int hq, hkv, grp;
  const uint8_t* pages;
  int n_pages;
  int64_t page_stride, head_stride;
  int page, page_blocks;  // tokens and blocks of a page
  uint32_t page_inv;      // 2^32 / page_blocks, rounded up
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t *seq_lens, *cu_q;
  int n;
  float scale;
  int causal, window;
  void* out;
  float* lse;
  uint8_t* ws;    // counters of the warp-MMA kernel's CTAs
  float* parts;   // and their parts: a place that does not depend on the kernel's shape
  uint32_t* tile_ws;  // the tile kernel's counters, 4 per unit
  float* tile_parts;  // and its parts, one per CTA
  int tiles;    // the tile kernel runs too
  int64_t tile_units;  // about how many units it has at most
  uint64_t wait_ns;   // bound of its waits
  uint32_t skip_tile; // test hook: tile of a CTA whose keys are never seen (all ones: none)
  int* sink;    // process error sink (host word) or null
};

// Probabilities enter the second product in fp16, relative to a row's reference. It is set kBelow
// under the largest logit (base 2) and moved when one exceeds it by kSlack: the largest probability
// lies in [2^10, 2^15.5], so that one of 2^-24 of it (17 nats below) is still a normal fp16 number,
// and below that a grid of 2^-34 of the largest is left. (From the largest logit itself, with a grid
// of 2^-24, 64K keys 18 nats below one are lost.) More room below leaves less above, where a new
// largest logit rescales O: a windowed batch of mixed lengths, 64 dims, takes 127.5 us with 10 as with
// 7, 131 with 11 and 136 with 12.
constexpr float kLow = -3e38f;   // softmax reference before any key
constexpr float kBelow = 10.f, kSlack = 15.5f;
constexpr float kLog2e = 1.4426950408889634f;

// Rows (query tokens times heads of a group) from which a request's queries go to the tiles of
// 128 rows of the tcgen05 kernel instead of the 16-row units of the warp-MMA kernel. A tile is one
// CTA's work, or a few CTAs' where there are few tiles; the units of a request are spread over all
// SMs, but read and decode the keys once per 16 rows. The tiles win from about nine full tiles on,
// whatever the keys, and from 48 rows where rows times heads times keys reach 2^21 (8 kv heads of 128
// dims, groups of 4, units against tiles: 32 prompts of 40 tokens 139 and 49 us, though one alone 17
// and 21; 68 rows over 4017 keys 37 and 35 us, over 517 keys 18 and 28; 128 rows over 30000 keys 125
// and 65; 8 requests of 36 rows over 4009 keys 69 and 68, 8 of 128 rows over 4032 152 and 52). The
// rule is a request's own: how many others there are is not known where it is asked.
constexpr float kTilesFrom = 1152.f, kTileRowsFrom = 48.f, kTileWorkFrom = 0x1p21f;

__device__ __forceinline__ bool to_tiles(const AttnParams& p, int nq, int len) {
  const float rows = (float)nq * p.grp, all = rows * p.hkv;
  const float keys = p.window > 0 ? fminf((float)len, (float)p.window + nq) : (float)len;
  return p.tiles && rows > 16.f && (all >= kTilesFrom || (rows >= kTileRowsFrom && all * keys >= kTileWorkFrom));
}

// What a request contributes to the schedule of the warp-MMA kernel.
struct Req {
  int nq, len, rbs, blk0, nblk;  // query rows' tokens, keys, row blocks, first key block, key blocks (>= 1)
};

template <int R>
__device__ __forceinline__ Req load_req(const AttnParams& p, int b) {
  Req r;
  const int c0 = max(p.cu_q[b], 0);
  r.nq = max(p.cu_q[b + 1] - c0, 0);
  r.len = min(max(p.seq_lens[b], 0), p.width * p.page);
  r.rbs = to_tiles(p, r.nq, r.len) ? 0 : (int)(((int64_t)r.nq * p.grp + R - 1) / R);
  r.blk0 = p.window > 0 ? max(0, r.len - r.nq - p.window + 1) / kBlkTokens : 0;
  r.nblk = max(1, (r.len + kBlkTokens - 1) / kBlkTokens - r.blk0);
  return r;
}

// Page of a request's block k, and the block's place in it.
__device__ __forceinline__ int page_of(const AttnParams& p, int k, int& in_page) {
  if (p.page_blocks == 1) {
    in_page = 0;
    return k;
  }
  int q = (int)__umulhi((uint32_t)k, p.page_inv);  // k / page_blocks, or one more
  int r = k - q * p.page_blocks;
  if (r < 0) { --q; r += p.page_blocks; }
  in_page = r;
  return q;
}

__device__ __forceinline__ uint32_t lop_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t r;  // (x & mask) | magic
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(magic));
  return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float lo_h(uint32_t x) { return __low2float(*reinterpret_cast<__half2*>(&x)); }
__device__ __forceinline__ float hi_h(uint32_t x) { return __high2float(*reinterpret_cast<__half2*>(&x)); }


// Floats of a CTA's part in the tile kernel: 128 rows of D dims, reference and sum.
__host__ __device__ constexpr int tile_part_floats(int d) { return 128 * (d + 2); }

// The requests of a batch that have query rows for the tiles, see int4_prompt.cu.
int launch_tiles(AttnParams& p, int d, cudaStream_t st);

}  // namespace ss
