// Attention of many query rows over 4-bit KV pages on the 5th-generation
// tensor cores (tcgen05): the tile kernel of int4_attention.
//
// A unit is (request, kv-head, 128 query rows); the rows of a group's heads and
// of consecutive tokens share a tile, so keys and values are decoded once for
// all of them. CTAs (one an SM) take units in turn, those with most keys of a
// request first, rounds in alternating direction; where there are few units their
// keys are cut into parts (fp32 rows of O, reference and sum in the workspace,
// joined by the last of them to arrive, in order). Per tile of 128 tokens:
//   decode    (8 warps)  codes -> fp16 operands in shared memory
//   S = Q K^T (1 thread) M = 128, N = 128, fp32 in TMEM, two buffers
//   softmax   (8 warps)  two threads a row, P as fp16 over its S in TMEM
//   O += P V  (1 thread) M = 128, N = D, fp32 in TMEM
// and the four run on different tiles at the same time, handing over through
// mbarriers (two stages of keys and values, two S buffers). Q and P are A
// operands in TMEM, which leaves shared memory to the two stages. Issuing an
// MMA takes the thread about 75 cycles beside the other warps' work, a tile of
// 64 tokens as long as one of 128.
//
// Keys enter as pairs of fp16 values, hi = fp16(c s) and lo = c s - hi (15 bits
// in all, so lo is exact), and q . z is one more K step of 16, z as stored
// against the row's group sums in two fp16 terms. One rounded fp16 key would
// move a logit by 3e-4, which rows with few keys show in their log-sum-exp; the
// second product costs 136 / 264 of the tensor time of a tile. Codes enter
// halved, since 15 s can be one place above fp16's largest: exact but where c and
// s / 2^-24 are odd and s is below 2^-13; there a key is off by 2^-24.
// Values are fp16(c s + z), probabilities fp16, or hi + lo (a second pass of
// P V) where the output is fp16 and the rounding would show. Row statistics
// and both products accumulate in fp32. O in TMEM is rescaled only when a logit
// comes 5.5 (base 2) above the row's largest so far.
//
// Measured: one causal prompt of 8192 tokens, 32 query heads on 8, calls on end for
// half a second: D = 128 bf16 938 us (586 TFLOP/s of the formula's 4 D a pair; the
// tensor cores do half as much again for lo), fp16 1150 us, D = 64 688 us. In bursts,
// before the power limit lowers the clocks, 870, 1035 and 690 us; the figures below
// are such bursts. A tile of 128 keys takes 1.9 us: the tensor pipe is busy 40 % of the time, issue slots 55 %, shared
// memory 46 %; no one of them is full, the chain decode - S - softmax - O of two
// tiles in flight is (a third tile has no room: two stages take 205 KB, and S, P,
// O and Q all 512 TMEM columns). When the kernel took 860 us, a softmax thread per row instead of two: 910 us;
// tiles of 64 keys 1322; Q and P in shared memory 1598. The registers follow from
// what a role keeps: with fewer than 120 the softmax spills O's rescale, and 28
// warps (16 decoding) at 72 took 1421 us.
//
// Every wait is bounded (2 s) and reports through the process error sink.
#include "int4_attn.cuh"
#include "tcgen05.cuh"

namespace ss {
namespace {

constexpr int kTileRows = 128, kTileKeys = 128;
constexpr int kMmaWarp = 0, kSoftWarp = 4, kSoftWarps = 8, kDecWarp = kSoftWarp + kSoftWarps, kDecWarps = 8;  // two warps issue MMAs
constexpr int kTileWarps = 20, kTileThreads = kTileWarps * 32;  // whole warpgroups: registers are moved between them
// Registers of a thread: 96 at launch; 8 * 120 + 8 * 88 + 4 * 64 = 20 * 96.
constexpr int kSoftRegs = 120, kDecRegs = 88, kMmaRegs = 64;
constexpr int kHalfKeys = kTileKeys / 2;  // of a softmax thread: a row is two threads' work
constexpr int kTileWaitCode = 32;
constexpr int kMinTiles = 4, kMaxSplit = 16;  // key tiles of a part, parts of a unit

template <int D>
struct Tile {
  static constexpr int kChunk = kTileKeys * 16 + 32;  // a dim chunk of keys; + 32: no bank conflicts
  static constexpr int kKey = D / 8 * kChunk;       // hi; lo behind it
  static constexpr int kZ = 2 * kTileKeys * 16;     // zeros, twice
  static constexpr int kVal = kTileKeys * D * 2;    // [8 tokens][dim chunk][token] 16 bytes
  static constexpr int kStage = 2 * kKey + kZ + kVal;
  static constexpr int kOffMisc = 2 * kStage;
  static constexpr int kOffRow = kOffMisc + 512 + kTileThreads * 4;
  static constexpr int kSmem = kOffRow + 6 * kTileRows * 4;
  // TMEM columns: two S, each overwritten by its P (hi, then lo; two fp16 a column), O, Q, its group sums
  static constexpr int kTO = 2 * kTileKeys, kTQ = kTO + D, kTSum = kTQ + D / 2;
  static constexpr int kCols = 512;
  static_assert(kTSum + 8 <= kCols, "TMEM");
};

__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {  // fp16 in, fp32 out, M = 128
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
}
// 32 columns of this thread's TMEM lane, fp32.
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// (a, b) = (x, y) * s + (a, b), packed fp32
__device__ __forceinline__ void fma_f32x2(float& a, float& b, float x, float y, float s) {
  asm("{\n .reg .b64 t, u, v;\n mov.b64 t, {%0, %1};\n mov.b64 u, {%2, %3};\n mov.b64 v, {%4, %4};\n"
      " fma.rn.f32x2 t, u, v, t;\n mov.b64 {%0, %1}, t;\n}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y), "f"(s));
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int N>
__device__ __forceinline__ void tc_st(uint32_t taddr, const uint32_t* v) {
  if constexpr (N == 16) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
  } else {
    static_assert(N == 8, "columns");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  }
}
// D[tmem] (+)= A[tmem] * B[smem]; the descriptor of B in two words, so that steps are immediates.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t id, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.u32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(id), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t hfms2(uint32_t a, uint32_t b, uint32_t c) {  // a b - c
  uint32_t r;
  asm("{\n .reg .b32 n;\n neg.f16x2 n, %3;\n fma.rn.f16x2 %0, %1, %2, n;\n}" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// The MMAs of a tile in stage ST. Shared memory starts at 16 * base; TMEM at 0. A descriptor's
// words: start address and bytes between core matrices along K; bytes along N (128) and version.
__host__ __device__ constexpr uint32_t b_word(int at, int lbo) { return (uint32_t)at / 16 | (uint32_t)lbo / 16 << 16; }
constexpr uint32_t kBHi = 128 >> 4 | 1u << 14;

template <int D, int ST>
__device__ __forceinline__ void issue_qk(uint32_t base) {
  using T = Tile<D>;
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // hi, lo
#pragma unroll
    for (int c = 0; c < D / 8; c += 2)
      tc_mma_ts(ST * kTileKeys, T::kTQ + c * 4, base + b_word(ST * T::kStage + half * T::kKey + c * T::kChunk, T::kChunk), kBHi,
                idesc(kTileKeys, false), (half | c) != 0);
  }
  tc_mma_ts(ST * kTileKeys, T::kTSum, base + b_word(ST * T::kStage + 2 * T::kKey, kTileKeys * 16), kBHi, idesc(kTileKeys, false), true);
}

template <int D, bool LO, int ST>
__device__ __forceinline__ void issue_pv(uint32_t base, bool acc) {
  using T = Tile<D>;
#pragma unroll
  for (int half = 0; half < (LO ? 2 : 1); ++half) {
#pragma unroll
    for (int c = 0; c < kTileKeys / 8; c += 2)
      tc_mma_ts(T::kTO, ST * kTileKeys + half * (kTileKeys / 2) + c * 4,
                base + b_word(ST * T::kStage + 2 * T::kKey + T::kZ + c * (D / 8 * 128), D / 8 * 128), kBHi, idesc(D, true),
                (half | c) != 0 || acc);
  }
}

// A unit: its rows, and the key tiles [kt0, kt1) that any of them sees.
struct Unit {
  int b, h, row0, rows, nq, len, tok0, kt0, kt1, all0, all1;  // rows see the keys [all0, all1) whole
};

__device__ __forceinline__ int tiles_of(const AttnParams& p, int b) {
  const int nq = max(p.cu_q[b + 1] - max(p.cu_q[b], 0), 0);
  int len = 0;
  if ((float)nq * p.grp * p.hkv < kTilesFrom) len = min(max(p.seq_lens[b], 0), p.width * p.page);
  return to_tiles(p, nq, len) ? (int)(((int64_t)nq * p.grp + kTileRows - 1) / kTileRows) : 0;
}
// Keys [beg, end) that the row of query token i sees.
__device__ __forceinline__ void row_keys(const AttnParams& p, int nq, int len, int i, int& beg, int& end) {
  const int pos = len - nq + i;
  end = p.causal ? max(0, min(len, pos + 1)) : len;
  beg = p.window > 0 ? max(0, pos - p.window + 1) : 0;
}

// SPLIT: units may be cut into parts by keys, see launch.
template <int D, bool LO, bool SPLIT>
__global__ void __launch_bounds__(kTileThreads, 1) attn_tile_kernel(const __grid_constant__ AttnParams p) {
  using B = Int4Blk<D>;
  using T = Tile<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kOffMisc);
  uint64_t* k_full = bars;         // [2] the 8 decode warps have written keys
  uint64_t* v_full = bars + 10;    // [2] and values
  uint64_t* o_done = bars + 2;     // [2] P V is done: the stage's values and its S are free
  uint64_t* s_full = bars + 4;     // [2] Q K^T is done: S is there, the stage's keys are free
  uint64_t* p_full = bars + 8;     // [2] the 8 softmax warps have written P
  uint64_t* q_full = bars + 13;    // and the unit's Q
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 14);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  uint8_t* s_hidden = reinterpret_cast<uint8_t*>(s_tmem + 2);  // [4][8] blocks of a tile without a page; read before S is freed
  int* s_sum = reinterpret_cast<int*>(smem + T::kOffMisc + 256);      // [20] warps' units
  int* s_cum = reinterpret_cast<int*>(smem + T::kOffMisc + 512);      // [threads] units before a thread's requests
  int* s_parts = reinterpret_cast<int*>(smem + T::kOffMisc + 384);    // [20] parts of the unit a warp is at
  int* s_ticket = s_parts + kTileWarps;                               // [4] whether rows' last part is this one
  float* s_top = reinterpret_cast<float*>(smem + T::kOffRow);         // [2 tiles][2 halves][128] largest logits of a row
  float* s_fac = s_top + 4 * kTileRows;                               // [128] from logits to base 2
  float* s_l = s_fac + kTileRows;                                     // [128] a half's sum

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // ---- setup ---------------------------------------------------------------
  grid_launch_dependents();  // the warp-MMA kernel of the same call: other rows, its own workspace
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full + s, kDecWarps);
      mbar_init(v_full + s, kDecWarps);
      mbar_init(o_done + s, 1);
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, kSoftWarps);
    }
    mbar_init(q_full, 4);
    mbar_init(bars + 12, 2);  // end of an abandoned unit's MMAs
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tc_alloc(s_tmem, T::kCols);
    tc_relinquish();
  }
  const int per = (p.n + kTileThreads - 1) / kTileThreads;
  const int b0 = min(p.n, tid * per), b1 = min(p.n, b0 + per);
  int units = 0;
  for (int b = b0; b < b1; ++b) units += tiles_of(p, b) * p.hkv;
  int inc = units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) s_sum[warp] = inc;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int total = 0, before = 0;
  for (int w = 0; w < kTileWarps; ++w) {
    if (w == warp) before = total;
    total += s_sum[w];
  }
  s_cum[tid] = before + inc - units;
  __syncthreads();
  if (tid == 0 && *s_tmem != 0) {  // all columns were asked for: they start at 0
    report_wait_failure(nullptr, p.sink, kTileWaitCode);
    *s_abort = 1;
  }
  constexpr uint32_t tmem = 0, t_o = T::kTO;

  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
      if (mbar_try_wait(bar, parity)) return true;
      if (*s_abort) return false;
      if (global_ns() - t0 > p.wait_ns) {
        if (!*s_abort) report_wait_failure(nullptr, p.sink, kTileWaitCode);
        *s_abort = 1;
        return false;
      }
    }
  };

  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  // With no more units than half the CTAs, a unit's keys are cut into parts of at least kMinTiles
  // tiles, one CTA each; for each 32 rows the last one to arrive joins them in order.
  const int split = SPLIT ? max(1, min(kMaxSplit, (int)gridDim.x / max(total, 1))) : 1;

  // The CTA's next unit; false when there is none. Each role walks the units by itself.
  int round = 0;
  auto next_unit = [&](Unit& un) -> bool {
    int u;
    do {  // longest first within a request, rounds in alternating direction: nearly equal sums
      if (round * (int64_t)gridDim.x >= total) return false;
      u = round * (int)gridDim.x + (int)(round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      ++round;
    } while (u >= total * split);
    int part = 0;
    if constexpr (SPLIT) {
      part = u / total;
      u -= part * total;
    }
    int a = 0, e = kTileThreads;
    while (e - a > 1) {
      const int mid = (a + e) >> 1;
      if (s_cum[mid] <= u) a = mid; else e = mid;
    }
    int at = s_cum[a], b = a * per, tiles = 0;
#pragma unroll 1
    for (;; ++b) {
      tiles = tiles_of(p, b);
      if (at + tiles * p.hkv > u) break;
      at += tiles * p.hkv;
    }
    const int qt = tiles - 1 - (u - at) / p.hkv;  // the last rows of a causal request see most keys
    un.b = b;
    un.h = (u - at) % p.hkv;
    un.tok0 = max(p.cu_q[b], 0);
    un.nq = max(p.cu_q[b + 1] - un.tok0, 0);
    un.len = min(max(p.seq_lens[b], 0), p.width * p.page);
    un.row0 = qt * kTileRows;
    un.rows = (int)min((int64_t)kTileRows, (int64_t)un.nq * p.grp - un.row0);
    int beg0, end0, beg1, end1;
    row_keys(p, un.nq, un.len, un.row0 / p.grp, beg0, end0);
    row_keys(p, un.nq, un.len, (un.row0 + un.rows - 1) / p.grp, beg1, end1);
    un.kt0 = beg0 / kTileKeys;
    un.kt1 = end1 <= beg0 ? un.kt0 : max(un.kt0, (end1 + kTileKeys - 1) / kTileKeys);
    un.all0 = beg1;
    un.all1 = end0;
    if constexpr (SPLIT) {
      const int per = max(kMinTiles, (un.kt1 - un.kt0 + split - 1) / split);
      const int parts = max(1, (un.kt1 - un.kt0 + per - 1) / per);
      if (part >= parts) return false;
      un.kt0 += part * per;
      un.kt1 = min(un.kt1, un.kt0 + per);
      if (lane == 0) s_parts[warp] = parts;
    }
    return true;
  };

  Unit un;
  uint32_t n0 = 0;  // tiles of this CTA's earlier units: the barriers' phases go on
  bool ok = true;   // no wait gave up
  if (warp >= kSoftWarp && warp < kDecWarp) {
    // ================= softmax: two threads per row, 64 keys of a tile each =======
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int pair = 1 + (warp & 3);  // named barrier of the two warps that share 32 rows
    // Both warps of a pair come here equally often, or one gives up in a wait: it then arrives
    // once (below), and its partner finds the flag set.
    auto pair_sync = [&]() -> bool {
      named_bar_sync(pair, 64);
      return __any_sync(0xffffffffu, *s_abort) == 0;
    };
    while (ok && next_unit(un)) {
      const int nt = un.kt1 - un.kt0;
      const int half = (warp - kSoftWarp) >> 2, r = tid & (kTileRows - 1), rr = un.row0 + r, i = rr / p.grp, hd = un.h * p.grp + rr % p.grp;
      const int64_t tok = un.tok0 + (int64_t)i;
      const bool live = r < un.rows && tok < p.n_tokens;
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      if (half == 0) {  // the row's queries, scaled by a power of two into [256, 512), and its group sums
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + tok * p.q_st + hd * p.q_sh;
        uint32_t w[D / 8][4];  // all of the row in flight
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          w[c][0] = w[c][1] = w[c][2] = w[c][3] = 0u;
          if (live) {
            if (p.q_vec) {
              const uint4 v = __ldg(reinterpret_cast<const uint4*>(qp) + c);
              w[c][0] = v.x; w[c][1] = v.y; w[c][2] = v.z; w[c][3] = v.w;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) w[c][e] = qp[c * 8 + 2 * e] | (uint32_t)qp[c * 8 + 2 * e + 1] << 16;
            }
          }
        }
        const bool f16 = p.dtype == SS_F16;
        float big = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = f16 ? lo_h(w[c][e]) : __uint_as_float(w[c][e] << 16);
            const float b = f16 ? hi_h(w[c][e]) : __uint_as_float(w[c][e] & 0xffff0000u);
            big = fmaxf(big, fmaxf(fabsf(a), fabsf(b)));
          }
        }
        int ex = 0;
        if (big > 0.f && big < INFINITY) ex = 135 - (int)(__float_as_uint(fmaxf(big, 1.2e-38f)) >> 23);
        float up = ex > 126 ? __uint_as_float(253u << 23) : __uint_as_float((uint32_t)(127 + ex) << 23);
        // fac > 0, so that the largest product is the largest logit: a negative scale turns the
        // queries round, a scale of 0 clears them
        s_fac[r] = p.scale == 0.f ? 1.f : 2.f * fabsf(p.scale) * kLog2e / up;
        up = p.scale < 0.f ? -up : p.scale == 0.f ? 0.f : up;
        uint32_t qs[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};  // group sums: 8 hi, 8 lo
        static_assert(B::G <= 8, "group sums fill one chunk");
        float sum[B::G];
#pragma unroll
        for (int g = 0; g < B::G; ++g) {
          sum[g] = 0.f;
          uint32_t qo[16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = w[g * 4 + c][e];
              f[2 * e] = f16 ? lo_h(x) : __uint_as_float(x << 16);
              f[2 * e + 1] = f16 ? hi_h(x) : __uint_as_float(x & 0xffff0000u);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dims (e, e + 4) side by side, as the key words' nibbles come
              qo[c * 4 + e] = pack_h2(f[e] * up, f[e + 4] * up);
              sum[g] += lo_h(qo[c * 4 + e]) + hi_h(qo[c * 4 + e]);
            }
          }
          tc_st<16>(tmem + lane_base + T::kTQ + g * 16, qo);
        }
#pragma unroll
        for (int g = 0; g < B::G; g += 2) {  // halved, as the keys are
          const float a = 0.5f * sum[g], b = 0.5f * sum[g + 1];
          qs[g / 2] = pack_h2(a, b);
          qs[4 + g / 2] = pack_h2(a - lo_h(qs[g / 2]), b - hi_h(qs[g / 2]));
        }
        tc_st<8>(tmem + lane_base + T::kTSum, qs);
        tc_wait_st();
        tc_fence_before();
      }
      ok = pair_sync();
      if (!SPLIT && !ok) break;  // parts arrive all the same
      const float fac = s_fac[r];
      if (ok && lane == 0 && half == 0 && nt > 0) mbar_arrive(q_full);  // and O of the unit before has been read

      int beg = 0, end = 0;
      if (r < un.rows) row_keys(p, un.nq, un.len, i, beg, end);
      float m = kLow, l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
      for (int j = 0; j < nt && ok; ++j) {
        const uint32_t n = n0 + j, buf = n & 1, ph = (n >> 1) & 1;
        if (!(ok = warp_wait(s_full + buf, ph))) break;
        tc_fence_after();
        float y[kHalfKeys];
        {
          uint32_t v0[32], v1[32];
          tc_ld32(tmem + lane_base + buf * kTileKeys + half * kHalfKeys, v0);
          tc_ld32(tmem + lane_base + buf * kTileKeys + half * kHalfKeys + 32, v1);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            y[e] = __uint_as_float(v0[e]);
            y[32 + e] = __uint_as_float(v1[e]);
          }
        }
        const uint32_t hid = *reinterpret_cast<const uint32_t*>(s_hidden + (n & 3) * 8 + half * 4);

        const int t0 = (un.kt0 + j) * kTileKeys + half * kHalfKeys;
        if (t0 < un.all0 || t0 + kHalfKeys > un.all1 || hid != 0) {
#pragma unroll
          for (int e = 0; e < kHalfKeys; ++e)
            if (t0 + e >= end || t0 + e < beg || (hid >> (e / 16 * 8) & 1)) y[e] = -INFINITY;
        }
        float tops[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int e = 4; e < kHalfKeys; e += 2) tops[e / 2 % 4] = fmax3(tops[e / 2 % 4], y[e], y[e + 1]);
        float top = fmaxf(fmax3(tops[0], tops[1], tops[2]), tops[3]) * fac;  // fac > 0
        // both halves of a row go by the same reference
        s_top[(buf * 2 + half) * kTileRows + r] = top;
        tc_fence_before();
        if (!(ok = pair_sync())) break;  // and both have read S
        tc_fence_after();
        top = fmaxf(top, s_top[(buf * 2 + (half ^ 1)) * kTileRows + r]);
        if (__any_sync(0xffffffffu, top > m + kSlack)) {
          const float mn = fmaxf(m, top - kBelow), f = ex2(m - mn);
          m = mn;
          l0 *= f;
          l1 *= f;
          l2 *= f;
          l3 *= f;
          if (j > 0) {  // O holds the tiles before: all of them, once the last one's P V is done
            if (!(ok = warp_wait(o_done + (buf ^ 1), ((n - 1) >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 32) {  // a half of the dims each
              uint32_t v[32];
              tc_ld32(t_o + lane_base + half * (D / 2) + c, v);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
              tc_st32(t_o + lane_base + half * (D / 2) + c, v);
            }
            tc_wait_st();
            tc_fence_before();
          }
        }
        // The exponent is one FMA; from 2^22 on its unrounded product strays from the reference by
        // whole units, so products are rounded before the difference there.
        float fac_x = fac, m_x = m;
        if (__any_sync(0xffffffffu, fabsf(m) > 0x1p22f && m != kLow)) {
#pragma unroll
          for (int e = 0; e < kHalfKeys; ++e) y[e] = __fadd_rn(__fmul_rn(y[e], fac), -m);
          fac_x = 1.f;
          m_x = 0.f;
        }
        // P over the S it comes from
#pragma unroll
        for (int c = 0; c < kHalfKeys; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float& a = y[c + 2 * e];
            float& b = y[c + 2 * e + 1];
            float x = -m_x, z = -m_x;
            fma_f32x2(x, z, a, b, fac_x);
            a = ex2(x);
            b = ex2(z);
            add_f32x2(e & 1 ? l2 : l0, e & 1 ? l3 : l1, a, b);
            w[e] = pack_h2(a, b);
          }
          const uint32_t at = tmem + lane_base + buf * kTileKeys + (half * kHalfKeys + c) / 2;
          tc_st<16>(at, w);
          if constexpr (LO) {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack_h2(y[c + 2 * e] - lo_h(w[e]), y[c + 2 * e + 1] - hi_h(w[e]));
            tc_st<16>(at + kTileKeys / 2, w);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + buf);
      }
      // ---- output ----
      float l = (l0 + l1) + (l2 + l3);
      if (half == 1) s_l[r] = l;
      ok = ok && pair_sync();
      if (half == 0) s_top[r] = l += s_l[r];
      ok = ok && pair_sync();
      l = s_top[r];
      if (ok && nt > 0) ok = warp_wait(o_done + ((n0 + nt - 1) & 1), ((n0 + nt - 1) >> 1) & 1);
      const int parts = SPLIT ? s_parts[warp] : 1;
      bool mine = ok;  // this CTA writes the rows
      if (SPLIT && parts > 1) {
        // Part c of unit u is CTA c total + u's: columns in fours, rows side by side.
        const int u = blockIdx.x % total;
        auto part_of = [&](int c) { return p.tile_parts + (size_t)(c * total + u) * tile_part_floats(D); };
        if (ok) {
          float* to = part_of(blockIdx.x / total);
          tc_fence_after();
#pragma unroll 1
          for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t v[32];
            tc_ld32(t_o + lane_base + c, v);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 8; ++x)
              __stcg(reinterpret_cast<uint4*>(to) + (c / 4 + x) * kTileRows + r, make_uint4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]));
          }
          if (half == 0) {
            __stcg(to + kTileRows * D + r, m);
            __stcg(to + kTileRows * (D + 1) + r, l);
          }
          __threadfence();
        }
        ok = ok && pair_sync();
        if (half == 0 && lane == 0) {  // a part that was given up arrives too: counters end at zero
          uint32_t* cnt = p.tile_ws + u * 4 + (warp & 3);
          const bool last = atomicAdd(cnt, 1u) == (uint32_t)parts - 1;
          if (last) *cnt = 0u;
          __threadfence();
          s_ticket[warp & 3] = last;
        }
        ok = ok && pair_sync();
        mine = ok && s_ticket[warp & 3];
        if (mine) {
          float mm = kLow;
#pragma unroll 4
          for (int c = 0; c < parts; ++c) mm = fmaxf(mm, __ldcg(part_of(c) + kTileRows * D + r));
          m = mm;
          l = 0.f;
#pragma unroll 4
          for (int c = 0; c < parts; ++c)
            l = fmaf(ex2(__ldcg(part_of(c) + kTileRows * D + r) - mm), __ldcg(part_of(c) + kTileRows * (D + 1) + r), l);
        }
      }
      if (mine) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (tok * p.hq + hd) * D + half * (D / 2);
#pragma unroll
        for (int c = 0; c < D / 2; c += 32) {
          uint32_t v[32];
          if ((!SPLIT || parts == 1) && nt > 0) {
            tc_ld32(t_o + lane_base + half * (D / 2) + c, v);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
            const int u = blockIdx.x % total;
#pragma unroll 2
            for (int k = 0; SPLIT && k < parts && parts > 1; ++k) {
              const float* from = p.tile_parts + (size_t)(k * total + u) * tile_part_floats(D);
              const float f = ex2(__ldcg(from + kTileRows * D + r) - m);
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float4 a = __ldcg(reinterpret_cast<const float4*>(from) + ((half * (D / 2) + c) / 4 + x) * kTileRows + r);
                v[4 * x] = __float_as_uint(fmaf(f, a.x, __uint_as_float(v[4 * x])));
                v[4 * x + 1] = __float_as_uint(fmaf(f, a.y, __uint_as_float(v[4 * x + 1])));
                v[4 * x + 2] = __float_as_uint(fmaf(f, a.z, __uint_as_float(v[4 * x + 2])));
                v[4 * x + 3] = __float_as_uint(fmaf(f, a.w, __uint_as_float(v[4 * x + 3])));
              }
            }
          }
          if (live) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // columns of a chunk: dims 0, 4, 1, 5, 2, 6, 3, 7
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e / 2 + e % 2 * 4] = __uint_as_float(v[x * 8 + e]) * inv;
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (p.dtype == SS_F16) {
                  w[e] = pack_h2(f[2 * e], f[2 * e + 1]);
                } else {
                  __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                  w[e] = *reinterpret_cast<uint32_t*>(&b);
                }
              }
              *reinterpret_cast<uint4*>(out + c + x * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (live && p.lse && half == 0) p.lse[tok * p.hq + hd] = l == 0.f ? -INFINITY : (m + log2f(l)) / kLog2e;
        tc_fence_before();
      }
      n0 += nt;
    }
    if (!ok) asm volatile("bar.arrive %0, 64;" ::"r"(pair) : "memory");
  } else if (warp >= kDecWarp) {
    // ================= decode: 64 threads per block of 16 tokens ================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDecRegs));
    while (ok && next_unit(un)) {
      const int nt = un.kt1 - un.kt0;
      const int d = tid - kDecWarp * 32, bi = d >> 6, piece = d & 63;
      constexpr int N = B::N, VW = 2 * B::W;          // key words and value words of a thread
      static_assert(B::G == N, "one key piece per token and lane");
      const int ktok = piece >> 2, kj = piece & 3;    // key piece: a token's words 4 g + kj
      const int vhi = D == 128 ? piece >> 5 : piece & 1, vl = D == 128 ? piece & 31 : piece >> 1;
      const int vi = vl >> 2, vj = vl & 3;            // value piece: tokens 8 vhi + 2 vj, + 1; words W vi ..
      constexpr int DB = kDecWarps / 2, H = kTileKeys / kBlkTokens / DB;  // blocks of a thread: bi, bi + DB, ..
      uint32_t kw[H][N], ks[H][N], vw[H][VW], vs[H][2];
      uint32_t there = 0;  // a bit per block
      int id[H], in_page[H];
      auto look_up = [&](int j) {  // pages of the unit's tile j: a tile before they are needed
#pragma unroll
        for (int hb = 0; hb < H; ++hb) {
          const int k = (un.kt0 + j) * (kTileKeys / kBlkTokens) + bi + DB * hb;
          id[hb] = -1;
          if (j < nt && k * kBlkTokens < un.len) id[hb] = __ldg(p.table + un.b * p.table_stride + page_of(p, k, in_page[hb]));
        }
      };
      auto load = [&]() {  // this thread's pieces of the tile that was looked up
        there = 0;
#pragma unroll
        for (int hb = 0; hb < H; ++hb) {
          if (id[hb] >= 0 && id[hb] < p.n_pages) {
            {
              there |= 1u << hb;
              const uint8_t* blk = p.pages + id[hb] * p.page_stride + un.h * p.head_stride + in_page[hb] * B::kBytes;
              auto get = [](const uint8_t* at, auto& v) {
                if constexpr (sizeof(v) == 16) {
                  const uint4 x = *reinterpret_cast<const uint4*>(at);
                  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                } else {
                  const uint2 x = *reinterpret_cast<const uint2*>(at);
                  v[0] = x.x; v[1] = x.y;
                }
              };
              get(blk + B::key_word(ktok, 0, kj), kw[hb]);
              get(blk + B::key_sz(ktok, 0), ks[hb]);
              get(blk + B::kV + piece * (VW * 4), vw[hb]);
              get(blk + B::value_sz(8 * vhi + 2 * vj, vi * B::W / 4), vs[hb]);
            }
          }
        }
      };
      look_up(0);
      load();
      look_up(1);
      for (int j = 0; j < nt; ++j) {
        const uint32_t n = n0 + j, st = n & 1, ph = (n >> 1) & 1;
        if (!(ok = warp_wait(s_full + st, ph ^ 1))) break;
        uint8_t* stage = smem + st * T::kStage;
        // values go to registers of their own, so that the next tile's loads start here
        uint32_t v_w[H][VW], v_s[H][2];
#pragma unroll
        for (int hb = 0; hb < H; ++hb) {
          const int t0 = (un.kt0 + j) * kTileKeys + (bi + DB * hb) * kBlkTokens;
          const bool have = there >> hb & 1;
          // places without a token yet, or without a page: zeros, whatever their bits
#pragma unroll
          for (int e = 0; e < VW; ++e) v_w[hb][e] = vw[hb][e];
#pragma unroll
          for (int e = 0; e < 2; ++e) v_s[hb][e] = have && t0 + 8 * vhi + 2 * vj + e < un.len ? vs[hb][e] : 0u;
          const bool key = have && t0 + ktok < un.len;
          const int row = (bi + DB * hb) * kBlkTokens + ktok;
          uint8_t* kd = stage + (row >> 3) * 128 + (row & 7) * 16;
#pragma unroll
          for (int g = 0; g < N; ++g) {
            ks[hb][g] = key ? ks[hb][g] : 0u;
            const uint32_t s2 = __byte_perm(ks[hb][g], 0, 0x1010);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = e < 2 ? kw[hb][g] : kw[hb][g] >> 8;
              const uint32_t c = e & 1 ? hsub2(lop_or(x, 0x00f000f0u, 0x50005000u), 0x50005000u)
                                       : hsub2(lop_or(x, 0x000f000fu, 0x60006000u), 0x60006000u);  // c / 2
              hi[e] = hmul2(c, s2);
              lo[e] = hfms2(c, s2, hi[e]);
            }
            *reinterpret_cast<uint4*>(kd + (4 * g + kj) * T::kChunk) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(kd + T::kKey + (4 * g + kj) * T::kChunk) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
          if (kj < 2) {  // zeros of the token's groups, against the sums' hi and against their lo
            uint32_t z[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int g = 0; g < N; g += 2) z[g / 2] = __byte_perm(ks[hb][g], ks[hb][g + 1], 0x7632);
            *reinterpret_cast<uint4*>(stage + 2 * T::kKey + kj * (kTileKeys * 16) + row * 16) = make_uint4(z[0], z[1], z[2], z[3]);
          }
          if (piece == 0) s_hidden[(n & 3) * 8 + bi + DB * hb] = have ? 0 : 1;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full + st);
        load();
        look_up(j + 2);

        if (!(ok = warp_wait(o_done + st, ph ^ 1))) break;
#pragma unroll
        for (int hb = 0; hb < H; ++hb) {
          uint8_t* vd = stage + 2 * T::kKey + T::kZ + ((bi + DB * hb) * 2 + vhi) * (D / 8 * 128) + 2 * vj * 16;
#pragma unroll
          for (int e = 0; e < VW; ++e) {  // word e: token e / W, dim chunk W vi + e % W
            const uint32_t s2 = __byte_perm(v_s[hb][e / B::W], 0, 0x1010), z2 = __byte_perm(v_s[hb][e / B::W], 0, 0x3232);
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t x = q < 2 ? v_w[hb][e] : v_w[hb][e] >> 8;
              const uint32_t c = q & 1 ? hsub2(lop_or(x, 0x00f000f0u, 0x54005400u), 0x54005400u)
                                       : hsub2(lop_or(x, 0x000f000fu, 0x64006400u), 0x64006400u);
              o[q] = hfma2(c, s2, z2);
            }
            *reinterpret_cast<uint4*>(vd + (B::W * vi + e % B::W) * 128 + e / B::W * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + st);
      }
      n0 += nt;
    }
  } else {
    // ================= MMA: a thread issues S, another one O =====================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    // Operands are constants but for the shared memory's base: the instruction takes them from
    // uniform registers, and values that vary cost more to bring there than the MMA itself.
    const uint32_t base = smem_u32(smem) >> 4;
    if (warp == kMmaWarp && lane == 0) {  // S = Q K^T
      uint32_t q_phase = 0;
      while (ok && next_unit(un)) {
        const int nt = un.kt1 - un.kt0;
        if (nt > 0) {
          ok = wait(q_full, q_phase);
          q_phase ^= 1;
        }
        for (int j = 0; j < nt && ok; ++j) {
          const uint32_t n = n0 + j, st = n & 1, ph = (n >> 1) & 1;
          ok = wait(o_done + st, ph ^ 1) && (n != p.skip_tile ? wait(k_full + st, ph) : wait(bars + 12, 0));
          if (!ok) break;
          tc_fence_after();
          if (st == 0) issue_qk<D, 0>(base); else issue_qk<D, 1>(base);
          tc_commit(s_full + st);
        }
        n0 += nt;
      }
    } else if (warp == kMmaWarp + 1 && lane == 0) {  // O += P V
      while (ok && next_unit(un)) {
        const int nt = un.kt1 - un.kt0;
        for (int j = 0; j < nt && ok; ++j) {
          const uint32_t n = n0 + j, st = n & 1, ph = (n >> 1) & 1;
          ok = wait(v_full + st, ph) && wait(p_full + st, ph);
          if (!ok) break;
          tc_fence_after();
          if (st == 0) issue_pv<D, LO, 0>(base, j > 0); else issue_pv<D, LO, 1>(base, j > 0);
          tc_commit(o_done + st);
        }
        n0 += nt;
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*s_abort && (tid == kMmaWarp * 32 || tid == kMmaWarp * 32 + 32)) {  // a wait gave up: what was issued must end before the CTA does
    tc_commit(bars + 12);
    mbar_wait_bounded(bars + 12, 0, 2000000000ull);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tc_dealloc(*s_tmem, T::kCols);
}

template <int D, bool LO, bool SPLIT>
int launch_kernel(AttnParams& p, cudaStream_t st) {
  static_assert(Tile<D>::kSmem <= 227 * 1024, "shared memory");
  const cudaError_t e = cudaFuncSetAttribute(attn_tile_kernel<D, LO, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<D>::kSmem);
  if (e != cudaSuccess) return fail(SS_ERR_CUDA, std::string("ss_int4_attention: ") + cudaGetErrorString(e));
  attn_tile_kernel<D, LO, SPLIT><<<sm_count(), kTileThreads, Tile<D>::kSmem, st>>>(p);
  return check_launch("ss_int4_attention");
}

template <int D, bool LO>
int launch(AttnParams& p, cudaStream_t st) {
  // Both variants are right for any number of units; the one that can cut them along the keys takes
  // 1 to 8 % more time where it cannot (a prompt of 8192: 871 against 860 us bf16, 1066 against 1020
  // fp16), and where it can, 64 query tokens over 30000 keys, 32 heads on 8, take 78 instead of 389 us.
  if (2 * p.tile_units <= sm_count()) return launch_kernel<D, LO, true>(p, st);
  return launch_kernel<D, LO, false>(p, st);
}

}  // namespace

int launch_tiles(AttnParams& p, int d, cudaStream_t st) {
  const bool lo = p.dtype == SS_F16;
  if (d == 64) return lo ? launch<64, true>(p, st) : launch<64, false>(p, st);
  return lo ? launch<128, true>(p, st) : launch<128, false>(p, st);
}

}  // namespace ss
