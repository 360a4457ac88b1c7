// Attention of ragged requests over 4-bit KV pages.
//
// Query row i of a request with q query rows and len keys stands at position
// len - q + i. It sees keys t <= position (causal) and t > position - window
// (window > 0). z_t = scale * q . k_t, p_t = e^(z_t - max z), and
//   out = sum p_t v_t / sum p_t,   lse = max z + ln sum p_t;
// a row that sees no key gives out = 0, lse = -inf.
//
// Split. A unit is (request, kv-head, up to R query rows): the rows share its
// keys, so a block is read once for all of them. The blocks of all units in a
// row are cut into ranges of equal cost, one per CTA (persistent, one or two CTAs
// on an SM). Every unit of a request counts the same keys, those that any of its
// rows sees: right for single tokens; of a long causal prompt (256 dims come here)
// the first units cost less than they count, and of one with a window the last
// units read keys that only the first rows see, and mask them. A unit
// cut by a range boundary leaves partial (o, m, l) rows in the workspace and the
// last CTA to arrive joins them in the order of the ranges, so results do not
// depend on timing. Lengths are read on the GPU: nothing waits for the host.
//
// One warp takes two 16-token blocks at a time (one for D = 256 and for 16 rows,
// whose state fills the registers), with its own ring of cp.async copies (20 D
// contiguous bytes a block) and its own softmax state; the warps meet at the end
// of a unit only. Two CTAs of 6 warps (D = 256: 4) share an SM, so that one joins
// its warps while the other streams; with no more units than SMs it is one of 12 (8).
//   S^T (16 tokens x 8 rows) by warp MMAs. With code c, scale s and zero z of
//   a (token, group): q . k = sum_g s_g (sum_d q_d c_d) + sum_g z_g (sum_d q_d).
//   A nibble masked out of its word is, read as fp16, the subnormal c 2^-24 or
//   c 2^-20: it enters the MMA as it is, the other power of two is in the
//   query's dims, and s_g is applied to the fp32 result, so keys are never
//   rounded. The zeros take one MMA more: z_g as stored against the row's group
//   sums in two fp16 terms.
//   Queries enter as fp16 after a power of two per row that puts the row's
//   largest magnitude in [256, 512): exact for fp16 and bf16 down to 2^-28 of
//   that magnitude.
//   O^T (D x 8 rows) += V^T P^T: two tokens' words are interleaved by byte
//   permutes so that a register holds a dim of two tokens; v = fp16(c s + z),
//   the one rounding of the values. Probabilities are fp16 pairs hi + lo
//   where the output is fp16 (their rounding would otherwise be as large as
//   the output's); for up to 4 rows lo uses the columns that are free anyway.
// The softmax reference of a row moves only when a logit comes 5.5 (base
// 2) above the largest so far: the usual block needs one vote and no shuffles.
//
// Measured (D = 128, 8 kv heads), calls on end for half a second, in brackets bursts
// of graph replays: 1 request of 524288 tokens, 64 heads, fp16 164 us (4.1 TB/s;
// 147 us); 32 requests of 500 to 16384 tokens, bf16 90 us (4.0 TB/s; 86 us); 1 of 777
// tokens 14 us (12 us). HBM would allow 103 and 55 us: a block costs about 340 warp
// instructions, 57 % of the issue slots at that rate, and what is left is
// latency within a warp's block (the registers hold 12 warps an SM). In bursts, one
// block at a time took 163 and 123 us; keys rounded from nibbles to fp16 by
// conversions 179 and 129 us.
#include <algorithm>

#include "int4_attn.cuh"

namespace ss {
namespace {

constexpr int kSegCost = 48;     // blocks' worth of time that the ends of a unit take
constexpr int kMinCost = 96;     // a range is not cut below this many blocks' worth

// Modes: query rows of a unit, and whether probabilities are hi + lo.
enum { kRows4, kRows8, kRows8Lo, kRows16, kRows16Lo };
__host__ __device__ constexpr int mode_rows(int m) { return m == kRows4 ? 4 : m <= kRows8Lo ? 8 : 16; }

// WIDE: one CTA of 12 warps on an SM instead of two of 6 (D = 256: of 8 instead of two of 4).
template <int D, int MODE, bool WIDE>
struct Shape {
  static constexpr int R = mode_rows(MODE);
  static constexpr int NR = R == 16 ? 2 : 1;       // 8-column tiles
  static constexpr bool LO = MODE == kRows8Lo || MODE == kRows16Lo;  // a second MMA for lo
  static constexpr int U = D == 256 || NR == 2 ? 1 : 2;  // blocks a warp takes at a time
  static constexpr int kCtas = (U == 2 || D == 256) && !WIDE ? 2 : 1;  // CTAs on an SM: one joins its warps while the other streams
  static constexpr int W = D == 256 ? (WIDE ? 8 : 4) : U == 1 ? 8 : WIDE ? 12 : 6;   // warps
  static constexpr int S = D == 64 ? 4 : D == 256 ? 3 : U == 2 ? 2 : 4;  // ring stages of a warp
  static constexpr int kRing = W * S * U * Int4Blk<D>::kBytes;
  static constexpr int kMerge = W * R * (D + 4) * 4;  // rows padded by 4 floats
  static constexpr int kSmem = kRing + kMerge + 2 * W * R * 4 + (W * 32 + 1) * 8 + W * 32 * (int)sizeof(Req);
};

// One CTA's walk over its range: unit after unit.
template <int R>
struct Walk {
  int b = 0, h = 0, rb = 0;  // unit
  int64_t at = 0;            // cost position of the unit's start
  Req r{};

  __device__ __forceinline__ int64_t cost() const { return r.nblk + kSegCost; }
  // reqs: the requests, in shared memory, or null where there are more than threads
  __device__ void skip_empty(const AttnParams& p, const Req* reqs) {
    while (b < p.n) {
      r = reqs ? reqs[b] : load_req<R>(p, b);
      if (r.rbs > 0) break;
      ++b;
    }
  }
  __device__ void next(const AttnParams& p, const Req* reqs) {
    at += cost();
    if (++rb < r.rbs) return;
    rb = 0;
    if (++h < p.hkv) return;
    h = 0;
    ++b;
    skip_empty(p, reqs);
  }
};

// D(16x8) += A(16x16) B(16x8) as mma_16816, free to be scheduled among independent ones.
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D = A B
__device__ __forceinline__ void mma0(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <int N>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&v)[N]) {
  if constexpr (N == 2) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = a.x; v[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 a = *reinterpret_cast<const uint4*>(p + 4 * i);
      v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
    }
  }
}

template <int D, int MODE, bool WIDE>
__global__ void __launch_bounds__(Shape<D, MODE, WIDE>::W * 32, Shape<D, MODE, WIDE>::kCtas) attn_decode_kernel(const __grid_constant__ AttnParams p) {
  using B = Int4Blk<D>;
  using Sh = Shape<D, MODE, WIDE>;
  constexpr int R = Sh::R, NR = Sh::NR, W = Sh::W, S = Sh::S, U = Sh::U, G = B::G, N = B::N, T = W * 32;
  constexpr int MT = D / 16;  // 16-dim tiles of O
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem + Sh::kRing);            // [W][R][D + 4]
  float* s_m = s_o + W * R * (D + 4);                                 // [W][R]
  float* s_l = s_m + W * R;                                           // [W][R]
  int64_t* s_cum = reinterpret_cast<int64_t*>(s_l + W * R);           // [T]
  int* s_last = reinterpret_cast<int*>(s_cum + T);                    // this CTA joins the unit's parts
  Req* s_req = reinterpret_cast<Req*>(s_last + 2);                    // [T] the requests, if there are no more

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gi = lane >> 2, gj = lane & 3;
  uint8_t* ring = smem + warp * S * U * B::kBytes;

  // ---- schedule: costs of the requests, thread by thread, then a scan -------
  const int per = (p.n + T - 1) / T;
  const int rb0 = min(p.n, tid * per), rb1 = min(p.n, rb0 + per);
  int64_t cost = 0, units = 0;
  const Req* reqs = per == 1 ? s_req : nullptr;
  const int cq0 = p.cu_q[0], cqn = p.cu_q[p.n];
  for (int b = rb0; b < rb1; ++b) {
    const Req r = load_req<R>(p, b);
    if (per == 1) s_req[b] = r;
    cost += (int64_t)r.rbs * p.hkv * (r.nblk + kSegCost);
    units += (int64_t)r.rbs * p.hkv;
  }
  int64_t inc = cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
    units += __shfl_xor_sync(0xffffffffu, units, o);
  }
  int64_t* s_w = reinterpret_cast<int64_t*>(s_o);  // [W] costs, [W] units
  if (lane == 31) s_w[warp] = inc;
  if (lane == 0) s_w[W + warp] = units;
  __syncthreads();
  int64_t total = 0, before = 0;
  units = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == warp) before = total;
    total += s_w[w];
    units += s_w[W + w];
  }
  s_cum[tid] = before + inc - cost;  // cost of the requests before this thread's
  __syncthreads();
  // tokens outside cu_q: zero rows
  {
    const int64_t first = min((int64_t)max(cq0, 0), p.n_tokens), last = min((int64_t)max(cqn, 0), p.n_tokens);
    const int64_t none = first + p.n_tokens - last, row = (int64_t)p.hq * D / 8;
    for (int64_t i = (int64_t)blockIdx.x * T + tid; i < none * row; i += (int64_t)gridDim.x * T) {
      int64_t t = i / row;
      t = t < first ? t : last + t - first;
      reinterpret_cast<uint4*>(p.out)[t * row + i % row] = make_uint4(0, 0, 0, 0);
      if (p.lse && i % row < p.hq) p.lse[t * p.hq + i % row] = -INFINITY;
    }
  }
  // as many ranges as SMs, but none smaller than a unit or kMinCost
  int64_t want = total < (1 << 22) ? (int64_t)(((uint32_t)total + kMinCost + kSegCost - 1) / (uint32_t)(kMinCost + kSegCost))
                                   : (total + kMinCost + kSegCost - 1) / (kMinCost + kSegCost);
  want = want < units ? units : want;
  const int nc = (int)(want < gridDim.x ? want : (int64_t)gridDim.x);
  if ((int)blockIdx.x >= nc) {
    grid_dependency_wait();
    return;
  }
  // (64-bit divisions take some 100 cycles each, and these stand before the first copy)
  const bool small = total < (1 << 22);  // products with nc + 1 <= 2 * 148 + 1 stay below 2^31
  auto range_start = [&](int i) -> int64_t {
    return small ? (int64_t)((uint32_t)i * (uint32_t)total / (uint32_t)nc) : i * total / nc;
  };
  auto cta_of = [&](int64_t c) {  // the range that holds c
    return small ? (int)(((uint32_t)(c + 1) * (uint32_t)nc - 1) / (uint32_t)total) : (int)(((c + 1) * nc - 1) / total);
  };
  const int64_t lo = range_start(blockIdx.x), hi = range_start(blockIdx.x + 1);

  Walk<R> walk;
  {
    int a = 0, e = T;  // the last thread whose requests start at or before lo
    while (e - a > 1) {
      const int mid = (a + e) >> 1;
      if (s_cum[mid] <= lo) a = mid; else e = mid;
    }
    walk.b = min(p.n, a * per);
    walk.at = s_cum[a];
    walk.skip_empty(p, reqs);
    for (;;) {
      const int64_t one = walk.cost(), all = one * walk.r.rbs * p.hkv;
      if (walk.at + all > lo) {
        const int64_t u = small ? (int64_t)((uint32_t)(lo - walk.at) / (uint32_t)one) : (lo - walk.at) / one;
        walk.h = (int)((uint32_t)u / (uint32_t)walk.r.rbs);
        walk.rb = (int)(u - (int64_t)walk.h * walk.r.rbs);
        walk.at += u * one;
        break;
      }
      walk.at += all;
      ++walk.b;
      walk.skip_empty(p, reqs);
    }
  }

  // key blocks [k0, k1) of the walk's unit that this CTA's range covers
  auto blocks = [&](const Walk<R>& w, int& k0, int& k1) {
    const int64_t body = w.at + kSegCost;
    const int64_t a = (lo > body ? lo : body) - body, e = (hi < body + w.r.nblk ? hi : body + w.r.nblk) - body;
    k0 = w.r.blk0 + (int)a;
    k1 = e > a ? w.r.blk0 + (int)e : k0;
    if (p.causal) {  // nothing after the last row of the unit
      const int last_row = (int)min((int64_t)w.r.nq * p.grp, (int64_t)(w.rb + 1) * R) - 1;
      const int end = min(w.r.len, w.r.len - w.r.nq + last_row / p.grp + 1);
      k1 = max(k0, min(k1, (max(end, 0) + kBlkTokens - 1) / kBlkTokens));
    }
    if (w.r.len == 0) k1 = k0;
    return e > a;  // this CTA takes part in the unit
  };

  // ---- copies: this warp's blocks in the order it will use them -------------
  Walk<R> pw = walk;
  int pk = 0, pk1 = 0, pn = 32;
  int64_t poff = 0;      // a lane's block among the next 32: its offset in the pool, -1 if it has none
  uint32_t hidden = 0;   // a bit per issued block: its table entry is outside the pool
  bool more = true;
  auto open = [&]() {  // the next unit in which this warp has a block
    while (true) {
      if (pw.b >= p.n || pw.at >= hi) { more = false; return; }
      blocks(pw, pk, pk1);
      pk += warp * U;
      pn = 32;
      if (pk < pk1) return;
      pw.next(p, reqs);
    }
  };
  open();
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
  auto issue = [&](int stage) {
    if (more) {
      if (pn == 32) {
        const int k = pk + lane / U * (W * U) + lane % U;
        int in_page;
        poff = -1;
        if (k < pk1) {
          const int id = p.table[pw.b * p.table_stride + page_of(p, k, in_page)];
          if (id >= 0 && id < p.n_pages) poff = id * p.page_stride + pw.h * p.head_stride + in_page * B::kBytes;
        }
        pn = 0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t off = __shfl_sync(0xffffffffu, poff, pn++);
        const uint8_t* src = p.pages + off + lane * 16;
        const uint32_t dst = ring_at + (stage * U + u) * B::kBytes;
        hidden <<= 1;
        if (off >= 0) {
#pragma unroll
          for (int i = 0; i < B::kBytes / 512; ++i) cp_async16(dst + i * 512, src + i * 512, 16);
          if (B::kBytes % 512 && lane < B::kBytes % 512 / 16) cp_async16(dst + B::kBytes / 512 * 512, src + B::kBytes / 512 * 512, 16);
        } else {  // no such block: zeros
          hidden |= 1u;
#pragma unroll
          for (int i = lane; i < B::kBytes / 16; i += 32) cp_async16(dst + (i - lane) * 16, p.pages, 0);
        }
      }
      pk += W * U;
      if (pk >= pk1) {
        pw.next(p, reqs);
        open();
      }
    } else {
      hidden <<= U;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(s);
  int stage = 0;

  // ---- unit after unit --------------------------------------------------------
  for (; walk.b < p.n && walk.at < hi; walk.next(p, reqs)) {
    int k0, k1;
    const bool part = blocks(walk, k0, k1);
    const Req r = walk.r;
    const int b = walk.b, tok0 = max(p.cu_q[b], 0);
    const int row0 = walk.rb * R, rows = min(R, (int)((int64_t)r.nq * p.grp - row0));
    if (!part) continue;  // uniform over the CTA: the range ends inside the unit's fixed cost

    // queries as B fragments: lane (i, j) holds dims 32 g + 8 j .. + 7 of row i
    uint32_t qf[NR][G][4];
    float fac[NR][2];
    uint32_t qz[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int col = nr * 8 + gi, row = MODE == kRows4 ? (col & 3) : col;
      float x[G][8], big = 0.f;
      const int tt = (row0 + row) / p.grp, hd = walk.h * p.grp + (row0 + row) % p.grp;
      const bool live = row < rows && tok0 + (int64_t)tt < p.n_tokens;
      const int64_t at = (tok0 + (int64_t)tt) * p.q_st + hd * p.q_sh + gj * 8;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + at;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t u[4] = {0u, 0u, 0u, 0u};
        if (live) {
          if (p.q_vec) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(qp + g * 32));
            u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = qp[g * 32 + 2 * e] | (uint32_t)qp[g * 32 + 2 * e + 1] << 16;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[g][2 * e] = p.dtype == SS_F16 ? lo_h(u[e]) : __uint_as_float(u[e] << 16);
          x[g][2 * e + 1] = p.dtype == SS_F16 ? hi_h(u[e]) : __uint_as_float(u[e] & 0xffff0000u);
          big = fmaxf(big, fmaxf(fabsf(x[g][2 * e]), fabsf(x[g][2 * e + 1])));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // 2^e with big * 2^e in [256, 512); 1 for rows of zeros or infinities
      int ex = 0;
      if (big > 0.f && big < INFINITY) ex = 135 - (int)(__float_as_uint(fmaxf(big, 1.2e-38f)) >> 23);
      const float up = ex > 126 ? __uint_as_float(253u << 23) : __uint_as_float((uint32_t)(127 + ex) << 23);
      float sum[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        sum[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // a register: dims e and e + 4, as the key words' nibbles come
          qf[nr][g][e] = pack_h2(x[g][e] * up, x[g][e + 4] * up);
          sum[g] += lo_h(qf[nr][g][e]) + hi_h(qf[nr][g][e]);
          if (e & 1) qf[nr][g][e] = hmul2(qf[nr][g][e], 0x2c002c00u);  // 2^-4: those codes come as 2^-20
        }
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
      }
      // group sums as the B fragment of the zeros' MMA: k = group hi, k + 8 = group lo
      float z0 = 0.f, z1 = 0.f;
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        if (gj == g / 2) { z0 = sum[g]; z1 = sum[g + 1]; }
      }
      qz[nr][0] = pack_h2(z0, z1);
      qz[nr][1] = pack_h2(z0 - lo_h(qz[nr][0]), z1 - hi_h(qz[nr][0]));
      const float back = p.scale * (kLog2e * 0x1p24f) / up;
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // the columns of this lane's accumulators
        const int cc = 2 * gj + c, from = cc * 4;
        fac[nr][c] = __shfl_sync(0xffffffffu, back, from);
      }
    }
    // keys [beg, end) that a column's row sees
    auto sees = [&](int nr, int c, int& beg, int& end) {
      const int cc = 2 * gj + c, rr = MODE == kRows4 ? (cc & 3) : nr * 8 + cc;
      const int pos = r.len - r.nq + (row0 + rr) / p.grp;
      end = rr >= rows ? 0 : p.causal ? min(r.len, pos + 1) : r.len;
      beg = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      return rr < rows;
    };
    // blocks in [all0, all1) are seen whole by every row of the unit
    int all0 = 0, all1 = 0x7fffffff;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        int beg, end;
        if (sees(nr, c, beg, end)) {
          all0 = max(all0, beg);
          all1 = min(all1, end);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all0 = max(all0, __shfl_xor_sync(0xffffffffu, all0, o));
      all1 = min(all1, __shfl_xor_sync(0xffffffffu, all1, o));
    }

    const int full0 = (all0 + kBlkTokens - 1) / kBlkTokens, full_n = max(0, all1 / kBlkTokens - full0);

    float o[NR][MT][4], m[NR][2], l[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nr][t][e] = 0.f;
      }
      m[nr][0] = m[nr][1] = kLow;
      l[nr][0] = l[nr][1] = 0.f;
    }

    for (int k = k0 + warp * U; k < k1; k += W * U) {
      const uint32_t gone = hidden >> ((S - 2) * U);  // bit U - 1 - u: block u is not there
      const bool edge = (uint32_t)(k - full0) >= (uint32_t)full_n || k + U > full0 + full_n || (gone & ((1u << U) - 1)) != 0;
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
      __syncwarp();
      issue(stage == 0 ? S - 1 : stage - 1);
      const uint8_t* blk0 = ring + stage * U * B::kBytes;
      stage = stage == S - 1 ? 0 : stage + 1;
      const int t0 = k * kBlkTokens;

      // ---- logits: S^T = K Q^T ----
      float s[U][NR][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint8_t* blk = blk0 + u * B::kBytes;
        uint32_t z[2] = {0u, 0u};  // zeros of tokens i, i + 8: groups 2j, 2j + 1
        if (2 * gj < G) {
          uint32_t a[2], c[2];
          lds(blk + B::key_sz(gi, 2 * gj), a);
          lds(blk + B::key_sz(gi + 8, 2 * gj), c);
          z[0] = __byte_perm(a[0], a[1], 0x7632);
          z[1] = __byte_perm(c[0], c[1], 0x7632);
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          mma0(s[u][nr], z[0], z[1], z[0], z[1], qz[nr][0], qz[nr][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][nr][e] *= 0x1p-24f;  // the codes' power of two
        }
#pragma unroll
        for (int c = 0; c < G / N; ++c) {
          uint32_t w0[N], w1[N], z0[N], z1[N];
          lds(blk + B::key_word(gi, c * N, gj), w0);
          lds(blk + B::key_word(gi + 8, c * N, gj), w1);
          lds(blk + B::key_sz(gi, c * N), z0);
          lds(blk + B::key_sz(gi + 8, c * N), z1);
#pragma unroll
          for (int g = 0; g < N; ++g) {
            uint32_t h0[4], h1[4];  // codes of dims (e, e + 4) times 2^-24 (even e) or 2^-20
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h0[e] = (e < 2 ? w0[g] : w0[g] >> 8) & (e & 1 ? 0x00f000f0u : 0x000f000fu);
              h1[e] = (e < 2 ? w1[g] : w1[g] >> 8) & (e & 1 ? 0x00f000f0u : 0x000f000fu);
            }
            const float s0 = lo_h(z0[g]), s1 = lo_h(z1[g]);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
              float a[4];
              mma0(a, h0[0], h1[0], h0[1], h1[1], qf[nr][c * N + g][0], qf[nr][c * N + g][1]);
              mma(a, h0[2], h1[2], h0[3], h1[3], qf[nr][c * N + g][2], qf[nr][c * N + g][3]);
              s[u][nr][0] = fmaf(s0, a[0], s[u][nr][0]);
              s[u][nr][1] = fmaf(s0, a[1], s[u][nr][1]);
              s[u][nr][2] = fmaf(s1, a[2], s[u][nr][2]);
              s[u][nr][3] = fmaf(s1, a[3], s[u][nr][3]);
            }
          }
        }
      }

      // ---- probabilities ----
      uint32_t ph[U][NR][2], pl[U][NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        float y[U][4], over = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[u][e] = fmaf(s[u][nr][e], fac[nr][e & 1], -m[nr][e & 1]);
        }
        if (edge) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            int beg, end;
            sees(nr, c, beg, end);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
              for (int e = c; e < 4; e += 2) {
                const int t = t0 + u * kBlkTokens + gi + (e >> 1) * 8;
                if ((gone >> (U - 1 - u) & 1) || t >= end || t < beg) y[u][e] = -INFINITY;
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) over = fmaxf(over, fmaxf(fmaxf(y[u][0], y[u][2]), fmaxf(y[u][1], y[u][3])));
        if (__any_sync(0xffffffffu, over > kSlack)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
              for (int e = c; e < 4; e += 2) {
                y[u][e] = y[u][e] == -INFINITY ? y[u][e] : s[u][nr][e] * fac[nr][c];
                top = fmaxf(top, y[u][e]);
              }
            }
#pragma unroll
            for (int sft = 4; sft < 32; sft <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sft));
            const float mn = fmaxf(m[nr][c], top - kBelow), f = ex2(m[nr][c] - mn);
            m[nr][c] = mn;
            l[nr][c] *= f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              y[u][c] -= mn;
              y[u][c + 2] -= mn;
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              o[nr][t][c] *= f;
              o[nr][t][c + 2] *= f;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[u][e] = ex2(y[u][e]);
          l[nr][0] += y[u][0] + y[u][2];
          l[nr][1] += y[u][1] + y[u][3];
          uint32_t a = pack_h2(y[u][0], y[u][1]), c = pack_h2(y[u][2], y[u][3]);
          if constexpr (MODE == kRows4) {  // columns 4-7 repeat rows 0-3: they take lo
            const uint32_t al = pack_h2(y[u][0] - lo_h(a), y[u][1] - hi_h(a)), cl = pack_h2(y[u][2] - lo_h(c), y[u][3] - hi_h(c));
            a = gj < 2 ? a : al;
            c = gj < 2 ? c : cl;
          }
          ph[u][nr][0] = transpose8x8(a);
          ph[u][nr][1] = transpose8x8(c);
          if constexpr (Sh::LO) {
            pl[u][nr][0] = transpose8x8(pack_h2(y[u][0] - lo_h(a), y[u][1] - hi_h(a)));
            pl[u][nr][1] = transpose8x8(pack_h2(y[u][2] - lo_h(c), y[u][3] - hi_h(c)));
          }
        }
      }

      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint8_t* blk = blk0 + u * B::kBytes;
        uint32_t vz[4], vw[4 * B::W];
        lds(blk + B::value_sz(2 * gj, gi * B::W / 4), vz);
#pragma unroll
        for (int c = 0; c < B::W; ++c) {
          uint32_t t4[4];
          lds(blk + B::kV + c * 512 + lane * 16, t4);
#pragma unroll
          for (int e = 0; e < 4; ++e) vw[4 * c + e] = t4[e];
        }
        if (edge) {  // places that hold no token yet: whatever bits they have
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t0 + u * kBlkTokens + 2 * gj + (e >> 1) * 8 + (e & 1) >= r.len) vz[e] = 0u;
        }
        uint32_t sc[2], zr[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          sc[hh] = __byte_perm(vz[2 * hh], vz[2 * hh + 1], 0x5410);
          zr[hh] = __byte_perm(vz[2 * hh], vz[2 * hh + 1], 0x7632);
        }
#pragma unroll
        for (int wi = 0; wi < B::W; ++wi) {
          uint32_t x[2][2];  // [hi][dims 0-3 | 4-7]: two tokens' nibbles side by side
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const uint32_t a = vw[(hh * 2) * B::W + wi], c = vw[(hh * 2 + 1) * B::W + wi];
            x[hh][0] = __byte_perm(a, c, 0x5410);
            x[hh][1] = __byte_perm(a, c, 0x7632);
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // a0: hi 0, dim n; a1: dim n + 4; a2, a3: hi 1
              const uint32_t xx = x[e >> 1][e & 1] >> (8 * (n >> 1));
              const uint32_t c = n & 1 ? hsub2(lop_or(xx, 0x00f000f0u, 0x54005400u), 0x54005400u)
                                       : hsub2(lop_or(xx, 0x000f000fu, 0x64006400u), 0x64006400u);
              a[e] = hfma2(c, sc[e >> 1], zr[e >> 1]);
            }
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
              mma(o[nr][wi * 4 + n], a[0], a[1], a[2], a[3], ph[u][nr][0], ph[u][nr][1]);
              if constexpr (Sh::LO) mma(o[nr][wi * 4 + n], a[0], a[1], a[2], a[3], pl[u][nr][0], pl[u][nr][1]);
            }
          }
        }
      }
      __syncwarp();
    }

    // ---- join the warps -------------------------------------------------------
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[nr][c] += __shfl_xor_sync(0xffffffffu, l[nr][c], sft);
        const int row = nr * 8 + 2 * gj + c;
        const bool mine = MODE != kRows4 || gj < 2;
        if (MODE == kRows4) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            o[nr][t][c] += __shfl_xor_sync(0xffffffffu, o[nr][t][c], 2);
            o[nr][t][c + 2] += __shfl_xor_sync(0xffffffffu, o[nr][t][c + 2], 2);
          }
        }
        if (mine) {
          float* dst = s_o + (warp * R + row) * (D + 4);
#pragma unroll
          for (int t = 0; t < MT; ++t) {  // place 16 t + 8 h + i: a warp's stores go to 32 banks
            dst[16 * t + gi] = o[nr][t][c];
            dst[16 * t + 8 + gi] = o[nr][t][c + 2];
          }
          if (gi == 0) {
            s_m[warp * R + row] = m[nr][c];
            s_l[warp * R + row] = l[nr][c];
          }
        }
      }
    }
    __syncthreads();
    const int64_t body = walk.at + kSegCost;
    const int c_first = cta_of(body), c_last = cta_of(body + r.nblk - 1);
    const bool whole = c_first == c_last;
    constexpr int kPart = R * (D + 2);
    // a CTA leaves at most two parts: of the unit it starts in (the first slot), and of the one it
    // ends in; only a unit's first CTA can have started in another one
    const int first_slot = range_start(c_first) >= walk.at ? 0 : 1;
    auto slot_of = [&](int c) { return p.parts + (size_t)(2 * c + (c == c_first ? first_slot : 0)) * kPart; };
    float* mine = whole ? nullptr : slot_of(blockIdx.x);
    auto finish = [&](int row, int dim, float4 v, float mm, float ll) {  // 4 dims of a row
      const int rr = row0 + row, hd = walk.h * p.grp + rr % p.grp;
      const int64_t t = tok0 + (int64_t)(rr / p.grp);
      if (t >= p.n_tokens) return;
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      const int64_t at = (t * p.hq + hd) * D + dim;
      uint2 u;
      if (p.dtype == SS_F16) {
        u = make_uint2(pack_h2(v.x * inv, v.y * inv), pack_h2(v.z * inv, v.w * inv));
      } else {
        __nv_bfloat162 a = __floats2bfloat162_rn(v.x * inv, v.y * inv), c = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        u = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&c));
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = u;
      if (p.lse && dim == 0) p.lse[t * p.hq + hd] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) / kLog2e;
    };
    for (int e = tid; e < rows * (D / 4); e += T) {
      const int row = e / (D / 4), dim = e % (D / 4) * 4;
      float mm = kLow, ll = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_m[w * R + row]);
      // dims 8 (i W + wi) + 4 h + n are in tile 4 wi + n
      const int x = dim / 8, at = x % B::W * 64 + dim / 4 % 2 * 8 + x / B::W;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = ex2(s_m[w * R + row] - mm);
        ll = fmaf(f, s_l[w * R + row], ll);
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] = fmaf(f, s_o[(w * R + row) * (D + 4) + at + 16 * n], v[n]);
      }
      const float4 v4 = make_float4(v[0], v[1], v[2], v[3]);
      if (whole) {
        finish(row, dim, v4, mm, ll);
      } else {
        __stcg(reinterpret_cast<float4*>(mine + row * D + dim), v4);
        if (dim == 0) {
          __stcg(mine + R * D + row, mm);
          __stcg(mine + R * D + R + row, ll);
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        uint32_t* cnt = reinterpret_cast<uint32_t*>(p.ws) + c_first;
        const uint32_t parts_n = c_last - c_first + 1;
        const uint32_t seen = atomicAdd(cnt, 1u);
        if (seen == parts_n - 1) *cnt = 0u;  // every part is in: the counter is ready for the next launch
        __threadfence();
        *s_last = seen == parts_n - 1;
      }
      __syncthreads();
      if (*s_last) {
        for (int e = tid; e < rows * (D / 4); e += T) {
          const int row = e / (D / 4), dim = e % (D / 4) * 4;
          float mm = kLow, ll = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = c_first; c <= c_last; ++c) {
            const float* src = slot_of(c);
            const float m2 = __ldcg(src + R * D + row), l2 = __ldcg(src + R * D + R + row);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src + row * D + dim));
            const float mn = fmaxf(mm, m2), f1 = ex2(mm - mn), f2 = ex2(m2 - mn);
            mm = mn;
            ll = f1 * ll + f2 * l2;
            v.x = f1 * v.x + f2 * x.x; v.y = f1 * v.y + f2 * x.y; v.z = f1 * v.z + f2 * x.z; v.w = f1 * v.w + f2 * x.w;
          }
          finish(row, dim, v, mm, ll);
        }
      }
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // The tile kernel of the same call may still run beside this one (programmatic dependent launch):
  // this grid ends after it, so that what follows on the stream finds both results.
  grid_dependency_wait();
}

// Workspace: a counter per CTA, then two parts per CTA of R rows of D + 2 floats
// (up to 16 rows for one CTA on an SM, up to 8 for two), and the same again for the tile kernel,
// which may run beside. Launches of every shape share it, so the counters' room is that of the
// most CTAs: a part never lies over a counter.
size_t attn_counter_bytes(int sms) { return ((size_t)sms * 2 * 4 + 15) / 16 * 16; }
size_t attn_part_bytes(int d, int sms) { return (size_t)sms * 2 * 16 * (d + 2) * 4; }
size_t attn_ws_bytes(int d, int sms) {
  return 2 * attn_counter_bytes(sms) + attn_part_bytes(d, sms) + (d == 256 ? 0 : (size_t)sms * tile_part_floats(d) * 4);
}

template <int D, int MODE, bool WIDE>
int launch_shape(AttnParams& p, cudaStream_t st) {
  using Sh = Shape<D, MODE, WIDE>;
  static_assert(Sh::kSmem <= 227 * 1024 / Sh::kCtas, "shared memory");
  const cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<D, MODE, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
  if (e != cudaSuccess) return fail(SS_ERR_CUDA, std::string("ss_int4_attention: ") + cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count() * Sh::kCtas);
  cfg.blockDim = dim3(Sh::W * 32);
  cfg.dynamicSmemBytes = Sh::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.tiles ? 1 : 0;  // beside the tile kernel: the two write different rows
  const cudaError_t e2 = cudaLaunchKernelEx(&cfg, attn_decode_kernel<D, MODE, WIDE>, p);
  if (e2 != cudaSuccess) {
    cudaGetLastError();
    return fail(SS_ERR_CUDA, std::string("ss_int4_attention: ") + cudaGetErrorString(e2));
  }
  return check_launch("ss_int4_attention");
}

template <int D, int MODE>
int launch_decode(AttnParams& p, int64_t most, cudaStream_t st) {
  if constexpr (Shape<D, MODE, false>::kCtas == 2) {
    // No more units than SMs: nothing to overlap the joins with, and a short unit is done in fewer
    // rounds by all warps (one request of 777 tokens 13.0 -> 12.2 us, one of 524288 156 -> 149 us; D =
    // 256, 32 heads on 8: 17 query tokens over 4000 keys 50 -> 35 us). With more it is the other way
    // round: D = 256, a prompt of 1000 tokens 412 -> 314 us, 8 of 180 tokens 323 -> 203 us.
    constexpr int R = mode_rows(MODE);
    if (std::min(p.n_tokens * p.grp / R + p.n, (most + R - 1) / R * p.n) * p.hkv <= sm_count()) return launch_shape<D, MODE, true>(p, st);
  }
  return launch_shape<D, MODE, false>(p, st);
}

template <int D>
int launch_mode(AttnParams& p, int64_t most, cudaStream_t st) {  // most: rows of a request
  const bool lo = p.dtype == SS_F16;
  if (most <= 4) return launch_decode<D, kRows4>(p, most, st);
  // D = 256: 16 rows spill (a prompt of 1000 tokens 427 us where 8 took 412, 17 query tokens 63 and 35)
  if (most <= 8 || D == 256) return lo ? launch_decode<D, kRows8Lo>(p, most, st) : launch_decode<D, kRows8>(p, most, st);
  if constexpr (D != 256) return lo ? launch_decode<D, kRows16Lo>(p, most, st) : launch_decode<D, kRows16>(p, most, st);
  return SS_OK;
}

}  // namespace
}  // namespace ss

using namespace ss;

extern "C" {

size_t ss_int4_attention_workspace(int d) { return attn_ws_bytes(d, sm_count()); }

size_t ss_int4_attention_counters(void) { return 2 * attn_counter_bytes(sm_count()); }

int ss_int4_attention(const ss_int4_attn_args* a, void* stream) {
  return c_entry([&]() -> int {
    SS_REQUIRE(a, "ss_int4_attention: null pointer");
    if (a->n_tokens == 0) return SS_OK;
    SS_REQUIRE(a->q && a->pages && a->block_table && a->seq_lens && a->cu_q && a->out,
               "ss_int4_attention: null pointer");
    SS_REQUIRE(a->dtype == SS_F16 || a->dtype == SS_BF16, "ss_int4_attention: queries must be fp16 or bf16");
    SS_REQUIRE(int4_head_dim_ok(a->d), "ss_int4_attention: head_dim must be 64, 128 or 256");
    SS_REQUIRE(a->hkv >= 1 && a->hq >= 1 && a->hq % a->hkv == 0,
               "ss_int4_attention: the query heads must be a multiple of the kv heads");
    SS_REQUIRE(a->n_tokens > 0 && a->n_requests >= 1 && a->n_pages >= 1 && a->width >= 1,
               "ss_int4_attention: empty batch, pool or table");
    SS_REQUIRE(a->page_size >= 16 && a->page_size % 16 == 0,
               "ss_int4_attention: page_size must be a multiple of 16");
    SS_REQUIRE((int64_t)a->width * a->page_size <= 0x7fffffff - 256,
               "ss_int4_attention: a table row must hold fewer than 2^31 tokens");
    SS_REQUIRE(((reinterpret_cast<uintptr_t>(a->pages) | (uintptr_t)a->page_stride | (uintptr_t)a->head_stride) & 15) == 0,
               "ss_int4_attention: the pool and its strides must be multiples of 16 bytes");
    SS_REQUIRE((reinterpret_cast<uintptr_t>(a->out) & 15) == 0, "ss_int4_attention: out must be 16-byte aligned");
    SS_REQUIRE(a->window >= 0 && a->max_q >= 1, "ss_int4_attention: window must not be negative, max_q positive");
    const int ctas = sm_count();
    if (!a->workspace || a->workspace_bytes < attn_ws_bytes(a->d, ctas) || (reinterpret_cast<uintptr_t>(a->workspace) & 15))
      return fail(SS_ERR_WORKSPACE, "ss_int4_attention: workspace null, too small or not 16-byte aligned");
    count_dispatch("ss_int4_attention");
    AttnParams p{};
    p.q = a->q; p.dtype = a->dtype; p.q_st = a->q_token_stride; p.q_sh = a->q_head_stride;
    p.q_vec = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(a->q_token_stride * 2) | (uintptr_t)(a->q_head_stride * 2)) & 15) == 0;
    p.n_tokens = a->n_tokens; p.hq = a->hq; p.hkv = a->hkv; p.grp = a->hq / a->hkv;
    p.pages = static_cast<const uint8_t*>(a->pages); p.n_pages = a->n_pages;
    p.page_stride = a->page_stride; p.head_stride = a->head_stride; p.page = a->page_size;
    p.page_blocks = a->page_size / kBlkTokens;
    p.page_inv = p.page_blocks == 1 ? 0u : (uint32_t)(((1ull << 32) + p.page_blocks - 1) / p.page_blocks);
    p.table = a->block_table; p.table_stride = a->table_stride; p.width = a->width;
    p.seq_lens = a->seq_lens; p.cu_q = a->cu_q; p.n = a->n_requests;
    // A window that no position exceeds hides nothing; without it, differences of positions and
    // windows stay far inside 32 bits (positions go down to minus the query tokens).
    const bool windowed = a->window > 0 && (int64_t)a->window < (int64_t)a->width * a->page_size;
    p.scale = a->scale; p.causal = a->causal; p.window = windowed ? a->window : 0;
    p.out = a->out; p.lse = a->lse;
    p.ws = static_cast<uint8_t*>(a->workspace);
    p.tile_ws = reinterpret_cast<uint32_t*>(p.ws + attn_counter_bytes(ctas));
    p.parts = reinterpret_cast<float*>(p.ws + 2 * attn_counter_bytes(ctas));
    p.tile_parts = reinterpret_cast<float*>(p.ws + 2 * attn_counter_bytes(ctas) + attn_part_bytes(a->d, ctas));
    const int64_t most = (int64_t)a->max_q * p.grp;
    p.tiles = most > 16 && a->d != 256;
    // The host does not know the lengths: a request's rows over 128, and one more for each request
    // with enough rows, or max_q's tiles for each. The hint may be wrong: it chooses a variant.
    const int64_t all_rows = p.n_tokens * p.grp;
    p.tile_units = std::min(all_rows / 128 + std::min<int64_t>(p.n, all_rows / 17), (most + 127) / 128 * p.n) * p.hkv;
    p.sink = error_sink();
    p.wait_ns = a->wait_limit_ns > 0 ? (uint64_t)a->wait_limit_ns : 2000000000ull;
    p.skip_tile = a->test_skip_tile > 0 ? (uint32_t)(a->test_skip_tile - 1) : 0xffffffffu;
    cudaStream_t st = as_stream(stream);
    if (p.tiles) {
      if (int rc = launch_tiles(p, a->d, st)) return rc;
    }
    return a->d == 64 ? launch_mode<64>(p, most, st) : a->d == 128 ? launch_mode<128>(p, most, st) : launch_mode<256>(p, most, st);
  });
}

}  // extern "C"
