// Log probabilities of given tokens, entropy and the k most probable tokens
// of each row of logits.
//
// M = max x, l = sum e^(x_i - M), A = sum e^(x_i - M) (x_i - M):
//   log p_i = x_i - M - ln l,   entropy = ln l - A / l.
// (Differences are taken before the change to base 2 for the hardware's exp2:
// x log2(e) overflows at the lowest values that masks use.)
// The k largest by (value descending, index ascending).
//
// A row whose logits are all -inf has no distribution: log p = -inf,
// entropy 0. A row that holds NaN or +inf gives NaN, and ids -1.
// A target < 0 gives 0 (padding), one >= vocab NaN.
//
// One pass over a row, by a CTA or, for few rows, by a cluster whose CTAs push
// their results into the first one's shared memory. A thread keeps
// (M, l, A) of its own elements in fp32 and rescales only when 16 new ones
// raise its maximum. The k-th largest of the threads' maxima bounds the k-th
// largest element from below, so only the few threads whose maximum reaches it
// hold candidates: their elements alone are read again (3 % of a row at k =
// 8, in whole sectors), by all threads together, and ranked against each other. Where more
// elements reach the bound than are listed (a constant row), those above it are
// listed and the first equal ones taken in order.
//
// Bound by HBM; an element costs about 5.5 issue slots, one of them exp2, at
// half of what an SM can issue at full bandwidth. 256 threads and five CTAs an
// SM, so that rows in their last phase overlap rows that stream: 2047 x 128256
// bf16, top 8: calls on end 110 to 114 us (4.7 TB/s), bursts of graph replays 104 to
// 106 us; with loads of 16 bytes, of whose sectors the second reading used half,
// 109 us in bursts, and then 112 with 512 threads and two CTAs. 333 x 50257 fp32,
// top 5: 16 us, and 17 to 21 with the host's calls; one row of 128256: 10 us, latency.
#include <cooperative_groups.h>

#include "common.cuh"

namespace ss {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSplit = 8;
constexpr int kLpCap = 1024;     // candidates of a CTA
constexpr int kLpVec = 32;       // bytes of a load: a whole sector, so that reading elements again wastes none
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e30f;   // stands for -inf in differences: its exponential is 0, times it is 0

struct LpParams {
  const void* x;
  int64_t rows, row_stride;
  int vocab;
  const int64_t* targets;
  int top;
  float *logprobs, *entropy, *top_lp;
  int32_t* top_ids;
};

struct Sums {
  float m, l, a;
};

__device__ __forceinline__ float lp_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ Sums merge(const Sums& x, const Sums& y) {
  Sums r;
  r.m = fmaxf(x.m, y.m);
  const float d1 = fmaxf(x.m - r.m, kFar), d2 = fmaxf(y.m - r.m, kFar);
  const float e1 = lp_ex2(d1 * kLog2e), e2 = lp_ex2(d2 * kLog2e);
  r.l = e1 * x.l + e2 * y.l;
  r.a = e1 * (x.a + d1 * x.l) + e2 * (y.a + d2 * y.l);
  return r;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Unsigned integers in the order of the floats (-0 and +0 alike).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ bool before(uint32_t k, int i, uint32_t k2, int i2) {  // ranks first
  return k > k2 || (k == k2 && i < i2);
}

struct Words {
  uint32_t w[8];
};
__device__ __forceinline__ Words load32(const void* p) {
  Words r;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
               : "l"(p));
  return r;
}

template <int DT>
struct Vec {
  static constexpr int E = DT == SS_F32 ? 8 : 16;  // elements of a load
  static __device__ __forceinline__ void get(const Words& u, float (&x)[E]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == SS_F32) {
        x[i] = __uint_as_float(u.w[i]);
      } else if constexpr (DT == SS_BF16) {
        x[2 * i] = __uint_as_float(u.w[i] << 16);
        x[2 * i + 1] = __uint_as_float(u.w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u.w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

// (a, b) op (x, y) as packed fp32
__device__ __forceinline__ void fma_f32x2(float& a, float& b, float x0, float x1, float y0, float y1) {
  asm("{\n .reg .b64 t, u, v;\n mov.b64 t, {%0, %1};\n mov.b64 u, {%2, %3};\n mov.b64 v, {%4, %5};\n"
      " fma.rn.f32x2 t, u, v, t;\n mov.b64 {%0, %1}, t;\n}"
      : "+f"(a), "+f"(b)
      : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}

// Adds n elements to the sums; m already covers them.
template <int N>
__device__ __forceinline__ void add_up(const float (&x)[N], float m, float (&l)[2], float (&a)[2]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float d0 = x[i], d1 = x[i + 1];
    add_f32x2(d0, d1, -m, -m);
    d0 = fmaxf(d0, kFar);  // -inf, and -inf - -inf
    d1 = fmaxf(d1, kFar);
    float t0 = d0, t1 = d1;
    mul_f32x2(t0, t1, kLog2e);
    const float e0 = lp_ex2(t0), e1 = lp_ex2(t1);
    add_f32x2(l[0], l[1], e0, e1);
    fma_f32x2(a[0], a[1], e0, e1, d0, d1);
  }
}

struct LpShared {
  Sums warp[kLpWarps];
  Sums sums;                     // this CTA's
  float tmax[kLpThreads];        // the threads' maxima
  uint32_t key[kLpCap];          // candidates
  int idx[kLpCap];
  uint32_t top_key[kLpMaxTop];   // this CTA's best, in order
  int top_idx[kLpMaxTop];
  uint32_t tau;
  int hot[kLpThreads];
  int n_hot, n_cand, n_top;
  // what the parts of a row push to the first one's shared memory
  uint32_t all_key[kLpMaxSplit * kLpMaxTop];
  int all_idx[kLpMaxSplit * kLpMaxTop];
  Sums all_sums[kLpMaxSplit];
  int wsum[kLpWarps];
};

// Ranks the n candidates of s and leaves the best k in order (dst may be s's own top).
__device__ __forceinline__ void rank_candidates(const uint32_t* key, const int* idx, int n, int k, uint32_t* dk, int* di) {
  for (int c = threadIdx.x; c < n; c += kLpThreads) {
    const uint32_t kc = key[c];
    const int ic = idx[c];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += before(key[j], idx[j], kc, ic);
    if (r < k) {
      dk[r] = kc;
      di[r] = ic;
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(kLpThreads, 5) logprobs_kernel(const __grid_constant__ LpParams p, int split) {
  constexpr int E = Vec<DT>::E;
  constexpr int kBits = DT == SS_BF16 ? 16 : DT == SS_F16 ? 19 : 32;  // of the fp32 key that tell two values apart
  constexpr uint32_t kMask = 0xffffffffu << (32 - kBits);
  __shared__ LpShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  constexpr int ES = DT == SS_F32 ? 4 : 2;
  const char* base = reinterpret_cast<const char*>(p.x) + row * p.row_stride * ES;
  // elements before the first 32-byte boundary, then whole loads, then the rest
  int head = (int)((kLpVec - (reinterpret_cast<uintptr_t>(base) & (kLpVec - 1))) & (kLpVec - 1)) / ES;
  head = min(head, p.vocab);
  const int vecs = (p.vocab - head) / E, tail0 = head + vecs * E;
  const int per = (vecs + split - 1) / split, v0 = min(vecs, part * per), v1 = min(vecs, v0 + per);
  const char* body = base + head * ES;
  if (tid == 0) s.n_hot = s.n_cand = 0;
  // the first part's shared memory is there once every CTA of the cluster has started
  if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ---- sums ----
  float m = -INFINITY, l[2] = {0.f, 0.f}, a[2] = {0.f, 0.f};
  auto raise = [&](float lm) {  // m must cover lm
    if (lm > m) {
      const float d = fmaxf(m - lm, kFar), e = lp_ex2(d * kLog2e);
      a[0] = e * fmaf(d, l[0], a[0]);
      a[1] = e * fmaf(d, l[1], a[1]);
      l[0] *= e;
      l[1] *= e;
    }
    m = max_nan(m, lm);
  };
  Words buf;
  if (v0 + tid < v1) buf = load32(body + (int64_t)(v0 + tid) * kLpVec);
  for (int v = v0 + tid; v < v1; v += kLpThreads) {
    float x[E];
    Vec<DT>::get(buf, x);
    if (v + kLpThreads < v1) buf = load32(body + (int64_t)(v + kLpThreads) * kLpVec);
    float lm = x[0];
#pragma unroll
    for (int i = 0; i < E; i += 2) lm = max3_nan(lm, x[i], x[i + 1]);
    raise(lm);
    add_up(x, m, l, a);
  }
  // the ragged ends belong to the first part: a thread takes at most one element of each
  const int n_ends = part == 0 ? head + p.vocab - tail0 : 0;
  const int end_at = tid < head ? tid : tail0 + tid - head;
  const float end_x = tid < n_ends ? load_as_f32(base, DT, end_at) : -INFINITY;
  if (tid < n_ends) {
    const float x[2] = {end_x, -INFINITY};
    raise(end_x);
    add_up(x, m, l, a);
  }
  s.tmax[tid] = m;
  Sums t{m, l[0] + l[1], a[0] + a[1]};
  float worst = m;  // NaN or +inf anywhere shows here
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums y{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.l, o), __shfl_xor_sync(0xffffffffu, t.a, o)};
    t = merge(t, y);
    worst = max_nan(worst, __shfl_xor_sync(0xffffffffu, worst, o));
  }
  if (lane == 0) s.warp[warp] = Sums{worst, t.l, t.a};
  __syncthreads();

  // ---- warp 0: the CTA's sums; the k-th largest of the threads' maxima ----
  const int k = p.top;
  if (warp == 0) {
    Sums y = lane < kLpWarps ? s.warp[lane] : Sums{-INFINITY, 0.f, 0.f};
    float w = y.m;
#pragma unroll
    for (int o = kLpWarps / 2; o > 0; o >>= 1) {
      const Sums z{__shfl_xor_sync(0xffffffffu, y.m, o), __shfl_xor_sync(0xffffffffu, y.l, o), __shfl_xor_sync(0xffffffffu, y.a, o)};
      w = max_nan(w, __shfl_xor_sync(0xffffffffu, w, o));
      y = merge(y, z);
    }
    if (lane == 0) s.sums = Sums{w, y.l, y.a};
    if (k > 0) {
      uint32_t key[kLpThreads / 32];
#pragma unroll
      for (int i = 0; i < kLpThreads / 32; ++i) key[i] = order_key(s.tmax[i * 32 + lane]);
      // bit by bit from the top; fp16 and bf16 values leave the low bits of fp32 alike
      uint32_t tau = 0;
      for (int b = 31; b >= 32 - kBits; --b) {
        const uint32_t trial = tau | 1u << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kLpThreads / 32; ++i) n += key[i] >= trial;
        if ((int)__reduce_add_sync(0xffffffffu, (unsigned)n) >= k) tau = trial;
      }
      if (lane == 0) s.tau = tau;
    }
  }
  __syncthreads();

  // ---- candidates: elements that reach tau ----
  if (k > 0) {
    const uint32_t tau = s.tau;
    auto offer = [&](float x, int i) {
      const uint32_t key = order_key(x);
      if (key >= tau) {
        const int c = atomicAdd(&s.n_cand, 1);  // the order of arrival does not matter: they are ranked
        if (c < kLpCap) {
          s.key[c] = key;
          s.idx[c] = i;
        }
      }
    };
    if (order_key(m) >= tau) s.hot[atomicAdd(&s.n_hot, 1)] = tid;
    __syncthreads();
    const int n_hot = s.n_hot, nv = (v1 - v0 + kLpThreads - 1) / kLpThreads;
    if (n_hot * nv <= 4096) {
      for (int w = tid; w < n_hot * nv; w += kLpThreads) {
        const int v = v0 + w / n_hot * kLpThreads + s.hot[w % n_hot];
        if (v < v1) {
          float x[E];
          Vec<DT>::get(load32(body + (int64_t)v * kLpVec), x);
#pragma unroll
          for (int i = 0; i < E; ++i) offer(x[i], head + v * E + i);
        }
      }
      if (tid < n_ends) offer(end_x, end_at);
    } else if (tid == 0) {
      s.n_cand = kLpCap + 1;  // many equal maxima
    }
    __syncthreads();
    bool listed = s.n_cand <= kLpCap;
    if (!listed) {
      // Many elements equal tau (a constant row, a mask): list those above it, which at most k - 1
      // threads hold, and take the first equal ones in the order of their indices.
      __syncthreads();
      if (tid == 0) s.n_hot = s.n_cand = 0;
      __syncthreads();
      auto above = [&](float x) { return (order_key(x) & kMask) > tau; };
      if (above(m)) s.hot[atomicAdd(&s.n_hot, 1)] = tid;
      __syncthreads();
      const int n_above = s.n_hot;
      auto list = [&](float x, int i) {
        if (above(x)) {
          const int c = atomicAdd(&s.n_cand, 1);
          if (c < kLpCap) {
            s.key[c] = order_key(x);
            s.idx[c] = i;
          }
        }
      };
      for (int w = tid; w < n_above * nv; w += kLpThreads) {
        const int v = v0 + w / n_above * kLpThreads + s.hot[w % n_above];
        if (v < v1) {
          float x[E];
          Vec<DT>::get(load32(body + (int64_t)v * kLpVec), x);
#pragma unroll
          for (int i = 0; i < E; ++i) list(x[i], head + v * E + i);
        }
      }
      if (tid < n_ends) list(end_x, end_at);
      __syncthreads();
      listed = s.n_cand + k <= kLpCap;
      int have = s.n_cand;
      // steps in the order of the indices: the row's head, the vectors, the row's tail
      for (int st = -1; listed && st <= nv && have < k; ++st) {
        float x[E];
        int at = 0, n = 0;  // this thread's elements of the step: at, at + 1, ...
        if (st < 0 || st == nv) {
          n = tid < n_ends && (tid < head) == (st < 0) ? 1 : 0;
          at = end_at;
          x[0] = end_x;
        } else if (v0 + st * kLpThreads + tid < v1) {
          const int v = v0 + st * kLpThreads + tid;
          Vec<DT>::get(load32(body + (int64_t)v * kLpVec), x);
          at = head + v * E;
          n = E;
        }
        int eq = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) eq |= (i < n && (order_key(x[i]) & kMask) == tau ? 1 : 0) << i;
        int inc = __popc(eq);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        if (lane == 31) s.wsum[warp] = inc;
        __syncthreads();
        int at_rank = have + inc - __popc(eq), total = 0;
        for (int w = 0; w < kLpWarps; ++w) {
          if (w < warp) at_rank += s.wsum[w];
          total += s.wsum[w];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (eq >> i & 1) {
            if (at_rank < k) {
              s.key[at_rank] = order_key(x[i]);
              s.idx[at_rank] = at + i;
            }
            ++at_rank;
          }
        }
        have += total;
        __syncthreads();
      }
      if (listed && tid == 0) s.n_cand = max(s.n_cand, min(have, k));
      __syncthreads();
    }
    if (listed) {
      if (tid == 0) s.n_top = min(k, s.n_cand);
      rank_candidates(s.key, s.idx, s.n_cand, k, s.top_key, s.top_idx);
    } else {
      // Many elements above tau too: one after the other, each the first in order after the one before.
      uint32_t pk = 0xffffffffu;
      int pi = -1, got = 0;
      for (int r = 0; r < k; ++r) {
        uint32_t bk = 0;
        int bi = 0x7fffffff;
        auto look = [&](float x, int i) {
          const uint32_t key = order_key(x);
          if (before(pk, pi, key, i) && (bi == 0x7fffffff || before(key, i, bk, bi))) { bk = key; bi = i; }
        };
        for (int v = v0 + tid; v < v1; v += kLpThreads) {
          float x[E];
          Vec<DT>::get(load32(body + (int64_t)v * kLpVec), x);
#pragma unroll
          for (int i = 0; i < E; ++i) look(x[i], head + v * E + i);
        }
        if (tid < n_ends) look(end_x, end_at);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint32_t k2 = __shfl_xor_sync(0xffffffffu, bk, o);
          const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
          if (i2 != 0x7fffffff && (bi == 0x7fffffff || before(k2, i2, bk, bi))) { bk = k2; bi = i2; }
        }
        __syncthreads();
        if (lane == 0) { s.key[warp] = bk; s.idx[warp] = bi; }
        __syncthreads();
        bk = 0; bi = 0x7fffffff;
        for (int w = 0; w < kLpWarps; ++w)
          if (s.idx[w] != 0x7fffffff && (bi == 0x7fffffff || before(s.key[w], s.idx[w], bk, bi))) { bk = s.key[w]; bi = s.idx[w]; }
        if (bi == 0x7fffffff) break;
        pk = bk;
        pi = bi;
        if (tid == 0) { s.top_key[got] = bk; s.top_idx[got] = bi; }
        ++got;
      }
      __syncthreads();
      if (tid == 0) s.n_top = got;
    }
  } else if (tid == 0) {
    s.n_top = 0;
  }
  __syncthreads();

  // ---- join the parts of a row ----
  Sums sum = s.sums;
  int n_top = s.n_top;
  const uint32_t* tk = s.top_key;
  const int* ti = s.top_idx;
  if (split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    LpShared* first = cluster.map_shared_rank(&s, 0);
    if (tid < k) {  // past this part's elements: what ranks behind everything
      first->all_key[part * k + tid] = tid < n_top ? s.top_key[tid] : 0u;
      first->all_idx[part * k + tid] = tid < n_top ? s.top_idx[tid] : 0x7fffffff - part * kLpMaxTop - tid;
    }
    if (tid == 0) first->all_sums[part] = sum;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (part != 0) return;
    float worst_m = -INFINITY;
    sum = s.all_sums[0];
    for (int c = 0; c < split; ++c) {
      worst_m = max_nan(worst_m, s.all_sums[c].m);
      if (c > 0) sum = merge(sum, s.all_sums[c]);
    }
    sum.m = worst_m;
    rank_candidates(s.all_key, s.all_idx, split * k, k, s.key, s.idx);
    __syncthreads();
    tk = s.key;
    ti = s.idx;
    n_top = min(k, p.vocab);
  }

  const bool bad = !(sum.m < INFINITY), none = sum.m == -INFINITY;
  const float nan = __int_as_float(0x7fffffff);
  const float ll = logf(sum.l);
  auto lp = [&](float x) { return bad ? nan : none ? -INFINITY : (x - sum.m) - ll; };
  if (tid < k) {
    const bool has = tid < n_top;
    const uint32_t u = has ? tk[tid] : 0u;
    const float x = __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
    p.top_ids[row * k + tid] = bad || !has ? -1 : ti[tid];
    p.top_lp[row * k + tid] = bad ? nan : has ? lp(x) : -INFINITY;
  }
  if (tid == kLpThreads - 1) {
    const int64_t tg = p.targets ? p.targets[row] : -1;
    p.logprobs[row] = tg < 0 ? 0.f : tg >= p.vocab ? nan : lp(load_as_f32(base, DT, tg));
    p.entropy[row] = bad ? nan : none ? 0.f : ll - sum.a / sum.l;
  }
}

// CTAs for a row: the split whose waves of CTAs (five an SM) take least, at about 9 GB/s a CTA
// and 3 us for what a CTA does after its pass.
int lp_split(int64_t rows, int64_t row_bytes) {
  const int64_t slots = 5LL * sm_count();
  int best = 1;
  double least = 0;
  for (int s = 1; s <= kLpMaxSplit; s *= 2) {
    const double waves = (double)((rows * s + slots - 1) / slots);
    const double t = waves * ((double)row_bytes / s / 9e3 + 3.0);
    if (s == 1 || t < least) { least = t; best = s; }
  }
  return best;
}

template <int DT>
int launch_logprobs(const LpParams& p, int split, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * split));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = split > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<DT>, p, split);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(SS_ERR_CUDA, std::string("ss_token_logprobs: ") + cudaGetErrorString(e));
  }
  return check_launch("ss_token_logprobs");
}

}  // namespace
}  // namespace ss

using namespace ss;

extern "C" int ss_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t row_stride,
                                 int vocab, const int64_t* targets, int top, float* logprobs,
                                 float* entropy, int32_t* top_ids, float* top_logprobs, void* stream) {
  return c_entry([&]() -> int {
    if (rows == 0) return SS_OK;
    SS_REQUIRE(logits && logprobs && entropy && rows > 0, "ss_token_logprobs: null pointer or negative count");
    SS_REQUIRE(dtype >= SS_F32 && dtype <= SS_BF16, "ss_token_logprobs: bad dtype");
    SS_REQUIRE(vocab >= 1, "ss_token_logprobs: empty vocabulary");
    SS_REQUIRE(top >= 0 && top <= kLpMaxTop, "ss_token_logprobs: top must be in [0, 32]");
    SS_REQUIRE(top == 0 || (top_ids && top_logprobs), "ss_token_logprobs: null pointer");
    SS_REQUIRE(rows <= 0x7fffffff / kLpMaxSplit, "ss_token_logprobs: too many rows");
    count_dispatch("ss_token_logprobs");
    LpParams p{logits, rows, row_stride, vocab, targets, top, logprobs, entropy, top_logprobs, top_ids};
    cudaStream_t st = as_stream(stream);
    const int split = lp_split(rows, (int64_t)vocab * (dtype == SS_F32 ? 4 : 2));
    if (dtype == SS_F32) return launch_logprobs<SS_F32>(p, split, st);
    if (dtype == SS_F16) return launch_logprobs<SS_F16>(p, split, st);
    return launch_logprobs<SS_BF16>(p, split, st);
  });
}
