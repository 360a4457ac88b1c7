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
// One CTA per row: one pass for the sums, then k passes that each take the
// next one in order.
#include "common.cuh"

namespace ss {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e30f;  // stands for -inf in differences: its exponential is 0, times it is 0

struct LpParams {
  const void* x;
  int64_t rows, row_stride;
  int vocab;
  const int64_t* targets;
  int top;
  float *logprobs, *entropy, *top_lp;
  int32_t* top_ids;
};

__device__ __forceinline__ bool before(float v, int i, float w, int j) {  // (v, i) ranks before (w, j)
  return v > w || (v == w && i < j);
}

template <int DT>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(LpParams p) {
  __shared__ float s_m[kLpWarps], s_l[kLpWarps], s_a[kLpWarps], s_v[kLpWarps];
  __shared__ int s_i[kLpWarps], s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const char* base = reinterpret_cast<const char*>(p.x) + row * p.row_stride * (DT == SS_F32 ? 4 : 2);
  if (tid == 0) s_bad = 0;
  float m = -INFINITY, l = 0.f, a = 0.f;
  bool bad = false;
  for (int i = tid; i < p.vocab; i += kLpThreads) {
    const float y = load_as_f32(base, DT, i);
    bad |= !(y < INFINITY);
    if (y > m) {
      const float d = fmaxf(m - y, kFar), e = exp2f(d * kLog2e);
      a = e * (a + d * l);
      l *= e;
      m = y;
    }
    const float d = fmaxf(y - m, kFar), e = exp2f(d * kLog2e);  // kFar too for -inf - -inf
    l += e;
    a += e * d;
  }
  if (bad) s_bad = 1;
  auto merge = [](float& m, float& l, float& a, float m2, float l2, float a2) {
    const float n = fmaxf(m, m2);
    const float d1 = fmaxf(m - n, kFar), d2 = fmaxf(m2 - n, kFar);
    const float e1 = exp2f(d1 * kLog2e), e2 = exp2f(d2 * kLog2e);
    a = e1 * (a + d1 * l) + e2 * (a2 + d2 * l2);
    l = e1 * l + e2 * l2;
    m = n;
  };
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o),
                a2 = __shfl_xor_sync(0xffffffffu, a, o);
    merge(m, l, a, m2, l2, a2);
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; s_a[warp] = a; }
  __syncthreads();
  m = s_m[0]; l = s_l[0]; a = s_a[0];
  for (int w = 1; w < kLpWarps; ++w) merge(m, l, a, s_m[w], s_l[w], s_a[w]);
  bad = s_bad;
  const float nan = __int_as_float(0x7fffffff);
  const float ll = logf(l);
  auto lp = [&](float x) { return bad ? nan : l > 0.f ? (x - m) - ll : -INFINITY; };
  if (tid == 0) {
    const int64_t t = p.targets ? p.targets[row] : -1;
    p.logprobs[row] = t < 0 ? 0.f : t >= p.vocab ? nan : lp(load_as_f32(base, DT, t));
    p.entropy[row] = bad ? nan : l > 0.f ? ll - a / l : 0.f;
  }
  float pv = INFINITY;
  int pi = -1;
  for (int k = 0; k < p.top; ++k) {
    float v = -INFINITY;
    int at = 0x7fffffff;
    if (!bad) {
      for (int i = tid; i < p.vocab; i += kLpThreads) {
        const float x = load_as_f32(base, DT, i);
        if (before(pv, pi, x, i) && before(x, i, v, at)) { v = x; at = i; }
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const float v2 = __shfl_xor_sync(0xffffffffu, v, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (before(v2, i2, v, at)) { v = v2; at = i2; }
    }
    __syncthreads();
    if (lane == 0) { s_v[warp] = v; s_i[warp] = at; }
    __syncthreads();
    v = s_v[0]; at = s_i[0];
    for (int w = 1; w < kLpWarps; ++w)
      if (before(s_v[w], s_i[w], v, at)) { v = s_v[w]; at = s_i[w]; }
    pv = v;
    pi = at;
    if (tid == 0) {
      const bool none = at == 0x7fffffff;
      p.top_ids[row * p.top + k] = none ? -1 : at;
      p.top_lp[row * p.top + k] = bad ? nan : none ? -INFINITY : lp(v);
    }
  }
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
    SS_REQUIRE(rows <= 0x7fffffff, "ss_token_logprobs: too many rows");
    count_dispatch("ss_token_logprobs");
    LpParams p{logits, rows, row_stride, vocab, targets, top, logprobs, entropy, top_logprobs, top_ids};
    cudaStream_t st = as_stream(stream);
    if (dtype == SS_F32) logprobs_kernel<SS_F32><<<(unsigned)rows, kLpThreads, 0, st>>>(p);
    else if (dtype == SS_F16) logprobs_kernel<SS_F16><<<(unsigned)rows, kLpThreads, 0, st>>>(p);
    else logprobs_kernel<SS_BF16><<<(unsigned)rows, kLpThreads, 0, st>>>(p);
    return check_launch("ss_token_logprobs");
  });
}
