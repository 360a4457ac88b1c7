// Attention of ragged requests over 4-bit KV pages.
//
// Query row i of a request with q query rows and len keys stands at position
// len - q + i. It sees keys t <= position (causal) and t > position - window
// (window > 0). z_t = scale * q . k_t, p_t = e^(z_t - max z), and
//   out = sum p_t v_t / sum p_t,   lse = max z + ln sum p_t;
// a row that sees no key gives out = 0, lse = -inf.
//
// One warp per (query token, query head), one key at a time, in fp32.
#include "int4_pages.cuh"

namespace ss {
namespace {

struct AttnParams {
  const void* q;
  int dtype;
  int64_t q_st, q_sh;
  int64_t n_tokens;
  int hq, hkv;
  const uint8_t* pages;
  int n_pages;
  int64_t page_stride, head_stride;
  int page;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t *seq_lens, *cu_q;
  int n;
  float scale;
  int causal, window;
  void* out;
  float* lse;
};

template <int D>
__global__ void __launch_bounds__(256) attn_rows_kernel(AttnParams p) {
  using B = Int4Blk<D>;
  constexpr int E = D / 32;  // dims of a lane: lane * E ..
  const int lane = threadIdx.x & 31;
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= p.n_tokens * p.hq) return;
  const int64_t t = row / p.hq;
  const int hq = (int)(row - t * p.hq), h = hq / (p.hq / p.hkv);
  float o[E] = {}, m = -INFINITY, l = 0.f;
  int lo = 0, hi = p.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  if (t >= p.cu_q[lo] && t < p.cu_q[lo + 1]) {
    const int len = min(max(p.seq_lens[lo], 0), p.width * p.page);
    const int pos = len - (p.cu_q[lo + 1] - p.cu_q[lo]) + (int)(t - p.cu_q[lo]);
    float q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = load_as_f32(p.q, p.dtype, t * p.q_st + hq * p.q_sh + lane * E + e) * p.scale;
    const int last = p.causal ? min(len - 1, pos) : len - 1;
    const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int x = lane * E / 8, g = lane * E / 32, n0 = lane * E % 8;
    for (int k = first; k <= last; ++k) {
      const int page = p.table[lo * p.table_stride + k / p.page];
      if (page < 0 || page >= p.n_pages) continue;
      const int in_page = k % p.page, tok = in_page & 15;
      const uint8_t* blk = p.pages + page * p.page_stride + h * p.head_stride + (int64_t)(in_page >> 4) * B::kBytes;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + B::key_word(tok, x >> 2, x & 3));
      const uint32_t ks = *reinterpret_cast<const uint32_t*>(blk + B::key_sz(tok, g));
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(blk + B::value_word(tok, x));
      const uint32_t vs = *reinterpret_cast<const uint32_t*>(blk + B::value_sz(tok, g));
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) z += q[e] * fmaf((float)((kw >> (4 * (n0 + e))) & 15), h2f(ks & 0xffff), h2f(ks >> 16));
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) z += __shfl_xor_sync(0xffffffffu, z, s);
      const float mn = fmaxf(m, z), a = m == mn ? 1.f : expf(m - mn), w = z == mn ? 1.f : expf(z - mn);
      m = mn;
      l = l * a + w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * fmaf((float)((vw >> (4 * (n0 + e))) & 15), h2f(vs & 0xffff), h2f(vs >> 16));
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) store_from_f32(p.out, p.dtype, row * D + lane * E + e, l == 0.f ? 0.f : o[e] / l);
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace ss

using namespace ss;

extern "C" int ss_int4_attention(const ss_int4_attn_args* a, void* stream) {
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
    SS_REQUIRE(((reinterpret_cast<uintptr_t>(a->pages) | (uintptr_t)a->page_stride | (uintptr_t)a->head_stride) & 15) == 0,
               "ss_int4_attention: the pool and its strides must be multiples of 16 bytes");
    SS_REQUIRE(a->window >= 0, "ss_int4_attention: window must not be negative");
    count_dispatch("ss_int4_attention");
    AttnParams p{};
    p.q = a->q; p.dtype = a->dtype; p.q_st = a->q_token_stride; p.q_sh = a->q_head_stride;
    p.n_tokens = a->n_tokens; p.hq = a->hq; p.hkv = a->hkv;
    p.pages = static_cast<const uint8_t*>(a->pages); p.n_pages = a->n_pages;
    p.page_stride = a->page_stride; p.head_stride = a->head_stride; p.page = a->page_size;
    p.table = a->block_table; p.table_stride = a->table_stride; p.width = a->width;
    p.seq_lens = a->seq_lens; p.cu_q = a->cu_q; p.n = a->n_requests;
    p.scale = a->scale; p.causal = a->causal; p.window = a->window;
    p.out = a->out; p.lse = a->lse;
    const int64_t warps = a->n_tokens * a->hq;
    const unsigned grid = (unsigned)((warps + 7) / 8);
    cudaStream_t st = as_stream(stream);
    if (a->d == 64) attn_rows_kernel<64><<<grid, 256, 0, st>>>(p);
    else if (a->d == 128) attn_rows_kernel<128><<<grid, 256, 0, st>>>(p);
    else attn_rows_kernel<256><<<grid, 256, 0, st>>>(p);
    return check_launch("ss_int4_attention");
  });
}
