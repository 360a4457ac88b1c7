// Writing rows into 4-bit KV pages by slot, and reading them back.
//
// A group of 32 dims of one token and head is stored as
//   x' = clamp(x, +-2^15), lo = min x', hi = max x'
//   s = fp16((hi - lo) / 15), z = fp16(lo)
//   c = clamp(rint((x' - z) / s), 0, 15), 0 where s = 0;   value = c * s + z
// (fp32 arithmetic, IEEE division, ties to even). A NaN makes its group's s
// and z NaN, so readers see NaN for the group and nothing else.
// Bound by HBM: a row is read once and 5 bits per value are written.
#include "int4_pages.cuh"

namespace ss {
namespace {

struct RowsParams {
  const void *k, *v;   // append: inputs; fetch: unused
  void *ko, *vo;       // fetch: outputs (N, H, D) contiguous
  int dtype;
  int64_t k_st, k_sh, v_st, v_sh;  // token and head strides of the inputs (elements)
  const int64_t* slots;
  int64_t n;
  int h;
  uint32_t h_inv;      // 2^32 / h, rounded up
  uint8_t* pages;
  int64_t page_stride, head_stride;  // bytes
  int page_blocks;     // 16-token blocks of a page
  uint32_t page_inv;   // 2^32 / page_blocks, rounded up
  int64_t n_slots;
};

// x / d for d >= 2 with inv = ceil(2^32 / d); the quotient of the product is x / d or one more.
__device__ __forceinline__ uint32_t quick_div(uint32_t x, uint32_t d, uint32_t inv, uint32_t& rem) {
  if (d == 1) {
    rem = 0;
    return x;
  }
  uint32_t q = __umulhi(x, inv);
  int r = (int)(x - q * d);
  if (r < 0) { --q; r += (int)d; }
  rem = (uint32_t)r;
  return q;
}

// Block of a slot in the pool and the token's place in it; null if the slot is outside the pool.
template <int D>
__device__ __forceinline__ uint8_t* block_of(const RowsParams& p, int64_t slot, uint32_t head, int& tok) {
  if (slot < 0 || slot >= p.n_slots) return nullptr;
  tok = (int)slot & 15;
  uint32_t in_page;
  const uint32_t page = quick_div((uint32_t)(slot >> 4), p.page_blocks, p.page_inv, in_page);
  return p.pages + page * p.page_stride + head * p.head_stride + (int64_t)in_page * Int4Blk<D>::kBytes;
}

// 8 consecutive elements as fp32.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (DT == SS_F32) {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (VEC) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
    uint32_t u[4];
    if constexpr (VEC) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = DT == SS_F16 ? h2f(u[i] & 0xffff) : bf2f(u[i] & 0xffff);
      x[2 * i + 1] = DT == SS_F16 ? h2f(u[i] >> 16) : bf2f(u[i] >> 16);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
  if constexpr (DT == SS_F32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SS_F16) {
        u[i] = pack_h2(x[2 * i], x[2 * i + 1]);
      } else {
        __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        u[i] = *reinterpret_cast<uint32_t*>(&b);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// min / max of three that keep NaN.
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// (a, b) = (a, b) * s + (c, d), packed fp32
__device__ __forceinline__ void fma_f32x2(float& a, float& b, float s, float c, float d) {
  asm("{\n .reg .b64 t, u, v;\n mov.b64 t, {%0, %1};\n mov.b64 u, {%2, %2};\n mov.b64 v, {%3, %4};\n"
      " fma.rn.f32x2 t, t, u, v;\n mov.b64 {%0, %1}, t;\n}"
      : "+f"(a), "+f"(b)
      : "f"(s), "f"(c), "f"(d));
}
__device__ __forceinline__ float mul_sat(float a, float b) {
  float r;
  asm("mul.rn.sat.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The 4 lanes of a group hold 8 values each: this lane's code word and the group's (s, z).
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& sz) {
  float lo = min3_nan(x[0], x[1], x[2]), hi = max3_nan(x[0], x[1], x[2]);
  lo = min3_nan(min3_nan(lo, x[3], x[4]), min3_nan(x[5], x[6], x[7]), x[7]);
  hi = max3_nan(max3_nan(hi, x[3], x[4]), max3_nan(x[5], x[6], x[7]), x[7]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float l2 = __shfl_xor_sync(0xffffffffu, lo, o), h2 = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = min3_nan(lo, l2, l2);
    hi = max3_nan(hi, h2, h2);
  }
  const bool nan = lo != lo;
  // the ends saturate; values beyond them go to the end codes by themselves
  lo = fminf(fmaxf(lo, -kInt4Max), kInt4Max);
  hi = fminf(fmaxf(hi, -kInt4Max), kInt4Max);
  const uint16_t sh = nan ? 0x7fff : f2h(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const uint16_t zh = nan ? 0x7fff : f2h(lo);
  sz = sh | (uint32_t)zh << 16;
  const float s = h2f(sh), z = h2f(zh);
  uint32_t w = 0;
  if (s > 0.f) {  // false for NaN
    // (x - z) / s by a reciprocal, clamped as a share of 15: off by less than 1e-5, so the nearest
    // integer is the division's unless the quotient comes that near to a half; then it is divided.
    const float r = __frcp_rn(s) * (1.f / 15.f);
    const float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to integers, ties to even
    float c[8], off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float a = x[i], b = x[i + 1];
      add_f32x2(a, b, -z, -z);
      a = mul_sat(a, r);
      b = mul_sat(b, r);
      float t = a, u = b;
      fma_f32x2(t, u, 15.f, kMagic, kMagic);
      add_f32x2(t, u, -kMagic, -kMagic);
      c[i] = t;
      c[i + 1] = u;
      fma_f32x2(a, b, 15.f, -t, -u);
      off = fmaxf(off, fmaxf(fabsf(a), fabsf(b)));
    }
    if (off > 0.49998f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], z), s)), 0.f), 15.f);
    }
    // four codes make an integer below 2^16, exact in fp32 and in the low bits of 2^23 + it
    const float w0 = fmaf(fmaf(c[3], 16.f, c[2]), 256.f, fmaf(c[1], 16.f, c[0])) + 8388608.f;
    const float w1 = fmaf(fmaf(c[7], 16.f, c[6]), 256.f, fmaf(c[5], 16.f, c[4])) + 8388608.f;
    w = __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x5410);
  }
  return w;
}

template <int D, int DT, bool VEC>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ RowsParams p) {
  using B = Int4Blk<D>;
  constexpr int X = D / 8;  // words of a row
  const int x = threadIdx.x % X;
  const uint32_t rows = (uint32_t)p.n * p.h, per = 256 / X, step = gridDim.x * per;
  // whole rows are in or out for a group of 4 lanes: X is a multiple of 8
  for (uint32_t row0 = blockIdx.x * per; row0 < rows; row0 += step) {
    const uint32_t row = row0 + threadIdx.x / X;
    uint32_t hd;
    const uint32_t t = quick_div(row, p.h, p.h_inv, hd);
    int tok;
    uint8_t* blk = row < rows ? block_of<D>(p, p.slots[t], hd, tok) : nullptr;
    float a[8] = {}, b[8] = {};
    if (blk) {
      load8<DT, VEC>(p.k, t * p.k_st + hd * p.k_sh + x * 8, a);
      load8<DT, VEC>(p.v, t * p.v_st + hd * p.v_sh + x * 8, b);
    }
    uint32_t ksz, vsz;
    const uint32_t kw = quantise8(a, ksz), vw = quantise8(b, vsz);
    if (!blk) continue;
    *reinterpret_cast<uint32_t*>(blk + B::key_word(tok, x >> 2, x & 3)) = kw;
    *reinterpret_cast<uint32_t*>(blk + B::value_word(tok, x)) = vw;
    if ((x & 3) == 0) {
      *reinterpret_cast<uint32_t*>(blk + B::key_sz(tok, x >> 2)) = ksz;
      *reinterpret_cast<uint32_t*>(blk + B::value_sz(tok, x >> 2)) = vsz;
    }
  }
}

__device__ __forceinline__ void dequant8(uint32_t w, uint32_t sz, float (&x)[8]) {
  const float s = h2f(sz & 0xffff), z = h2f(sz >> 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w >> (4 * i)) & 15), s, z);
}

template <int D, int DT>
__global__ void __launch_bounds__(256) fetch_kernel(const __grid_constant__ RowsParams p) {
  using B = Int4Blk<D>;
  constexpr int X = D / 8;
  const int x = threadIdx.x % X;
  const uint32_t rows = (uint32_t)p.n * p.h, per = 256 / X, step = gridDim.x * per;
  for (uint32_t row = blockIdx.x * per + threadIdx.x / X; row < rows; row += step) {
    uint32_t hd;
    const uint32_t t = quick_div(row, p.h, p.h_inv, hd);
    int tok;
    const uint8_t* blk = block_of<D>(p, p.slots[t], hd, tok);
    float a[8] = {}, b[8] = {};
    if (blk) {
      dequant8(*reinterpret_cast<const uint32_t*>(blk + B::key_word(tok, x >> 2, x & 3)),
               *reinterpret_cast<const uint32_t*>(blk + B::key_sz(tok, x >> 2)), a);
      dequant8(*reinterpret_cast<const uint32_t*>(blk + B::value_word(tok, x)),
               *reinterpret_cast<const uint32_t*>(blk + B::value_sz(tok, x >> 2)), b);
    }
    const int64_t at = ((int64_t)row * X + x) * 8;
    store8<DT>(p.ko, at, a);
    store8<DT>(p.vo, at, b);
  }
}

int rows_grid(int64_t threads) {
  const int64_t want = (threads + 255) / 256, cap = 16LL * sm_count();
  return (int)(want < cap ? want : cap);
}

// Sizes that the two entry points share.
void set_sizes(RowsParams& p, int64_t n, int h, int64_t n_pages, int page_size) {
  auto inv = [](int d) { return d < 2 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); };
  p.n = n;
  p.h = h;
  p.h_inv = inv(h);
  p.page_blocks = page_size / kBlkTokens;
  p.page_inv = inv(p.page_blocks);
  p.n_slots = n_pages * page_size;
}

template <int D>
int launch_append(const RowsParams& p, bool vec, cudaStream_t st) {
  const int g = rows_grid(p.n * p.h * (D / 8));
#define SS_APPEND(DT)                                                     \
  if (vec) append_kernel<D, DT, true><<<g, 256, 0, st>>>(p);              \
  else append_kernel<D, DT, false><<<g, 256, 0, st>>>(p)
  if (p.dtype == SS_F32) { SS_APPEND(SS_F32); }
  else if (p.dtype == SS_F16) { SS_APPEND(SS_F16); }
  else { SS_APPEND(SS_BF16); }
#undef SS_APPEND
  return check_launch("ss_int4_append");
}

template <int D>
int launch_fetch(const RowsParams& p, cudaStream_t st) {
  const int g = rows_grid(p.n * p.h * (D / 8));
  if (p.dtype == SS_F32) fetch_kernel<D, SS_F32><<<g, 256, 0, st>>>(p);
  else if (p.dtype == SS_F16) fetch_kernel<D, SS_F16><<<g, 256, 0, st>>>(p);
  else fetch_kernel<D, SS_BF16><<<g, 256, 0, st>>>(p);
  return check_launch("ss_int4_fetch");
}

int check_pool(const void* pages, int64_t n_pages, int64_t page_stride, int64_t head_stride, int64_t n, int h,
               int page_size, int d) {
  SS_REQUIRE(pages, "int4 pages: null pointer");
  SS_REQUIRE(int4_head_dim_ok(d), "int4 pages: head_dim must be 64, 128 or 256");
  SS_REQUIRE(page_size >= 16 && page_size % 16 == 0, "int4 pages: page_size must be a multiple of 16");
  SS_REQUIRE(n_pages >= 1 && h >= 1, "int4 pages: empty pool");
  SS_REQUIRE(n <= 0x7fffffff / h && n_pages <= (int64_t)0x7fffffff / (page_size / kBlkTokens),
             "int4 pages: 2^31 rows or blocks or more");
  SS_REQUIRE(((reinterpret_cast<uintptr_t>(pages) | (uintptr_t)page_stride | (uintptr_t)head_stride) & 15) == 0,
             "int4 pages: the pool and its strides must be multiples of 16 bytes");
  return SS_OK;
}

}  // namespace
}  // namespace ss

using namespace ss;

extern "C" {

int ss_int4_append(const void* k, const void* v, int dtype, int64_t k_token_stride,
                   int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                   const int64_t* slots, int64_t n, int n_heads, int d, void* pages,
                   int64_t n_pages, int64_t page_stride, int64_t head_stride, int page_size,
                   void* stream) {
  return c_entry([&]() -> int {
    if (n == 0) return SS_OK;
    SS_REQUIRE(k && v && slots && n > 0, "ss_int4_append: null pointer or negative count");
    SS_REQUIRE(dtype >= SS_F32 && dtype <= SS_BF16, "ss_int4_append: bad dtype");
    if (int rc = check_pool(pages, n_pages, page_stride, head_stride, n, n_heads, page_size, d)) return rc;
    count_dispatch("ss_int4_append");
    RowsParams p{};
    p.k = k; p.v = v; p.dtype = dtype;
    p.k_st = k_token_stride; p.k_sh = k_head_stride; p.v_st = v_token_stride; p.v_sh = v_head_stride;
    p.slots = slots;
    p.pages = static_cast<uint8_t*>(pages);
    p.page_stride = page_stride; p.head_stride = head_stride;
    set_sizes(p, n, n_heads, n_pages, page_size);
    const int es = dtype == SS_F32 ? 4 : 2;
    const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                       (uintptr_t)((k_token_stride | k_head_stride | v_token_stride | v_head_stride) * es)) & 15) == 0;
    cudaStream_t st = as_stream(stream);
    return d == 64 ? launch_append<64>(p, vec, st) : d == 128 ? launch_append<128>(p, vec, st)
                                                              : launch_append<256>(p, vec, st);
  });
}

int ss_int4_fetch(const int64_t* slots, int64_t n, int n_heads, int d, const void* pages,
                  int64_t n_pages, int64_t page_stride, int64_t head_stride, int page_size,
                  void* k_out, void* v_out, int dtype, void* stream) {
  return c_entry([&]() -> int {
    if (n == 0) return SS_OK;
    SS_REQUIRE(k_out && v_out && slots && n > 0, "ss_int4_fetch: null pointer or negative count");
    SS_REQUIRE(dtype >= SS_F32 && dtype <= SS_BF16, "ss_int4_fetch: bad dtype");
    SS_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0,
               "ss_int4_fetch: outputs must be 16-byte aligned");
    if (int rc = check_pool(pages, n_pages, page_stride, head_stride, n, n_heads, page_size, d)) return rc;
    count_dispatch("ss_int4_fetch");
    RowsParams p{};
    p.ko = k_out; p.vo = v_out; p.dtype = dtype;
    p.slots = slots;
    p.pages = static_cast<uint8_t*>(const_cast<void*>(pages));
    p.page_stride = page_stride; p.head_stride = head_stride;
    set_sizes(p, n, n_heads, n_pages, page_size);
    cudaStream_t st = as_stream(stream);
    return d == 64 ? launch_fetch<64>(p, st) : d == 128 ? launch_fetch<128>(p, st) : launch_fetch<256>(p, st);
  });
}

}  // extern "C"
