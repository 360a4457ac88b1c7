// Writing rows into 4-bit KV pages by slot, and reading them back.
//
// A group of 32 dims of one token and head is stored as
//   x' = clamp(x, +-2^15), lo = min x', hi = max x'
//   s = fp16((hi - lo) / 15), z = fp16(lo)
//   c = clamp(rint((x' - z) / s), 0, 15), 0 where s = 0;   value = c * s + z
// (fp32 arithmetic, IEEE division, ties to even). A NaN makes its group's s
// and z NaN, so readers see NaN for the group and nothing else.
//
// A row is read once and 5 bits per value are written: HBM is the floor, but
// quantising costs about 10 instructions a value, so a write of 16-bit rows is
// bound by issue (74 % of the slots): two lanes a group, 16 keys and 16 values
// a thread, so that what a row costs once (slot, page, addresses) is shared by
// 32 values. 49999 tokens x 8 heads x 128, every 7th of them padding, calls on end:
// write 68 us from fp16 (3.4 TB/s), 77 from bf16, 81 from fp32 (5.0 TB/s); with 8 + 8
// values a thread it was 96 us from fp16. Read back 51 us to fp16 (5.1 TB/s); 121 us
// to fp32 (3.8 TB/s).
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

// 16 consecutive elements as they are stored.
template <int DT>
struct Raw {
  static constexpr int N = DT == SS_F32 ? 16 : 8;
  uint32_t u[N];

  template <bool VEC>
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    if constexpr (VEC) {
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(base) + at * (DT == SS_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const uint4 a = __ldcs(p + i);
        u[4 * i] = a.x; u[4 * i + 1] = a.y; u[4 * i + 2] = a.z; u[4 * i + 3] = a.w;
      }
    } else if constexpr (DT == SS_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = reinterpret_cast<const uint32_t*>(base)[at + i];
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    }
  }
  __device__ __forceinline__ void get(float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (DT == SS_F32) {
        x[i] = __uint_as_float(u[i]);
      } else if constexpr (DT == SS_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
};

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
__device__ __forceinline__ float mul_sat(float a, float b) {
  float r;
  asm("mul.rn.sat.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The two lanes of a group hold 16 values each: this lane's two code words and the group's (s, z).
__device__ __forceinline__ void quantise16(const float (&x)[16], uint32_t (&w)[2], uint32_t& sz) {
  float lo = x[0], hi = x[0], lo2 = x[1], hi2 = x[1];
#pragma unroll
  for (int i = 2; i < 14; i += 4) {
    lo = min3_nan(lo, x[i], x[i + 1]);
    hi = max3_nan(hi, x[i], x[i + 1]);
    lo2 = min3_nan(lo2, x[i + 2], x[i + 3]);
    hi2 = max3_nan(hi2, x[i + 2], x[i + 3]);
  }
  lo = min3_nan(min3_nan(lo, x[14], x[15]), lo2, lo2);
  hi = max3_nan(max3_nan(hi, x[14], x[15]), hi2, hi2);
  const float lo3 = __shfl_xor_sync(0xffffffffu, lo, 1), hi3 = __shfl_xor_sync(0xffffffffu, hi, 1);
  lo = min3_nan(lo, lo3, lo3);
  hi = max3_nan(hi, hi3, hi3);
  const bool nan = lo != lo;
  // The ends saturate. Values below go to code 0 by themselves (z = -2^15 then); values above do not
  // always go to the code of 2^15, where z or s is rounded up: such a group is divided, see below.
  const bool above = hi > kInt4Max;
  lo = fminf(fmaxf(lo, -kInt4Max), kInt4Max);
  hi = fminf(fmaxf(hi, -kInt4Max), kInt4Max);
  const uint16_t sh = nan ? 0x7fff : f2h(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const uint16_t zh = nan ? 0x7fff : f2h(lo);
  sz = sh | (uint32_t)zh << 16;
  const float s = h2f(sh), z = h2f(zh);
  w[0] = w[1] = 0u;
  if (s > 0.f) {  // false for NaN
    // (x - z) / s by a reciprocal, clamped as a share of 15: off by less than 1e-5, so the nearest
    // integer is the division's unless the quotient comes that near to a half; then it is divided.
    const float r = __frcp_rn(s) * (1.f / 15.f);
    const float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to integers, ties to even
    float c[16], off = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float q = mul_sat(x[i] - z, r);
      c[i] = fmaf(q, 15.f, kMagic) - kMagic;
      off = fmaxf(off, fabsf(fmaf(q, 15.f, -c[i])));
    }
    if (off > 0.49998f || above) {
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(fminf(x[i], kInt4Max), z), s)), 0.f), 15.f);
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {  // four codes make an integer below 2^16, exact in the low bits of 2^23 + it
      const float* e = c + 8 * v;
      const float w0 = fmaf(fmaf(e[3], 16.f, e[2]), 256.f, fmaf(e[1], 16.f, e[0])) + 8388608.f;
      const float w1 = fmaf(fmaf(e[7], 16.f, e[6]), 256.f, fmaf(e[5], 16.f, e[4])) + 8388608.f;
      w[v] = __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x5410);
    }
  }
}

template <int D, int DT, bool VEC>
__global__ void __launch_bounds__(256, 4) append_kernel(const __grid_constant__ RowsParams p) {
  using B = Int4Blk<D>;
  constexpr int X = D / 16;  // threads of a row: 16 dims of its key and of its value each
  const int y = threadIdx.x % X;
  const uint32_t rows = (uint32_t)p.n * p.h, per = 256 / X, step = gridDim.x * per;
  // whole rows are in or out for the two lanes of a group
  for (uint32_t row0 = blockIdx.x * per; row0 < rows; row0 += step) {
    const uint32_t row = row0 + threadIdx.x / X;
    uint32_t hd;
    const uint32_t t = quick_div(row, p.h, p.h_inv, hd);
    int tok;
    uint8_t* blk = row < rows ? block_of<D>(p, __ldg(p.slots + t), hd, tok) : nullptr;
    Raw<DT> k{}, v{};
    if (blk) {
      k.template load<VEC>(p.k, t * p.k_st + hd * p.k_sh + y * 16);
      v.template load<VEC>(p.v, t * p.v_st + hd * p.v_sh + y * 16);
    }
    uint32_t w[2], ksz, vsz;
    float x[16];
    k.get(x);
    quantise16(x, w, ksz);
    if (blk) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<uint32_t*>(blk + B::key_word(tok, y >> 1, 2 * (y & 1) + e)) = w[e];
    }
    v.get(x);
    quantise16(x, w, vsz);
    if (blk) {
      if constexpr (B::W > 1) {  // two words of one piece
        *reinterpret_cast<uint2*>(blk + B::value_word(tok, 2 * y)) = make_uint2(w[0], w[1]);
      } else {
        *reinterpret_cast<uint32_t*>(blk + B::value_word(tok, 2 * y)) = w[0];
        *reinterpret_cast<uint32_t*>(blk + B::value_word(tok, 2 * y + 1)) = w[1];
      }
      if ((y & 1) == 0) {
        *reinterpret_cast<uint32_t*>(blk + B::key_sz(tok, y >> 1)) = ksz;
        *reinterpret_cast<uint32_t*>(blk + B::value_sz(tok, y >> 1)) = vsz;
      }
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
  const int g = rows_grid(p.n * p.h * (D / 16));
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
