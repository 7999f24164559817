// c4s_kv.cuh -- the paged key-value cache of the decoder's attention: new
// tokens' keys and values written into it (as they are, or quantized as they
// are written) and read back densely.
//
// Quantization, per group of 32 or 64 consecutive elements of a (token, head)
// row (the affine scheme of c4s_quantize_affine, decided exactly):
//     scale = (max - min) / n,  bias = min,  n = 2^bits - 1,
//     code  = the integer nearest to n (x - min) / (max - min), ties to even,
//     value = scale code + bias  (one fp32 FMA).
// The quotient is formed in fp32, with a relative error below 2^-21.3 (two
// differences' roundings of 2^-24, the approximate factor's two units in the
// last place): for a quotient of up to n = 255 that is below 2^-13, for 15
// below 2^-17. Where it falls that near to a tie the decision is repeated in
// fp64, in which the differences and the products are exact for 16-bit inputs
// whose exponents lie within 40 of each other (a bf16 element further below the
// group's largest counts as zero where it alone would decide a tie).
// A group with a non-finite element reads back as NaN throughout; a constant
// group has scale 0 and reads back exactly.
//
// One thread works 8 consecutive elements (16 B of the source) of a key row
// and the same 8 of the value row: a group is 4 or 8 neighbouring lanes of one
// warp, and its minimum and maximum take two or three shuffles. A CTA works a
// few whole tokens; where each lies is found once, by one thread per token.
// Both kernels are bound by HBM (the source's bytes once, the cache's once)
// and close to it by instructions: integer codes are made and taken apart
// with the float format's own bits, without conversions.
#pragma once

namespace c4s {

constexpr int KV_NT = 256;
// Units of 8 elements that a CTA works (at least one token, at most KV_TOKS;
// fewer where CTAs would be few). What a CTA pays to find its tokens is spread
// over them: 131072 tokens of 8 x 128 to 8-bit codes and back take 568 us with
// 512, 530 with 1024, 520 with 2048, 522 with 4096. Rows kept in 16 bits are
// bound by HBM and want their CTAs to end evenly: 64 ragged prompts of up to
// 1500 tokens of 20 x 64 and back take 182 us with 1024, 187 with 2048.
constexpr int KV_UNITS = 2048, KV_UNITS16 = 1024;
constexpr int KV_TOKS = 64;

struct KvCache {
  unsigned char* k;
  unsigned char* v;
  unsigned char* k_sb;
  unsigned char* v_sb;
  long long page_stride, head_stride, token_stride;          // bytes
  long long sb_page_stride, sb_head_stride, sb_token_stride;  // bytes
  int num_pages, page_size, heads, dim, group;
};

struct KvArgs {
  KvCache c;
  const int* table;                   // [B, max_pages], rows table_ld apart
  long long table_ld;
  int max_pages, B;
  const void* k;                      // dense side: [T, heads, dim] by its strides (elements)
  const void* v;
  long long tstride, hstride;
  bool vec;                           // its rows are 16-byte aligned
  long long T;
  int units, per_cta;                              // per token; tokens per CTA
  PageDiv udiv, cdiv;                              // by the units of a token, of a head
  const long long* off;               // [B + 1] or null: token t is sequence t's
  const int* pos;                     // [B] position of a sequence's first token (< 0: skip it)
  unsigned* errflags;
};

template <typename T> struct Cvt;
template <> struct Cvt<__nv_bfloat16> {
  static __device__ __forceinline__ float f(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 t(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Cvt<__half> {
  static __device__ __forceinline__ float f(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half t(float x) { return __float2half_rn(x); }
};
template <> struct Cvt<float> {
  static __device__ __forceinline__ float f(float x) { return x; }
  static __device__ __forceinline__ float t(float x) { return x; }
};

// 8 consecutive elements; `vec`: 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, T (&x)[8]) {
  if (vec) {
    constexpr int N = (int)(8 * sizeof(T) / 16);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      memcpy(&x[i * 16 / sizeof(T)], &w, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const T (&x)[8]) {
  if (vec) {
    constexpr int N = (int)(8 * sizeof(T) / 16);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint4 w;
      memcpy(&w, &x[i * 16 / sizeof(T)], 16);
      __stcs(reinterpret_cast<uint4*>(p) + i, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
}

// x / n, n = 2^BITS - 1, correctly rounded for normal quotients: the product with 1 / n and one
// correction by its exact remainder.
template <int BITS> __device__ __forceinline__ float div_n(float x) {
  constexpr float n = (float)((1 << BITS) - 1), r = 1.0f / n;
  const float q = x * r;
  return fmaf(fmaf(-n, q, x), r, q);
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float c;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// Codes of 8 elements whose group has the extremes lo and hi, one a word. The
// sum with 1.5 2^23 rounds to an integer (ties to even) and has it in its low
// bits. Where the estimate is near the border h between two codes, the sign of
// n (x - lo) - h (hi - lo) decides, exactly. 16-bit values on a common grid
// make true ties (3 % of normally distributed ones), so this is no rare case:
// with a division in fp64 there, writing 64000 tokens of 20 heads of 64 took
// 285 us, with products 212; in fp32 with the roundings' errors carried 233.
template <int BITS>
__device__ __forceinline__ void kv_codes(const float (&x)[8], float lo, float hi, unsigned (&q)[8]) {
  constexpr float n = (float)((1 << BITS) - 1), R = 12582912.0f;
  constexpr float NEAR = 0.5f - (BITS == 8 ? 0x1p-13f : 0x1p-17f);
  const float inv = __fdividef(n, hi - lo);
  if (inv > 1e-30f && inv < 1e30f) {
    float e[8], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = x[i] - lo, v = fmaf(d, inv, R);
      q[i] = __float_as_uint(v);                   // the code in the low byte (the bits above are dropped)
      e[i] = fmaf(d, inv, R - v);
      far = fmaxf(far, fabsf(e[i]));
    }
    if (far > NEAR) {
      const double span = (double)hi - lo;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(e[i]) > NEAR) {
          const float low = __uint_as_float(q[i]) - R + (e[i] > 0.0f ? 0.0f : -1.0f);    // the lower of the two codes
          const double s = fma(-((double)low + 0.5), span, ((double)x[i] - lo) * (double)n);
          const unsigned c = (unsigned)low;
          q[i] = s > 0.0 ? c + 1 : s < 0.0 ? c : c + (c & 1);
        }
    }
  } else {
    // a constant group, a range past fp32's or near its smallest numbers, or no number at all
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double r = hi > lo ? rint(((double)x[i] - lo) * (double)n / ((double)hi - lo)) : 0.0;
      q[i] = (unsigned)fminf(fmaxf((float)r, 0.0f), n);
    }
  }
}

// Where a CTA's tokens lie: offsets of a token's slot, of its scales (head 0);
// found by one thread per token.
struct KvPlace {
  long long row, sb;
  int state;                                       // 0: nothing to do, 1: a place, 2: no page
};
__device__ __forceinline__ void kv_places(const KvArgs& a, KvPlace* pl) {
  const int i = threadIdx.x;
  if (i < a.per_cta) {
    const long long tok = (long long)blockIdx.x * a.per_cta + i;
    KvPlace p{0, 0, 0};
    int b = 0;
    if (tok < a.T && (a.off == nullptr || token_sequence(a.off, a.B, tok, b))) {
      if (a.off == nullptr) b = (int)tok;
      const int p0 = a.pos[b];
      int page, slot;
      if (p0 >= 0) {
        p.state = 2;
        if (kv_locate(a.table + (long long)b * a.table_ld, a.max_pages, a.c.num_pages, a.c.page_size,
                      p0 + (a.off ? tok - a.off[b] : 0), page, slot)) {
          p.state = 1;
          p.row = (long long)page * a.c.page_stride + (long long)slot * a.c.token_stride;
          p.sb = (long long)page * a.c.sb_page_stride + (long long)slot * a.c.sb_token_stride;
        } else {
          atomicOr(a.errflags, C4S_DEVERR_KV_PAGE);
        }
      }
    }
    pl[i] = p;
  }
  __syncthreads();
}

__device__ __forceinline__ long long kv_row(const KvCache& c, int page, int head, int slot) {
  return (long long)page * c.page_stride + (long long)head * c.head_stride + (long long)slot * c.token_stride;
}
__device__ __forceinline__ long long kv_sb(const KvCache& c, int page, int head, int slot) {
  return (long long)page * c.sb_page_stride + (long long)head * c.sb_head_stride + (long long)slot * c.sb_token_stride;
}

// One row's 8 elements into the cache. Every lane of the warp takes part in
// the shuffles; `live` lanes store.
template <typename T, int BITS>
__device__ __forceinline__ void kv_put(const T (&x)[8], unsigned char* row, unsigned char* sb, int chunk, int glanes,
                                       bool live) {
  if constexpr (BITS == 16) {
    if (live) store8(reinterpret_cast<T*>(row) + 8 * chunk, true, x);
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Cvt<T>::f(x[i]);
    // a NaN in the group becomes both
    float lo = min_nan(min_nan(min_nan(f[0], f[1]), min_nan(f[2], f[3])), min_nan(min_nan(f[4], f[5]), min_nan(f[6], f[7])));
    float hi = max_nan(max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3])), max_nan(max_nan(f[4], f[5]), max_nan(f[6], f[7])));
    for (int o = 1; o < glanes; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(FULL, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(FULL, hi, o));
    }
    unsigned q[8];
    kv_codes<BITS>(f, lo, hi, q);
    if (!live) return;
    if ((chunk & (glanes - 1)) == 0) {
      const float d = hi - lo, nan = __int_as_float(0x7fc00000);
      const float scale = d < INFINITY ? div_n<BITS>(d) : div_n<BITS>(hi) - div_n<BITS>(lo);
      const bool fine = hi < INFINITY && lo > -INFINITY;
      *reinterpret_cast<float2*>(sb + 8 * (chunk / glanes)) = fine ? make_float2(scale, lo) : make_float2(nan, nan);
    }
    if constexpr (BITS == 8) {
      uint2 w;
      w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
      w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
      *reinterpret_cast<uint2*>(row + 8 * chunk) = w;
    } else {
      unsigned w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= (q[i] & 15u) << (4 * i);
      *reinterpret_cast<unsigned*>(row + 4 * chunk) = w;
    }
  }
}

template <typename T, int BITS>
__global__ void __launch_bounds__(KV_NT) kv_write_kernel(KvArgs a) {
  __shared__ KvPlace pl[KV_TOKS];
  grid_dep_wait();                                 // the projection that made the new rows
  grid_dep_launch();
  kv_places(a, pl);
  const int glanes = a.c.group >> 3, total = a.per_cta * a.units;
  for (int u0 = 0; u0 < total; u0 += KV_NT) {
    const int u = u0 + threadIdx.x;
    const int tk = min(page_of(a.udiv, u), a.per_cta - 1);
    const int r = u - tk * a.units, head = page_of(a.cdiv, r), chunk = r - head * (a.c.dim >> 3);
    const bool live = u < total && pl[tk].state == 1;
    T xk[8], xv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) xk[i] = xv[i] = Cvt<T>::t(0.0f);
    if (live) {
      const long long s = ((long long)blockIdx.x * a.per_cta + tk) * a.tstride + (long long)head * a.hstride + 8 * chunk;
      load8(static_cast<const T*>(a.k) + s, a.vec, xk);
      load8(static_cast<const T*>(a.v) + s, a.vec, xv);
    }
    const long long row = live ? pl[tk].row + (long long)head * a.c.head_stride : 0;
    const long long sb = BITS != 16 && live ? pl[tk].sb + (long long)head * a.c.sb_head_stride : 0;
    kv_put<T, BITS>(xk, a.c.k + row, a.c.k_sb + sb, chunk, glanes, live);
    kv_put<T, BITS>(xv, a.c.v + row, a.c.v_sb + sb, chunk, glanes, live);
  }
}

// 8 elements of a row's values. TC: type of 16-bit cache rows (unused for
// codes); TO: type of the output. A code's byte becomes the float 2^23 + code.
template <typename TC, typename TO, int BITS>
__device__ __forceinline__ void kv_get(const unsigned char* row, const unsigned char* sb, int chunk, int glanes,
                                       TO (&y)[8]) {
  if constexpr (BITS == 16) {
    TC x[8];
    load8(reinterpret_cast<const TC*>(row) + 8 * chunk, true, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = Cvt<TO>::t(Cvt<TC>::f(x[i]));
  } else {
    const float2 p = *reinterpret_cast<const float2*>(sb + 8 * (chunk / glanes));
    uint2 w;
    if constexpr (BITS == 8) {
      w = __ldcs(reinterpret_cast<const uint2*>(row + 8 * chunk));
    } else {
      const unsigned v = __ldcs(reinterpret_cast<const unsigned*>(row + 4 * chunk));
      w = make_uint2(v & 0x0f0f0f0fu, (v >> 4) & 0x0f0f0f0fu);       // even, odd elements
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned word = BITS == 8 ? (i < 4 ? w.x : w.y) : (i & 1 ? w.y : w.x);
      const unsigned sel = 0x7440u + (BITS == 8 ? (i & 3) : (i >> 1));
      const float f = __uint_as_float(__byte_perm(word, 0x4b000000u, sel)) - 8388608.0f;
      y[i] = Cvt<TO>::t(fmaf(p.x, f, p.y));
    }
  }
}

template <typename TC, typename TO, int BITS>
__global__ void __launch_bounds__(KV_NT) kv_read_kernel(KvArgs a) {
  __shared__ KvPlace pl[KV_TOKS];
  grid_dep_wait();                                 // the writes of earlier kernels
  grid_dep_launch();
  kv_places(a, pl);
  const int total = a.per_cta * a.units;
  for (int u = threadIdx.x; u < total; u += KV_NT) {
    const int tk = page_of(a.udiv, u);
    const int r = u - tk * a.units, head = page_of(a.cdiv, r), chunk = r - head * (a.c.dim >> 3);
    const int state = pl[tk].state;
    if (state == 0) continue;
    TO yk[8], yv[8];
    if (state == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) yk[i] = yv[i] = Cvt<TO>::t(0.0f);
    } else {
      const long long row = pl[tk].row + (long long)head * a.c.head_stride;
      const long long sb = BITS != 16 ? pl[tk].sb + (long long)head * a.c.sb_head_stride : 0;
      kv_get<TC, TO, BITS>(a.c.k + row, a.c.k_sb + sb, chunk, a.c.group >> 3, yk);
      kv_get<TC, TO, BITS>(a.c.v + row, a.c.v_sb + sb, chunk, a.c.group >> 3, yv);
    }
    const long long s = ((long long)blockIdx.x * a.per_cta + tk) * a.tstride + (long long)head * a.hstride + 8 * chunk;
    store8(static_cast<TO*>(const_cast<void*>(a.k)) + s, a.vec, yk);
    store8(static_cast<TO*>(const_cast<void*>(a.v)) + s, a.vec, yv);
  }
}

}  // namespace c4s
