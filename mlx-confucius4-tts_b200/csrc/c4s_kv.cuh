// c4s_kv.cuh -- the paged key-value cache of the decoder's attention: new
// tokens' keys and values written into it (as they are, or quantized as they
// are written) and read back densely.
//
// Quantization, per group of 32 or 64 consecutive elements of a (token, head)
// row (the affine scheme of c4s_quantize_affine, decided exactly):
//     scale = (max - min) / n,  bias = min,  n = 2^bits - 1,
//     code  = the integer nearest to n (x - min) / (max - min), ties to even,
//     value = scale code + bias  (one fp32 FMA).
// The quotient is formed in fp32, whose error here is below 2^-14 of a step
// (255 times three roundings of 2^-24 and an approximate product); where it
// falls within 2^-12 of a tie the decision is repeated in fp64, in which the
// differences and the product are exact for 16-bit inputs. A group with a
// non-finite element reads back as NaN throughout; a constant group has scale
// 0 and reads back exactly.
//
// One thread works 8 consecutive elements (16 B of the source) of a key row
// and the same 8 of the value row: a group is 4 or 8 neighbouring lanes of one
// warp, and its minimum and maximum take two or three shuffles. Both kernels
// are bound by HBM: bytes of the source once, of the cache once.
#pragma once

namespace c4s {

constexpr int KV_NT = 256;

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

// Codes of 8 elements whose group has the extremes lo and hi.
template <int BITS>
__device__ __forceinline__ void kv_codes(const float (&x)[8], float lo, float hi, unsigned (&q)[8]) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float inv = n / (hi - lo);
  const bool plain = inv > 0.0f && inv < 3.0e38f;   // neither a range past fp32's, nor one near its smallest
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = (x[i] - lo) * inv;
    float r = rintf(t);
    if (!plain || fabsf(t - r) > 0.5f - 0x1p-12f)
      r = hi > lo ? (float)rint(((double)x[i] - lo) * (double)n / ((double)hi - lo)) : 0.0f;
    q[i] = (unsigned)fminf(fmaxf(r, 0.0f), n);
  }
}

// Where unit u (8 elements of a head of a token) lies; false: nothing to do.
__device__ __forceinline__ bool kv_unit(const KvArgs& a, long long u, long long& tok, int& head, int& chunk, int& b,
                                        int& page, int& slot, bool& bad) {
  const int per_head = a.c.dim >> 3, per_tok = per_head * a.c.heads;
  tok = u / per_tok;
  const int r = (int)(u - tok * per_tok);
  head = r / per_head;
  chunk = r - head * per_head;
  bad = false;
  if (tok >= a.T) return false;
  long long j = 0;
  if (a.off) {
    if (!token_sequence(a.off, a.B, tok, b)) return false;
    j = tok - a.off[b];
  } else {
    b = (int)tok;
  }
  const int p0 = a.pos[b];
  if (p0 < 0) return false;
  bad = !kv_locate(a.table + (long long)b * a.table_ld, a.max_pages, a.c.num_pages, a.c.page_size, p0 + j, page, slot);
  return true;
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
    float f[8], lo = INFINITY, hi = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = Cvt<T>::f(x[i]);
      lo = fminf(lo, f[i]);
      hi = fmaxf(hi, f[i]);
      odd |= !(fabsf(f[i]) < INFINITY);
    }
    if (odd) hi = INFINITY;
    for (int o = 1; o < glanes; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(FULL, hi, o));
    }
    const bool fine = hi < INFINITY;
    unsigned q[8];
    kv_codes<BITS>(f, lo, hi, q);
    if (!live) return;
    constexpr float n = (float)((1 << BITS) - 1);
    if ((chunk & (glanes - 1)) == 0) {
      const float d = hi - lo;
      const float scale = d < INFINITY ? d / n : hi / n - lo / n;
      *reinterpret_cast<float2*>(sb + 8 * (chunk / glanes)) =
          fine ? make_float2(scale, lo) : make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    }
    if constexpr (BITS == 8) {
      uint2 w;
      w.x = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
      w.y = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
      *reinterpret_cast<uint2*>(row + 8 * chunk) = w;
    } else {
      unsigned w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= q[i] << (4 * i);
      *reinterpret_cast<unsigned*>(row + 4 * chunk) = w;
    }
  }
}

template <typename T, int BITS>
__global__ void __launch_bounds__(KV_NT) kv_write_kernel(KvArgs a) {
  grid_dep_wait();                                 // the projection that made the new rows
  grid_dep_launch();
  const long long u = (long long)blockIdx.x * KV_NT + threadIdx.x;
  long long tok;
  int head, chunk, b, page = 0, slot = 0;
  bool bad;
  const bool mine = kv_unit(a, u, tok, head, chunk, b, page, slot, bad);
  if (mine && bad && head == 0 && chunk == 0) atomicOr(a.errflags, C4S_DEVERR_KV_PAGE);
  const bool live = mine && !bad;
  T xk[8], xv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) xk[i] = xv[i] = Cvt<T>::t(0.0f);
  if (live) {
    const long long s = tok * a.tstride + (long long)head * a.hstride + 8 * chunk;
    load8(static_cast<const T*>(a.k) + s, a.vec, xk);
    load8(static_cast<const T*>(a.v) + s, a.vec, xv);
  }
  const long long row = live ? kv_row(a.c, page, head, slot) : 0;
  const long long sb = BITS != 16 && live ? kv_sb(a.c, page, head, slot) : 0;
  const int glanes = a.c.group >> 3;
  kv_put<T, BITS>(xk, a.c.k + row, a.c.k_sb + sb, chunk, glanes, live);
  kv_put<T, BITS>(xv, a.c.v + row, a.c.v_sb + sb, chunk, glanes, live);
}

// TC: type of 16-bit cache rows (unused for codes); TO: type of the output.
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
    if constexpr (BITS == 8) {
      const uint2 w = __ldcs(reinterpret_cast<const uint2*>(row + 8 * chunk));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i] = Cvt<TO>::t(fmaf(p.x, (float)(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu), p.y));
    } else {
      const unsigned w = __ldcs(reinterpret_cast<const unsigned*>(row + 4 * chunk));
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = Cvt<TO>::t(fmaf(p.x, (float)((w >> (4 * i)) & 0xfu), p.y));
    }
  }
}

template <typename TC, typename TO, int BITS>
__global__ void __launch_bounds__(KV_NT) kv_read_kernel(KvArgs a) {
  grid_dep_wait();                                 // the writes of earlier kernels
  grid_dep_launch();
  const long long u = (long long)blockIdx.x * KV_NT + threadIdx.x;
  long long tok;
  int head, chunk, b, page = 0, slot = 0;
  bool bad;
  if (!kv_unit(a, u, tok, head, chunk, b, page, slot, bad)) return;
  TO yk[8], yv[8];
  if (bad) {
    if (head == 0 && chunk == 0) atomicOr(a.errflags, C4S_DEVERR_KV_PAGE);
#pragma unroll
    for (int i = 0; i < 8; ++i) yk[i] = yv[i] = Cvt<TO>::t(0.0f);
  } else {
    const long long row = kv_row(a.c, page, head, slot);
    const long long sb = BITS != 16 ? kv_sb(a.c, page, head, slot) : 0;
    kv_get<TC, TO, BITS>(a.c.k + row, a.c.k_sb + sb, chunk, a.c.group >> 3, yk);
    kv_get<TC, TO, BITS>(a.c.v + row, a.c.v_sb + sb, chunk, a.c.group >> 3, yv);
  }
  const long long s = tok * a.tstride + (long long)head * a.hstride + 8 * chunk;
  store8(static_cast<TO*>(const_cast<void*>(a.k)) + s, a.vec, yk);
  store8(static_cast<TO*>(const_cast<void*>(a.v)) + s, a.vec, yv);
}

}  // namespace c4s
