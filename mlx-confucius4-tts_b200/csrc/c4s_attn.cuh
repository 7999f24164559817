// c4s_attn.cuh -- attention of one new token per sequence over the paged
// key-value cache (c4s_kv.cuh).
//
//     o[b, h] = sum_p softmax_p(c q[b, h] . k[p, h / G]) v[p, h / G],
//     p over the visible positions [start_b, len_b),
//
// in one pass over the keys and values with the running maximum m and sum l
// of the softmax: a tile with scores s moves m to m' = max(m, s), multiplies l
// and o by 2^(m - m') and adds 2^(s - m') and 2^(s - m') v. Parts of a
// sequence are joined by the same rule.
//
// What bounds it: every key and value row is read once from HBM and used by
// the G query heads that share it, 4 G flops per element. The kernel's work is
// to keep enough of those rows in flight.
//   * The tiles of all (sequence, head) segments form one list, split evenly
//     over all warps of the grid (c4s_kvidx.cuh), so that one long sequence,
//     many short ones and ragged batches all fill the machine, and lengths are
//     read on the device only (the call can be captured).
//   * Each warp runs its own pipeline of ATT stages of cp.async copies into
//     its own part of shared memory: no barrier of the CTA in the loop. Rows
//     are found through the page table by the lane that owns the token, one
//     tile ahead of the copies that need them.
//   * Scores and products go through mma.m16n8k16 with the TOKENS as rows
//     (S^T = K q^T, O^T = V^T P^T), since one new token has few query heads
//     per key head and sixteen rows of queries would be empty. The tensor
//     cores run far below their rate; tcgen05's 128 rows and its TMEM round
//     trips buy nothing here.
//   * P is not rounded to 16 bits: it is split into a high and a low half
//     that take two columns of the same product (a score block of 16 tokens x
//     4 heads makes 8 columns), so the output's error is its own rounding.
//     fp16 halves are taken of 2^15 P (full precision down to 2^-29 of the
//     largest weight); bf16 keys and values take bf16 halves.
//   * 8- and 4-bit codes enter the products as exact fp16 integers; scale and
//     bias act on the scores and on P: q.k = scale (q.code) + bias sum(q),
//     p v = (p scale) code + p bias, per group. q is scaled by a power of two
//     into fp16's upper range, p scale by the largest scale seen so far.
#pragma once

namespace c4s {

constexpr int ATT_WARPS = 4;                       // per CTA
constexpr int ATT_MAXB = 512;                      // sequences per launch (their prefix sums in shared memory)
constexpr int ATT_WARP_SMEM = 27648;               // stages of one warp: two CTAs of four warps per SM

struct AttnArgs {
  KvCache c;
  const int* table;
  long long table_ld;
  int max_pages, B;
  const void* q;                                   // [B, heads_q, D] by its strides (elements)
  long long qb, qh;
  int G;                                           // query heads per key head
  const int* len;
  const int* start;                                // or null
  float scale;                                     // times log2(e)
  void* out;
  long long ob, oh;
  float* part_o;                                   // [W][2][NQ][D]
  float* part_ml;                                  // [W][2][NQ][2]
  unsigned* errflags;
};

template <int D, int BITS, int GS>
struct AttnCfg {
  static constexpr int ROW = D * BITS / 8;                     // bytes of a cache row
  static constexpr int NG = BITS == 16 ? 1 : D / GS;           // quantization groups of a row
  static constexpr int TOK = ROW > (BITS == 16 ? 128 : 96) ? 16 : 32;   // tokens per tile
  // 16-bit rows: 8 rows of a matrix fall on different banks with an odd number of 16-byte chunks per
  // row; codes: rows 32 bytes (mod 64) apart
  static constexpr int PITCH = BITS == 16 ? ROW + 16 : (ROW % 64 == 32 ? ROW : ROW + 32);
  static constexpr int CH = ROW / 16;                          // 16-byte chunks per row
  static constexpr int STAGE = 2 * TOK * (PITCH + (BITS == 16 ? 0 : 8 * NG));   // bytes: keys, values, their scales
  static constexpr int STAGES = ATT_WARP_SMEM / STAGE < 4 ? ATT_WARP_SMEM / STAGE : 4;
  static constexpr int SMEM = ATT_WARPS * STAGES * STAGE;
  static_assert(TOK * CH % 32 == 0 && STAGES >= 3 && STAGE % 16 == 0, "whole copies per warp");
};

__device__ __forceinline__ void cp16(unsigned dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp8(unsigned dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool TRANS>
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// {low half: a, high half: b}
template <typename T> __device__ __forceinline__ unsigned pack2(T a, T b) {
  unsigned short x, y;
  memcpy(&x, &a, 2);
  memcpy(&y, &b, 2);
  return (unsigned)x | (unsigned)y << 16;
}
// p as a high and a low 16-bit half, hi + lo = p to 16 (bf16) or 22 (fp16) bits
template <typename T> __device__ __forceinline__ unsigned split2(float p) {
  const T hi = Cvt<T>::t(p);
  return pack2<T>(hi, Cvt<T>::t(p - Cvt<T>::f(hi)));
}
// four bytes {1024 + x} as two half2 minus 1024: codes as fp16 integers
__device__ __forceinline__ unsigned half_codes(unsigned magic) {
  unsigned y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(magic), "r"(0x64006400u));
  return y;
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(FULL, v, 1);
  return v + __shfl_xor_sync(FULL, v, 2);
}
__device__ __forceinline__ float rows_sum(float v) {        // over the eight lanes that share t
  v += __shfl_xor_sync(FULL, v, 4);
  v += __shfl_xor_sync(FULL, v, 8);
  return v + __shfl_xor_sync(FULL, v, 16);
}
__device__ __forceinline__ float rows_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
  return fmaxf(v, __shfl_xor_sync(FULL, v, 16));
}

// P[0..B]: exclusive prefix sums of the sequences' tiles (all threads of a
// CTA of 32 ATT_WARPS threads; `red` holds one value per warp).
__device__ __forceinline__ void attn_prefix(const AttnArgs& a, int tok, long long* P, long long* red) {
  const int tid = threadIdx.x, nt = 32 * ATT_WARPS;
  const int lane = tid & 31, warp = tid >> 5;
  long long base = 0;
  for (int b0 = 0; b0 < a.B; b0 += nt) {
    const int b = b0 + tid;
    long long x = 0;
    if (b < a.B) {
      long long lo, hi;
      kv_visible(a.len[b], a.start ? a.start[b] : 0, a.max_pages, a.c.page_size, lo, hi);
      x = kv_tiles(lo, hi, tok);
    }
    long long s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(FULL, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) red[warp] = s;
    __syncthreads();
    long long before = base, all = base;
    for (int w = 0; w < ATT_WARPS; ++w) {
      if (w < warp) before += red[w];
      all += red[w];
    }
    if (b < a.B) P[b] = before + s - x;
    base = all;
    __syncthreads();
  }
  if (tid == 0) P[a.B] = base;
  __syncthreads();
}

// A place in the list of tiles: tile i of nt of head block h of sequence b.
struct AttnCursor {
  int b, h, HB;
  long long i, nt, lo, hi;
  __device__ __forceinline__ void sequence(const AttnArgs& a, const long long* P) {
    kv_visible(a.len[b], a.start ? a.start[b] : 0, a.max_pages, a.c.page_size, lo, hi);
    nt = P[b + 1] - P[b];
  }
  __device__ __forceinline__ void seek(const AttnArgs& a, const long long* P, int heads, long long tile) {
    HB = heads;
    b = split_sequence(P, a.B, tile / HB);
    sequence(a, P);
    const long long r = tile - P[b] * HB;
    h = (int)(r / nt);
    i = r - h * nt;
  }
  // to the next tile; the caller knows that there is one
  __device__ __forceinline__ void next(const AttnArgs& a, const long long* P) {
    if (++i < nt) return;
    i = 0;
    if (++h < HB) return;
    h = 0;
    do ++b; while (P[b + 1] == P[b]);
    sequence(a, P);
  }
};

// D: head dimension; BITS: of the cache (16: rows of T); GS: quantization
// group (of codes); NQ: query heads per pass, 4 or 8.
template <typename T, int D, int BITS, int GS, int NQ>
__global__ void __launch_bounds__(32 * ATT_WARPS) attn_kernel(AttnArgs a) {
  using Cfg = AttnCfg<D, BITS, GS>;
  using M = typename std::conditional<BITS == 16, T, __half>::type;   // type of the products' operands
  constexpr bool CODES = BITS != 16;
  constexpr int TOK = Cfg::TOK, PITCH = Cfg::PITCH, CH = Cfg::CH, ST = Cfg::STAGES, MB = TOK / 16;
  constexpr int NG = Cfg::NG;
  constexpr int KS = D / 16;                       // k-steps of a score block, and row blocks of O^T
  constexpr int QN = NQ / 4;                       // query heads that a lane owns
  constexpr int STAGE = Cfg::STAGE;
  constexpr float PSCALE = std::is_same<M, __half>::value ? 32768.0f : 1.0f;
  extern __shared__ __align__(16) unsigned char asm_raw[];
  __shared__ long long P[ATT_MAXB + 1];
  __shared__ long long red[ATT_WARPS];
  __shared__ unsigned tmask[ATT_WARPS][ST];        // a stage's visible tokens

  grid_dep_wait();                                 // the cache's and the query's producers
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  attn_prefix(a, TOK, P, red);
  const int QB = (a.G + NQ - 1) / NQ;              // passes over a key head's query heads
  const int HB = a.c.heads * QB, Hq = a.c.heads * a.G;

  // sequences with nothing to see: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (P[b + 1] != P[b]) continue;
    for (int j = threadIdx.x; j < Hq * D; j += 32 * ATT_WARPS)
      static_cast<T*>(a.out)[(long long)b * a.ob + (long long)(j / D) * a.oh + j % D] = Cvt<T>::t(0.0f);
  }

  const long long tiles = P[a.B] * HB;
  const int W = split_workers(tiles, gridDim.x * ATT_WARPS);
  const int w = warp * gridDim.x + blockIdx.x;     // few tiles spread over the SMs first
  if (w >= W) return;
  const long long t0 = split_begin(tiles, W, w), t1 = split_begin(tiles, W, w + 1);

  unsigned char* my = asm_raw + (size_t)warp * ST * STAGE;
  const unsigned my_s = smem_u32(my);

  // ---- the copies' side: one tile looked up ahead of the one being copied ----
  AttnCursor look;
  look.seek(a, P, HB, t0);
  long long looked = t0;                           // tiles looked up so far
  int lk_page = 0, lk_slot = 0, lk_head = 0;
  bool lk_ok = false;
  auto lookup = [&]() {                            // the page of this lane's token of the next tile
    if (looked > t0) look.next(a, P);
    ++looked;
    const long long pos = look.lo + look.i * TOK + lane;
    const bool in = lane < TOK && pos < look.hi;
    lk_head = look.h / QB;
    lk_ok = in && kv_locate(a.table + (long long)look.b * a.table_ld, a.max_pages, a.c.num_pages, a.c.page_size, pos,
                            lk_page, lk_slot);
    if (in && !lk_ok) atomicOr(a.errflags, C4S_DEVERR_KV_PAGE);
  };
  auto issue = [&](int stage) {                    // copies the tile that was looked up
    const unsigned mask = __ballot_sync(FULL, lk_ok);
    if (lane == 0) tmask[warp][stage] = mask;
    const long long off = lk_ok ? kv_row(a.c, lk_page, lk_head, lk_slot) : 0;
    const unsigned sk = my_s + stage * STAGE, sv = sk + TOK * PITCH;
#pragma unroll
    for (int j = 0; j < TOK * CH / 32; ++j) {
      const int idx = j * 32 + lane, row = idx / CH, c = idx - row * CH;
      const long long ro = __shfl_sync(FULL, off, row) + c * 16;
      const bool ok = (mask >> row) & 1u;
      cp16(sk + row * PITCH + c * 16, a.c.k + (ok ? ro : 0), ok);
      cp16(sv + row * PITCH + c * 16, a.c.v + (ok ? ro : 0), ok);
    }
    if constexpr (CODES) {
      const long long so = lk_ok ? kv_sb(a.c, lk_page, lk_head, lk_slot) : 0;
      const unsigned ss = sk + 2 * TOK * PITCH + lane * NG * 8;
      if (lane < TOK) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          cp8(ss + n * 8, a.c.k_sb + so + (lk_ok ? n * 8 : 0), lk_ok);
          cp8(ss + TOK * NG * 8 + n * 8, a.c.v_sb + so + (lk_ok ? n * 8 : 0), lk_ok);
        }
      }
    }
  };

  // ---- the products' side ----
  AttnCursor cur;
  cur.seek(a, P, HB, t0);
  unsigned qf[KS][2];                              // q as the B operand: column g, k-step's four elements
  float qmul[QN], qsum[CODES ? NG : 1][QN];
  float m[QN], l[QN], o[QN][KS][4], ob[CODES ? NG : 1][QN];
  float smax = 0.0f;                               // codes: largest value scale so far

  auto begin_segment = [&]() {
    const int qb = cur.h % QB, kvh = cur.h / QB;
    const int col = NQ == 4 ? ((g & 1) ? -1 : g >> 1) : g;          // query head of column g
    const int j = qb * NQ + col;
    const bool have = col >= 0 && j < a.G;
    const T* q = static_cast<const T*>(a.q) + (long long)cur.b * a.qb + (have ? (long long)(kvh * a.G + j) * a.qh : 0);
    float x[KS][4];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int d;
        if (!CODES) d = 16 * s + 2 * t + (e & 1) + 8 * (e >> 1);
        else if (BITS == 8) d = 32 * (s >> 1) + 8 * t + 4 * (s & 1) + e;
        else d = 32 * (s >> 1) + 8 * t + 2 * (s & 1) + (e >> 1) + 4 * (e & 1);   // a pair is (i, i + 4)
        x[s][e] = have ? Cvt<T>::f(q[d]) : 0.0f;
      }
    float up = 1.0f, down = 1.0f;
    if constexpr (CODES) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][e]));
      top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
      top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
      // 2^e with 2^13 <= top 2^e < 2^14, e within fp32's exponents
      int e = 140 - (int)((__float_as_uint(top) >> 23) & 0xffu);      // 13 - (exponent - 127)
      e = max(-100, min(100, e));
      up = __uint_as_float((unsigned)(127 + e) << 23);
      down = __uint_as_float((unsigned)(127 - e) << 23);
      float gs[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) gs[n] = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          x[s][e2] *= up;
          gs[16 * s / GS] += __half2float(__float2half_rn(x[s][e2]));
        }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float v = quad_sum(gs[n]);
#pragma unroll
        for (int u = 0; u < QN; ++u) qsum[n][u] = __shfl_sync(FULL, v, 4 * (2 * t + u));
      }
    }
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      qmul[u] = a.scale * __shfl_sync(FULL, down, 4 * (2 * t + u));
      m[u] = -INFINITY;
      l[u] = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][s][e] = 0.0f;
#pragma unroll
      for (int n = 0; n < NG; ++n) ob[CODES ? n : 0][u] = 0.0f;
    }
    smax = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s][0] = pack2<M>(Cvt<M>::t(x[s][0]), Cvt<M>::t(x[s][1]));
      qf[s][1] = pack2<M>(Cvt<M>::t(x[s][2]), Cvt<M>::t(x[s][3]));
    }
  };

  auto compute = [&](int stage) {
    const unsigned sk = my_s + stage * STAGE, sv = sk + TOK * PITCH;
    const unsigned char* pk = my + stage * STAGE;
    const unsigned char* pv = pk + TOK * PITCH;
    const float2* ksb = reinterpret_cast<const float2*>(pk + 2 * TOK * PITCH);
    const float2* vsb = ksb + TOK * NG;
    const unsigned mask = tmask[warp][stage];
    // scores of the tile: rows g and g + 8 of each 16-token block, the lane's query heads
    float s[MB][2][QN];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float acc[NG][4];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
      if constexpr (!CODES) {
        const unsigned base = sk + (mb * 16 + (lane & 15)) * PITCH + (lane >> 4) * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          unsigned r[4];
          ldsm4<false>(r, base + ks * 32);
          mma16816<M>(acc[0], r, qf[ks][0], qf[ks][1]);
        }
      } else {
        const unsigned char* r0 = pk + (mb * 16 + g) * PITCH + t * BITS;     // 8 codes: BITS bytes
        const unsigned char* r1 = r0 + 8 * PITCH;
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
          unsigned f[2][4];
          if constexpr (BITS == 8) {
            const uint2 x = *reinterpret_cast<const uint2*>(r0 + 32 * blk);
            const uint2 y = *reinterpret_cast<const uint2*>(r1 + 32 * blk);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned xw = h ? x.y : x.x, yw = h ? y.y : y.x;
              f[h][0] = half_codes(__byte_perm(xw, 0x64646464u, 0x4140));
              f[h][1] = half_codes(__byte_perm(yw, 0x64646464u, 0x4140));
              f[h][2] = half_codes(__byte_perm(xw, 0x64646464u, 0x4342));
              f[h][3] = half_codes(__byte_perm(yw, 0x64646464u, 0x4342));
            }
          } else {
            const unsigned x = *reinterpret_cast<const unsigned*>(r0 + 16 * blk);
            const unsigned y = *reinterpret_cast<const unsigned*>(r1 + 16 * blk);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f[h][0] = half_codes(((x >> (8 * h)) & 0x000f000fu) | 0x64006400u);
              f[h][1] = half_codes(((y >> (8 * h)) & 0x000f000fu) | 0x64006400u);
              f[h][2] = half_codes(((x >> (8 * h + 4)) & 0x000f000fu) | 0x64006400u);
              f[h][3] = half_codes(((y >> (8 * h + 4)) & 0x000f000fu) | 0x64006400u);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) mma16816<M>(acc[32 * blk / GS], f[h], qf[2 * blk + h][0], qf[2 * blk + h][1]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tok = mb * 16 + 8 * r + g;
        const bool seen = (mask >> tok) & 1u;
        float2 sb[NG];
        if constexpr (CODES)
#pragma unroll
          for (int n = 0; n < NG; ++n) sb[n] = ksb[tok * NG + n];
#pragma unroll
        for (int u = 0; u < QN; ++u) {
          float v;
          if constexpr (CODES) {
            v = 0.0f;
#pragma unroll
            for (int n = 0; n < NG; ++n) v = fmaf(sb[n].x, acc[n][2 * r + u], fmaf(sb[n].y, qsum[n][u], v));
          } else {
            v = acc[0][2 * r + u];
          }
          s[mb][r][u] = seen ? v * qmul[u] : -INFINITY;
        }
      }
    }
    // running maximum and sum
    float alpha[QN], base[QN];
    bool moved = false;
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      float mx = s[0][0][u];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) mx = fmaxf(mx, fmaxf(s[mb][0][u], s[mb][1][u]));
      mx = fmaxf(m[u], rows_max(mx));
      base[u] = mx == -INFINITY ? 0.0f : mx;
      alpha[u] = exp2f(m[u] - base[u]);
      moved |= mx != m[u];
      m[u] = mx;
    }
    float beta = 1.0f, sinv = 1.0f;
    if constexpr (CODES) {
      // scales are >= 0 (or NaN): their bits order as they do
      unsigned top = 0u;
      if (lane < TOK)
#pragma unroll
        for (int n = 0; n < NG; ++n) top = max(top, __float_as_uint(vsb[lane * NG + n].x) & 0x7fffffffu);
      const float ns = __uint_as_float(max(__reduce_max_sync(FULL, top), __float_as_uint(smax)));
      if (!(ns == smax)) {
        beta = smax / ns;
        smax = ns;
        moved = true;
      }
      sinv = smax > 0.0f || smax != smax ? PSCALE / smax : 0.0f;
    }
    if (__any_sync(FULL, moved)) {
#pragma unroll
      for (int u = 0; u < QN; ++u) {
        l[u] *= alpha[u];
        if constexpr (CODES)
#pragma unroll
          for (int n = 0; n < NG; ++n) ob[n][u] *= alpha[u];
        const float f = alpha[u] * beta;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[u][ks][e] *= f;
      }
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      unsigned pf[CODES ? NG : 1][QN][2];          // P^T as the B operand: tokens 2t, 2t+1 (+8) of column g
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float2 sb[NG];
        if constexpr (CODES)
#pragma unroll
          for (int n = 0; n < NG; ++n) sb[n] = vsb[(mb * 16 + 8 * r + g) * NG + n];
#pragma unroll
        for (int u = 0; u < QN; ++u) {
          const float p = exp2f(s[mb][r][u] - base[u]);
          l[u] += p;
          if constexpr (CODES) {
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              ob[n][u] = fmaf(p, sb[n].y, ob[n][u]);
              pf[n][u][r] = transpose8x8(split2<M>(p * (sb[n].x * sinv)));
            }
          } else {
            pf[0][u][r] = transpose8x8(split2<M>(p * PSCALE));
          }
        }
      }
      if constexpr (!CODES) {
        const unsigned vb = sv + (mb * 16 + (lane & 7) + ((lane >> 4) << 3)) * PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          unsigned r[4];
          ldsm4<true>(r, vb + ks * 32);
#pragma unroll
          for (int u = 0; u < QN; ++u) mma16816<M>(o[u][ks], r, pf[0][u][0], pf[0][u][1]);
        }
      } else {
        // a group of GS dims: this lane's GS / 8 consecutive ones (from g GS / 8) for tokens 2t, 2t+1, +8, +9
        const unsigned char* r0 = pv + (mb * 16 + 2 * t) * PITCH + g * (GS * BITS / 64);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const unsigned char* rn = r0 + n * (GS * BITS / 8);
          unsigned f[GS / 16][4];                  // [row block][a0..a3]
#pragma unroll
          for (int hv = 0; hv < 2; ++hv) {         // tokens 2t, 2t+1, then 2t+8, 2t+9
            const unsigned char* ra = rn + 8 * hv * PITCH;
            const unsigned char* rb = ra + PITCH;
            if constexpr (BITS == 8) {
#pragma unroll
              for (int wd = 0; wd < GS / 32; ++wd) {
                const unsigned xa = reinterpret_cast<const unsigned*>(ra)[wd];
                const unsigned xb = reinterpret_cast<const unsigned*>(rb)[wd];
                const unsigned lo = __byte_perm(xa, xb, 0x5140), hi = __byte_perm(xa, xb, 0x7362);
                f[2 * wd][2 * hv] = half_codes(__byte_perm(lo, 0x64646464u, 0x4140));
                f[2 * wd][2 * hv + 1] = half_codes(__byte_perm(lo, 0x64646464u, 0x4342));
                f[2 * wd + 1][2 * hv] = half_codes(__byte_perm(hi, 0x64646464u, 0x4140));
                f[2 * wd + 1][2 * hv + 1] = half_codes(__byte_perm(hi, 0x64646464u, 0x4342));
              }
            } else {
#pragma unroll
              for (int wd = 0; wd < GS / 32; ++wd) {
                const unsigned xa = reinterpret_cast<const unsigned short*>(ra)[wd];
                const unsigned xb = reinterpret_cast<const unsigned short*>(rb)[wd];
                const unsigned x = xa | xb << 16;
                f[2 * wd][2 * hv] = half_codes((x & 0x000f000fu) | 0x64006400u);
                f[2 * wd][2 * hv + 1] = half_codes(((x >> 4) & 0x000f000fu) | 0x64006400u);
                f[2 * wd + 1][2 * hv] = half_codes(((x >> 8) & 0x000f000fu) | 0x64006400u);
                f[2 * wd + 1][2 * hv + 1] = half_codes(((x >> 12) & 0x000f000fu) | 0x64006400u);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < GS / 16; ++j)
#pragma unroll
            for (int u = 0; u < QN; ++u) mma16816<M>(o[u][n * (GS / 16) + j], f[j], pf[n][u][0], pf[n][u][1]);
        }
      }
    }
  };

  // the segment (or this warp's part of it) is done: to the output, or to the parts
  auto end_segment = [&](bool first, bool last) {
    const int qb = cur.h % QB, kvh = cur.h / QB;
    const float back = CODES ? smax / PSCALE : 1.0f / PSCALE;
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      const int jq = NQ == 4 ? t : 2 * t + u;      // within the pass
      const int j = qb * NQ + jq;
      const float lt = rows_sum(l[u]);
      float bias[CODES ? NG : 1];
      if constexpr (CODES)
#pragma unroll
        for (int n = 0; n < NG; ++n) bias[n] = rows_sum(ob[n][u]);
      if (j >= a.G) continue;
      const bool whole = first && last;
      const float f = whole ? 1.0f / lt : 1.0f;
      T* out = static_cast<T*>(a.out) + (long long)cur.b * a.ob + (long long)(kvh * a.G + j) * a.oh;
      const long long slot = ((long long)w * 2 + (first ? 1 : 0)) * NQ + jq;
      float* po = a.part_o + slot * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = (o[u][ks][2 * e] + o[u][ks][2 * e + 1]) * back;
          int d;
          if constexpr (CODES) {
            constexpr int RB = GS / 16;            // row blocks per group
            d = (ks / RB) * GS + g * (GS / 8) + 2 * (ks % RB) + e;
            v += bias[ks / RB];
          } else {
            d = 16 * ks + 8 * e + g;
          }
          if (whole) out[d] = Cvt<T>::t(v * f);
          else po[d] = v;
        }
      if (!whole && g == 0) {
        a.part_ml[slot * 2] = m[u];
        a.part_ml[slot * 2 + 1] = lt;
      }
    }
  };

  lookup();
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    if (t0 + s < t1) {
      issue(s);
      if (looked < t1) lookup();
    }
    cp_commit();
  }
  long long seg_first = cur.i;                     // first tile of the segment that is this warp's
  begin_segment();
  int stage = 0;
  for (long long n = t0; n < t1; ++n) {
    cp_wait<ST - 2>();
    __syncwarp();
    if (n + ST - 1 < t1) {
      issue(stage == 0 ? ST - 1 : stage - 1);
      if (looked < t1) lookup();
    }
    cp_commit();
    compute(stage);
    stage = stage + 1 == ST ? 0 : stage + 1;
    const bool seg_end = cur.i + 1 == cur.nt;
    if (seg_end || n + 1 == t1) end_segment(seg_first == 0, seg_end);
    if (n + 1 < t1) {
      cur.next(a, P);
      if (seg_end) {
        seg_first = 0;
        begin_segment();
      }
    }
  }
}

// Joins the segments that a border between two warps' shares cuts: the CTA of
// the warp that began one (blockIdx.x) sums the parts of all warps up to the
// one that ended it, in that order of weights whatever their timing.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(32 * ATT_WARPS) attn_join_kernel(AttnArgs a, int tok) {
  constexpr int NTH = 32 * ATT_WARPS;
  __shared__ long long P[ATT_MAXB + 1];
  __shared__ long long red[ATT_WARPS];
  __shared__ float fred[ATT_WARPS];
  __shared__ __align__(16) float osum[NTH / (D / 4) + 1][D];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  attn_prefix(a, tok, P, red);
  const int QB = (a.G + NQ - 1) / NQ, HB = a.c.heads * QB;
  const long long tiles = P[a.B] * HB;
  const int W = split_workers(tiles, gridDim.x), w = blockIdx.x;
  if (w >= W) return;
  const long long t0 = split_begin(tiles, W, w), t1 = split_begin(tiles, W, w + 1);
  AttnCursor cur;
  cur.seek(a, P, HB, t1 - 1);
  const long long seg0 = t1 - 1 - cur.i, seg1 = seg0 + cur.nt;
  if (seg0 < t0 || seg1 <= t1) return;             // begun by an earlier warp, or not cut
  const int last = split_owner(tiles, W, seg1 - 1);
  const int qb = cur.h % QB, kvh = cur.h / QB;
  const int parts = last - w + 1;
  auto slot = [&](int i, int jq) { return ((long long)(w + i) * 2 + (i == 0 ? 1 : 0)) * NQ + jq; };
  for (int jq = 0; jq < NQ && qb * NQ + jq < a.G; ++jq) {
    float mx = -INFINITY;
    for (int i = tid; i < parts; i += NTH) mx = fmaxf(mx, a.part_ml[slot(i, jq) * 2]);
    mx = warp_reduce(mx, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) fred[warp] = mx;
    __syncthreads();
    mx = fred[0];
    for (int i = 1; i < ATT_WARPS; ++i) mx = fmaxf(mx, fred[i]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    __syncthreads();
    constexpr int COLS = D / 4, GR = NTH / COLS;   // threads: GR groups of parts x COLS columns of four
    const int col = tid % COLS, gr = tid / COLS;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
    if (gr < GR) {
      for (int i = gr; i < parts; i += GR) {
        const long long s = slot(i, jq);
        const float f = exp2f(a.part_ml[s * 2] - base);
        const float4 v = reinterpret_cast<const float4*>(a.part_o + s * D)[col];
        l = fmaf(f, a.part_ml[s * 2 + 1], l);
        o.x = fmaf(f, v.x, o.x);
        o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z);
        o.w = fmaf(f, v.w, o.w);
      }
      reinterpret_cast<float4*>(osum[gr])[col] = o;
      if (col == 0) osum[GR][gr] = l;
    }
    __syncthreads();
    float lt = 0.0f;
    for (int i = 0; i < GR; ++i) lt += osum[GR][i];
    T* out = static_cast<T*>(a.out) + (long long)cur.b * a.ob + (long long)(kvh * a.G + qb * NQ + jq) * a.oh;
    for (int d = tid; d < D; d += NTH) {
      float v = 0.0f;
      for (int i = 0; i < GR; ++i) v += osum[i][d];
      out[d] = Cvt<T>::t(v / lt);
    }
    __syncthreads();
  }
}

}  // namespace c4s
