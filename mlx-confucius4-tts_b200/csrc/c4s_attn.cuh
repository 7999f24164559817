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
//     p v = (p scale) code + p bias, per group (of codes centred on zero). q is scaled by a power of two
//     into fp16's upper range, p scale by the largest scale seen so far.
#pragma once

namespace c4s {

constexpr int ATT_CTAS = 2;                        // per SM: what registers and shared memory are sized for
constexpr int ATT_MAXB = 256;                      // sequences per launch (their prefix sums in shared memory)
constexpr int ATT_JOIN_NT = 128;

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
  PageDiv pdiv;                                    // by the page size
  float* part_o;                                   // [warps][2][NQ][D]
  float* part_ml;                                  // [warps][2][NQ][2]
  int4* cut;                                       // [warps] the segment that a warp began and did not end:
                                                   // {parts (0: none), sequence, key head, pass}
  unsigned* errflags;
};

// Two CTAs per SM, of eight warps (six where a lane holds two query heads, or
// where rows are long): more warps hide more of a tile's chain of dependent
// steps (copy, product, maximum, exponential, product) than longer tiles do.
template <int D, int BITS, int GS, int NQ>
struct AttnCfg {
  static constexpr int ROW = D * BITS / 8;                     // bytes of a cache row
  static constexpr int NG = BITS == 16 ? 1 : D / GS;           // quantization groups of a row
  static constexpr int TOK = ROW <= (BITS == 16 ? 128 : 96) ? 32 : 16;              // tokens per tile
  static constexpr int PITCH = BITS == 16 && ROW % 128 ? ROW + 16 : ROW;
  static constexpr int CH = ROW / 16;                          // 16-byte chunks per row
  static constexpr int STAGE = 2 * TOK * (PITCH + (BITS == 16 ? 0 : 8 * NG));   // bytes: keys, values, their scales
  static constexpr int ROOM8 = 13900, ROOM6 = 18500;           // bytes a warp of eight, of six
  static constexpr int WARPS = NQ == 4 && ROOM8 / STAGE >= 2 ? 8 : 6;
  static constexpr int ROOM = WARPS == 8 ? ROOM8 : ROOM6;
  static constexpr int STAGES = ROOM / STAGE < 4 ? ROOM / STAGE : 4;
  static constexpr int SMEM = WARPS * STAGES * STAGE;
  // lanes copy row groups: RL lanes a row (its chunks), RG rows at once, RPG rows a lane group
  static constexpr int RG = CH > 8 ? 2 : CH > 4 ? 4 : CH > 2 ? 8 : 16;
  static constexpr int RPG = TOK / RG;
  static_assert(STAGES >= 2 && STAGE % 16 == 0 && CH * RG <= 32 && RPG % 2 == 0, "a tile's copies");

  // Row r's 16-byte chunks are stored at chunk ^ swz(r), so that the rows that
  // one read instruction touches lie on different banks: eight rows of 128
  // (or 256) bytes for ldmatrix; for codes the four rows whose 32 bytes a
  // half-warp reads. 192-byte rows are padded instead.
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (BITS == 16) return ROW % 128 == 0 ? (r & 7) : 0;
    else if constexpr (ROW == 128) return 2 * (((r & 7) + ((r >> 2) & 1)) & 3);
    else if constexpr (ROW == 64) return 2 * ((r >> 1) & 1);
    else return 0;
  }
};

__device__ __forceinline__ void cp16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// ... zeros in its place where !ok (nothing is read)
__device__ __forceinline__ void cp16z(unsigned dst, const void* src, bool ok) {
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
// Two halves 1024 + code to code - 2^(BITS - 1): exact, and centred, since sums
// of codes of one sign would carry the accumulator's truncation as a bias.
template <int BITS> __device__ __forceinline__ unsigned half_codes(unsigned magic) {
  unsigned y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(magic), "r"(BITS == 8 ? 0x64806480u : 0x64086408u));
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

// P[0..B]: exclusive prefix sums of the sequences' tiles (all threads of the
// CTA; `red` holds one value per warp).
template <int WARPS>
__device__ __forceinline__ void attn_prefix(const AttnArgs& a, int tok, int* P, int* red) {
  constexpr int NTH = 32 * WARPS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += NTH) {
    const int b = b0 + tid;
    int x = 0;
    if (b < a.B) {
      long long lo, hi;
      kv_visible(a.len[b], a.start ? a.start[b] : 0, a.max_pages, a.c.page_size, lo, hi);
      x = (int)kv_tiles(lo, hi, tok);
    }
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(FULL, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) red[warp] = s;
    __syncthreads();
    int before = base, all = base;
    for (int w = 0; w < WARPS; ++w) {
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

// A place in the list of tiles: tile i of nt of pass qb over key head kvh of
// sequence b, whose visible positions are [lo, hi).
struct AttnCursor {
  int b, kvh, qb, i, nt;
  unsigned lo, hi;
  __device__ __forceinline__ void sequence(const AttnArgs& a, const int* P) {
    long long l, h;
    kv_visible(a.len[b], a.start ? a.start[b] : 0, a.max_pages, a.c.page_size, l, h);
    lo = (unsigned)l;
    hi = (unsigned)h;
    nt = P[b + 1] - P[b];
  }
  __device__ __forceinline__ void seek(const AttnArgs& a, const int* P, int QB, long long tile) {
    const int HB = a.c.heads * QB;
    const long long x = tile / HB;
    b = split_sequence(P, a.B, x);
    sequence(a, P);
    const long long r = tile - (long long)P[b] * HB;
    const int h = (int)(r / nt);
    i = (int)(r - (long long)h * nt);
    kvh = h / QB;
    qb = h - kvh * QB;
  }
  // to the next segment; the caller knows that there is one
  __device__ __forceinline__ void next_segment(const AttnArgs& a, const int* P, int QB) {
    i = 0;
    if (++qb < QB) return;
    qb = 0;
    if (++kvh < a.c.heads) return;
    kvh = 0;
    do ++b; while (P[b + 1] == P[b]);
    sequence(a, P);
  }
};

// D: head dimension; BITS: of the cache (16: rows of T); GS: quantization
// group (of codes); NQ: query heads per pass, 4 or 8.
template <typename T, int D, int BITS, int GS, int NQ>
__global__ void __launch_bounds__(32 * AttnCfg<D, BITS, GS, NQ>::WARPS, ATT_CTAS) attn_kernel(AttnArgs a) {
  using Cfg = AttnCfg<D, BITS, GS, NQ>;
  using M = typename std::conditional<BITS == 16, T, __half>::type;   // type of the products' operands
  constexpr bool CODES = BITS != 16;
  constexpr int TOK = Cfg::TOK, PITCH = Cfg::PITCH, ST = Cfg::STAGES, MB = TOK / 16, WARPS = Cfg::WARPS;
  constexpr int NG = Cfg::NG;
  constexpr int KS = D / 16;                       // k-steps of a score block, and row blocks of O^T
  constexpr int QN = NQ / 4;                       // query heads that a lane owns
  constexpr int STAGE = Cfg::STAGE;
  constexpr float PSCALE = std::is_same<M, __half>::value ? 32768.0f : 1.0f;
  constexpr float MID = (float)(1 << (BITS - 1));  // codes: value = scale (code - MID) + (bias + MID scale)
  constexpr unsigned ALL = TOK == 32 ? 0xffffffffu : 0xffffu;
  extern __shared__ __align__(128) unsigned char asm_raw[];
  __shared__ int P[ATT_MAXB + 1];
  __shared__ int red[WARPS];
  __shared__ unsigned tmask[WARPS][ST];            // a stage's visible tokens
  __shared__ __align__(16) long long roff[WARPS][TOK];   // byte offsets of the rows of the tile being copied

  grid_dep_wait();                                 // the cache's and the query's producers
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  attn_prefix<WARPS>(a, TOK, P, red);
  const int QB = (a.G + NQ - 1) / NQ;              // passes over a key head's query heads

  // sequences with nothing to see: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (P[b + 1] != P[b]) continue;
    for (int j = threadIdx.x; j < a.c.heads * a.G * D; j += 32 * WARPS)
      static_cast<T*>(a.out)[(long long)b * a.ob + (long long)(j / D) * a.oh + j % D] = Cvt<T>::t(0.0f);
  }

  const long long tiles = (long long)P[a.B] * (a.c.heads * QB);
  const int W = split_workers(tiles, gridDim.x * WARPS);
  const int w = warp * gridDim.x + blockIdx.x;     // few tiles spread over the SMs first
  if (w >= W) {
    if (lane == 0) a.cut[w] = make_int4(0, 0, 0, 0);
    return;
  }
  const long long t0 = split_begin(tiles, W, w);
  const int count = (int)(split_begin(tiles, W, w + 1) - t0);

  unsigned char* my = asm_raw + warp * (ST * STAGE);
  const unsigned my_s = smem_u32(my);

  // ---- the copies' side: the page of each lane's token is looked up one tile ahead of its copy ----
  AttnCursor look;
  look.seek(a, P, QB, t0);
  int looked = 0;                                  // tiles looked up so far
  int lk_page = 0, lk_slot = 0;
  bool lk_in = false;
  auto lookup = [&]() {
    if (looked++ > 0 && ++look.i == look.nt) look.next_segment(a, P, QB);
    const unsigned pos = look.lo + look.i * TOK + lane;
    lk_in = lane < TOK && pos < look.hi;
    if (lk_in) {                                   // inside the table: hi is cut to its width
      const int pi = page_of(a.pdiv, (int)pos);
      lk_page = a.table[look.b * a.table_ld + pi];
      lk_slot = (int)pos - pi * a.c.page_size;
    }
  };
  // this lane's part in the copies: chunk c of rows rg RPG .. + RPG - 1
  constexpr int CH = Cfg::CH, RG = Cfg::RG, RPG = Cfg::RPG;
  const int rg = lane / CH, rc = lane - rg * CH;
  auto issue = [&](int stage, int kvh) {           // copies the tile that was looked up
    const bool ok = lk_in && (unsigned)lk_page < (unsigned)a.c.num_pages;
    if (lk_in && !ok) atomicOr(a.errflags, C4S_DEVERR_KV_PAGE);
    const unsigned mask = __ballot_sync(FULL, ok);
    if (lane == 0) tmask[warp][stage] = mask;
    if (lane < TOK) roff[warp][lane] = ok ? kv_row(a.c, lk_page, kvh, lk_slot) : 0;
    __syncwarp();
    const unsigned sk = my_s + stage * STAGE;
    if (rg < RG) {
      const unsigned char* kb = a.c.k + rc * 16;
      const unsigned char* vb = a.c.v + rc * 16;
      const longlong2* ro = reinterpret_cast<const longlong2*>(&roff[warp][rg * RPG]);
      const unsigned mine = mask >> (rg * RPG);
#pragma unroll
      for (int j = 0; j < RPG; j += 2) {
        const longlong2 o = ro[j / 2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = rg * RPG + j + e;
          const unsigned dst = sk + r * PITCH + ((rc ^ Cfg::swz(r)) << 4);
          const long long of = e ? o.y : o.x;
          if (mask == ALL) {
            cp16(dst, kb + of);
            cp16(dst + TOK * PITCH, vb + of);
          } else {
            const bool in = (mine >> (j + e)) & 1u;
            cp16z(dst, kb + of, in);
            cp16z(dst + TOK * PITCH, vb + of, in);
          }
        }
      }
    }
    if constexpr (CODES) {
      if (lane < TOK) {
        const long long so = ok ? kv_sb(a.c, lk_page, kvh, lk_slot) : 0;
        const unsigned ss = sk + 2 * TOK * PITCH + lane * NG * 8;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          cp8(ss + n * 8, a.c.k_sb + so + n * 8, ok);
          cp8(ss + TOK * NG * 8 + n * 8, a.c.v_sb + so + n * 8, ok);
        }
      }
    }
  };

  // ---- the products' side ----
  AttnCursor cur = look;
  unsigned qf[KS][2];                              // q as the B operand: column g, k-step's four elements
  float qmul[QN], qsum[CODES ? NG : 1][QN];
  float m[QN], l[QN], o[QN][KS][4], ob[CODES ? NG : 1][QN];
  float smax = 0.0f;                               // codes: largest value scale so far

  auto begin_segment = [&]() {
    const int qb = cur.qb, kvh = cur.kvh;
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
        const unsigned base = sk + (mb * 16 + (lane & 15)) * PITCH;
        const int x = Cfg::swz(lane & 15) ^ (lane >> 4);       // chunk 2 ks + (lane >> 4) of its row
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          unsigned r[4];
          ldsm4<false>(r, base + (((2 * ks) ^ x) << 4));
          mma16816<M>(acc[0], r, qf[ks][0], qf[ks][1]);
        }
      } else {
        const unsigned char* r0 = pk + (mb * 16 + g) * PITCH;                // rows g and g + 8: one swizzle
        const unsigned char* r1 = r0 + 8 * PITCH;
        const int x = Cfg::swz(g);
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
          unsigned f[2][4];
          if constexpr (BITS == 8) {
            const int at = ((2 * blk) ^ x) * 16 + t * 8;                     // 8 codes
            const uint2 u = *reinterpret_cast<const uint2*>(r0 + at);
            const uint2 v = *reinterpret_cast<const uint2*>(r1 + at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned xw = h ? u.y : u.x, yw = h ? v.y : v.x;
              f[h][0] = half_codes<BITS>(__byte_perm(xw, 0x64646464u, 0x4140));
              f[h][1] = half_codes<BITS>(__byte_perm(yw, 0x64646464u, 0x4140));
              f[h][2] = half_codes<BITS>(__byte_perm(xw, 0x64646464u, 0x4342));
              f[h][3] = half_codes<BITS>(__byte_perm(yw, 0x64646464u, 0x4342));
            }
          } else {
            const int at = (blk ^ x) * 16 + t * 4;                           // 8 codes
            const unsigned u = *reinterpret_cast<const unsigned*>(r0 + at);
            const unsigned v = *reinterpret_cast<const unsigned*>(r1 + at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f[h][0] = half_codes<BITS>(((u >> (8 * h)) & 0x000f000fu) | 0x64006400u);
              f[h][1] = half_codes<BITS>(((v >> (8 * h)) & 0x000f000fu) | 0x64006400u);
              f[h][2] = half_codes<BITS>(((u >> (8 * h + 4)) & 0x000f000fu) | 0x64006400u);
              f[h][3] = half_codes<BITS>(((v >> (8 * h + 4)) & 0x000f000fu) | 0x64006400u);
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
            for (int n = 0; n < NG; ++n)
              v = fmaf(sb[n].x, acc[n][2 * r + u], fmaf(fmaf(sb[n].x, MID, sb[n].y), qsum[n][u], v));
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
              ob[n][u] = fmaf(p, fmaf(sb[n].x, MID, sb[n].y), ob[n][u]);
              pf[n][u][r] = transpose8x8(split2<M>(p * (sb[n].x * sinv)));
            }
          } else {
            pf[0][u][r] = transpose8x8(split2<M>(p * PSCALE));
          }
        }
      }
      if constexpr (!CODES) {
        const unsigned vb = sv + (mb * 16 + (lane & 7) + ((lane >> 4) << 3)) * PITCH;
        const int x = Cfg::swz(lane & 7) ^ ((lane >> 3) & 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          unsigned r[4];
          ldsm4<true>(r, vb + (((2 * ks) ^ x) << 4));
#pragma unroll
          for (int u = 0; u < QN; ++u) mma16816<M>(o[u][ks], r, pf[0][u][0], pf[0][u][1]);
        }
      } else {
        // a group of GS dims: this lane's GS / 8 consecutive ones (from g GS / 8) for tokens 2t, 2t+1, +8, +9
        const unsigned char* r0 = pv + (mb * 16 + 2 * t) * PITCH;
        constexpr int LB = GS * BITS / 64;         // a lane's bytes of the group: 8, 4 or 2
        const int xa = Cfg::swz(2 * t), xb = Cfg::swz(2 * t + 1);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const int at = n * (GS * BITS / 8) + g * LB;
          const int ca = (((at >> 4) ^ xa) << 4) + (at & 15), cb = (((at >> 4) ^ xb) << 4) + (at & 15) + PITCH;
          unsigned f[GS / 16][4];                  // [row block][a0..a3]
#pragma unroll
          for (int hv = 0; hv < 2; ++hv) {         // tokens 2t, 2t+1, then 2t+8, 2t+9
            const unsigned char* ra = r0 + 8 * hv * PITCH + ca;
            const unsigned char* rb = r0 + 8 * hv * PITCH + cb;
            unsigned wa[2], wb[2];
            if constexpr (LB == 8) {
              const uint2 p = *reinterpret_cast<const uint2*>(ra), q = *reinterpret_cast<const uint2*>(rb);
              wa[0] = p.x, wa[1] = p.y, wb[0] = q.x, wb[1] = q.y;
            } else if constexpr (LB == 4) {
              wa[0] = *reinterpret_cast<const unsigned*>(ra), wb[0] = *reinterpret_cast<const unsigned*>(rb);
            } else {
              wa[0] = *reinterpret_cast<const unsigned short*>(ra), wb[0] = *reinterpret_cast<const unsigned short*>(rb);
            }
            if constexpr (BITS == 8) {
#pragma unroll
              for (int wd = 0; wd < GS / 32; ++wd) {
                const unsigned lo = __byte_perm(wa[wd], wb[wd], 0x5140), hi = __byte_perm(wa[wd], wb[wd], 0x7362);
                f[2 * wd][2 * hv] = half_codes<BITS>(__byte_perm(lo, 0x64646464u, 0x4140));
                f[2 * wd][2 * hv + 1] = half_codes<BITS>(__byte_perm(lo, 0x64646464u, 0x4342));
                f[2 * wd + 1][2 * hv] = half_codes<BITS>(__byte_perm(hi, 0x64646464u, 0x4140));
                f[2 * wd + 1][2 * hv + 1] = half_codes<BITS>(__byte_perm(hi, 0x64646464u, 0x4342));
              }
            } else {
#pragma unroll
              for (int wd = 0; wd < GS / 32; ++wd) {           // 16 bits: four codes of each token
                const unsigned x = __byte_perm(wa[0], wb[0], wd ? 0x7632 : 0x5410);
                f[2 * wd][2 * hv] = half_codes<BITS>((x & 0x000f000fu) | 0x64006400u);
                f[2 * wd][2 * hv + 1] = half_codes<BITS>(((x >> 4) & 0x000f000fu) | 0x64006400u);
                f[2 * wd + 1][2 * hv] = half_codes<BITS>(((x >> 8) & 0x000f000fu) | 0x64006400u);
                f[2 * wd + 1][2 * hv + 1] = half_codes<BITS>(((x >> 12) & 0x000f000fu) | 0x64006400u);
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
    const int qb = cur.qb, kvh = cur.kvh;
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
    if (s < count) {
      issue(s, look.kvh);
      __syncwarp();                                // the row offsets have been read
      if (looked < count) lookup();
    }
    cp_commit();
  }
  int seg_first = cur.i;                           // first tile of the segment that is this warp's
  begin_segment();
  int stage = 0;
  for (int n = 0; n < count; ++n) {
    cp_wait<ST - 2>();
    __syncwarp();
    if (n + ST - 1 < count) {
      issue(stage == 0 ? ST - 1 : stage - 1, look.kvh);
      if (looked < count) lookup();
    }
    cp_commit();
    compute(stage);
    stage = stage + 1 == ST ? 0 : stage + 1;
    const bool seg_end = cur.i + 1 == cur.nt;
    if (seg_end || n + 1 == count) end_segment(seg_first == 0, seg_end);
    if (n + 1 < count) {
      ++cur.i;
      if (seg_end) {
        cur.next_segment(a, P, QB);
        seg_first = 0;
        begin_segment();
      }
    } else if (lane == 0) {
      const bool cuts = seg_first == 0 && !seg_end;
      const long long end = t0 + n - cur.i + cur.nt;           // the tile behind the segment
      a.cut[w] = make_int4(cuts ? split_owner(tiles, W, end - 1) - w + 1 : 0, cur.b, cur.kvh, cur.qb);
    }
  }
}

// Joins the segments that a border between two warps' shares cuts: CTA (w, j)
// sums, for query head j of the pass, the parts of the segment that warp w
// began, in an order that depends on nothing but the lengths.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(ATT_JOIN_NT) attn_join_kernel(AttnArgs a) {
  constexpr int NTH = ATT_JOIN_NT, COLS = D / 4, GR = NTH / COLS;   // GR groups of parts x COLS columns of four
  __shared__ float fred[NTH / 32];
  __shared__ __align__(16) float osum[GR][D];
  __shared__ float lsum[GR];
  grid_dep_wait();
  grid_dep_launch();
  const int w = blockIdx.x, jq = blockIdx.y;
  const int4 cut = a.cut[w];
  const int parts = cut.x, j = cut.w * NQ + jq;
  if (parts == 0 || j >= a.G) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // part 0 is the warp's own (it began the segment), the others are what later warps continued
  auto slot = [&](int i) { return ((long long)(w + i) * 2 + (i == 0 ? 1 : 0)) * NQ + jq; };
  float mx = -INFINITY;
  for (int i = tid; i < parts; i += NTH) mx = fmaxf(mx, a.part_ml[slot(i) * 2]);
  mx = warp_reduce(mx, [](float x, float y) { return fmaxf(x, y); });
  if (lane == 0) fred[warp] = mx;
  __syncthreads();
  mx = fred[0];
#pragma unroll
  for (int i = 1; i < NTH / 32; ++i) mx = fmaxf(mx, fred[i]);
  const float base = mx == -INFINITY ? 0.0f : mx;
  const int col = tid % COLS, gr = tid / COLS;
  if (gr < GR) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
#pragma unroll 4
    for (int i = gr; i < parts; i += GR) {
      const long long s = slot(i);
      const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[s];
      const float4 v = reinterpret_cast<const float4*>(a.part_o + s * D)[col];
      const float f = exp2f(ml.x - base);
      l = fmaf(f, ml.y, l);
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    }
    reinterpret_cast<float4*>(osum[gr])[col] = o;
    if (col == 0) lsum[gr] = l;
  }
  __syncthreads();
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < GR; ++i) l += lsum[i];
  T* out = static_cast<T*>(a.out) + (long long)cut.y * a.ob + (long long)(cut.z * a.G + j) * a.oh;
  if (tid < D) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < GR; ++i) v += osum[i][tid];
    out[tid] = Cvt<T>::t(v / l);
  }
}

}  // namespace c4s
