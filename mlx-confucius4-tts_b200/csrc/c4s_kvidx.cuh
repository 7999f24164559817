// c4s_kvidx.cuh -- index arithmetic of the paged key-value cache and of the
// attention's split over its length, shared by the kernels and compiled for
// the host by the CPU tests (no CUDA header is needed).
//
// Position p of sequence b lies in page table[b][p / page_size] at slot
// p % page_size. A position past the table's width, or a page outside the
// cache, has no place (kv_locate returns false; no address is formed from it).
//
// The attention's work is the list of every (sequence, head block) segment's
// tiles, in that order: sequence b has nt[b] tiles for each of its HB head
// blocks, P is the exclusive prefix sum of nt, and tile i of head block h is
// number P[b] HB + h nt[b] + i of T = P[B] HB. Worker w of W (never more
// workers than tiles) takes the tiles [T w / W, T (w + 1) / W): at least one,
// shares differ by at most one whatever the lengths, and a segment cut by a
// share's border is joined from the parts of consecutive workers.
#pragma once

#ifdef __CUDACC__
#define C4S_HD __host__ __device__ __forceinline__
#else
#define C4S_HD inline
#endif

namespace c4s {

C4S_HD bool kv_locate(const int* table_row, int max_pages, int num_pages, int page_size, long long pos, int& page,
                      int& slot) {
  const long long pi = (pos >= 0 && pos <= 0x7fffffffLL) ? (long long)((unsigned)pos / (unsigned)page_size)
                                                         : (pos < 0 ? -1 : pos / page_size);
  if (pi < 0 || pi >= max_pages) return false;
  const int pg = table_row[pi];
  if (pg < 0 || pg >= num_pages) return false;
  page = pg;
  slot = (int)(pos - pi * page_size);
  return true;
}

// Division by a page size d in a loop: for 0 <= n < 2^31 and d >= 1, with
// s = ceil(log2 d) and m = floor(2^(31+s) / d) + 1 (at most 2^32), n / d is
// n m >> (31 + s): m d = 2^(31+s) + e with 0 < e <= d <= 2^s, so n m / 2^(31+s)
// exceeds n / d by n e / (d 2^(31+s)) < 1 / d.
struct PageDiv {
  unsigned long long mul;
  int shift;
};
C4S_HD PageDiv page_div(int d) {
  int s = 0;
  while (s < 31 && (1LL << s) < d) ++s;
  return {((1ULL << (31 + s)) / (unsigned)d) + 1, 31 + s};
}
C4S_HD int page_of(const PageDiv& p, int n) { return (int)(((unsigned long long)(unsigned)n * p.mul) >> p.shift); }

// The visible positions [lo, hi) of a sequence: its length, cut to what the
// page table can name, from its first visible position on.
C4S_HD void kv_visible(int len, int start, int max_pages, int page_size, long long& lo, long long& hi) {
  const long long cap = (long long)max_pages * page_size;
  hi = len < 0 ? 0 : (len < cap ? len : cap);
  lo = start < 0 ? 0 : start;
  if (lo > hi) lo = hi;
}

C4S_HD long long kv_tiles(long long lo, long long hi, int tok) { return (hi - lo + tok - 1) / tok; }

// Workers that have a tile, of at most `most`.
C4S_HD int split_workers(long long T, int most) { return T < most ? (int)T : most; }

// First tile of worker w's share, and the worker whose share holds a tile.
C4S_HD long long split_begin(long long T, int W, int w) {
  return (long long)((unsigned long long)T * (unsigned)w / (unsigned)W);
}
C4S_HD int split_owner(long long T, int W, long long tile) {
  return (int)((((unsigned long long)tile + 1) * (unsigned)W - 1) / (unsigned long long)T);
}

// Largest b in [0, B) with P[b] <= x, for 0 <= x < P[B]: the sequence of tile
// x * HB + anything. Sequences without tiles (P[b] == P[b + 1]) are passed over.
template <typename I>
C4S_HD int split_sequence(const I* P, int B, long long x) {
  int a = 0, e = B;
  while (e - a > 1) {
    const int m = (a + e) >> 1;
    if (P[m] <= x) a = m; else e = m;
  }
  return a;
}

// Sequence of token t in the offsets off[0..B] (each sequence's tokens are
// contiguous): the last b with off[b] <= t; false where t is no sequence's.
C4S_HD bool token_sequence(const long long* off, int B, long long t, int& b) {
  int a = 0, e = B;
  while (e - a > 1) {
    const int m = (a + e) >> 1;
    if (off[m] <= t) a = m; else e = m;
  }
  b = a;
  return off[a] <= t && t < off[a + 1];
}

}  // namespace c4s
