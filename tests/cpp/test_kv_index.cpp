// Index arithmetic of the paged cache and of the attention's split
// (csrc/c4s_kvidx.cuh), compiled for the host: page lookups stay inside the
// table and the cache, shares tile the work, every tile has one owner.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../mlx-confucius4-tts_b200/csrc/c4s_kvidx.cuh"

using namespace c4s;

#define CHECK(x)                                              \
  do {                                                        \
    if (!(x)) {                                               \
      std::printf("line %d: %s\n", __LINE__, #x);             \
      return 1;                                               \
    }                                                         \
  } while (0)

int main() {
  std::mt19937_64 r(5);
  // page lookups
  {
    std::vector<int> row = {3, -1, 7, 2, 100};
    int pg = -5, sl = -5;
    CHECK(kv_locate(row.data(), 5, 8, 16, 0, pg, sl) && pg == 3 && sl == 0);
    CHECK(kv_locate(row.data(), 5, 8, 16, 63, pg, sl) && pg == 2 && sl == 15);
    CHECK(!kv_locate(row.data(), 5, 8, 16, 16, pg, sl));       // a page of -1
    CHECK(!kv_locate(row.data(), 5, 7, 16, 40, pg, sl));       // a page past the cache
    CHECK(!kv_locate(row.data(), 5, 8, 16, 64, pg, sl));
    CHECK(!kv_locate(row.data(), 5, 8, 16, 80, pg, sl));       // past the table
    CHECK(!kv_locate(row.data(), 5, 8, 16, -1, pg, sl));
    CHECK(!kv_locate(row.data(), 5, 8, 1, 1LL << 40, pg, sl));
    CHECK(!kv_locate(row.data(), 5, 8, 1, 0x7fffffffLL, pg, sl));
    std::vector<int> big(3, 0);
    big[2] = 9;
    CHECK(kv_locate(big.data(), 3, 10, 1500000000, 3000000001LL, pg, sl) && pg == 9 && sl == 1);
  }
  // the loop's division
  for (int it = 0; it < 300000; ++it) {
    const int d = it < 3000 ? it + 1 : 1 + (int)(r() % (it % 2 ? 70000u : 0x7fffffffu));
    const PageDiv p = page_div(d);
    CHECK(p.mul <= (1ULL << 32));
    const int edge = (int)((r() % (0x80000000ULL / d)) * d);
    for (int n : {0, 1, d - 1, edge, edge > 0 ? edge - 1 : 0, (int)(r() & 0x7fffffff), 0x7fffffff, 0x7ffffffe})
      CHECK(page_of(p, n) == n / d);
  }
  // visible ranges
  {
    long long lo, hi;
    kv_visible(-3, 0, 4, 16, lo, hi);
    CHECK(lo == 0 && hi == 0);
    kv_visible(100, 0, 4, 16, lo, hi);
    CHECK(lo == 0 && hi == 64);
    kv_visible(10, 12, 4, 16, lo, hi);
    CHECK(lo == 10 && hi == 10);
    kv_visible(10, -7, 4, 16, lo, hi);
    CHECK(lo == 0 && hi == 10);
    kv_visible(0x7fffffff, 5, 0x7fffffff, 0x7fffffff, lo, hi);
    CHECK(lo == 5 && hi == 0x7fffffff);
    CHECK(kv_tiles(0, 0, 32) == 0 && kv_tiles(0, 1, 32) == 1 && kv_tiles(3, 35, 32) == 1 && kv_tiles(3, 36, 32) == 2);
  }
  // shares and owners
  for (int it = 0; it < 4000; ++it) {
    const int most = 1 + (int)(r() % 2400);
    const long long T = it % 3 == 0 ? 1 + (long long)(r() % 64) : 1 + (long long)(r() % (it % 3 == 1 ? 40000 : (1LL << 37)));
    const int W = split_workers(T, most);
    CHECK(W >= 1 && W <= most && W <= T);
    CHECK(split_begin(T, W, 0) == 0 && split_begin(T, W, W) == T);
    for (int j = 0; j < 50; ++j) {
      const int w = (int)(r() % W);
      const long long a = split_begin(T, W, w), b = split_begin(T, W, w + 1);
      CHECK(a < b && b - a <= T / W + 1);                      // no worker without a tile
      CHECK(split_owner(T, W, a) == w && split_owner(T, W, b - 1) == w);
      const long long t = (long long)(r() % (unsigned long long)T);
      const int o = split_owner(T, W, t);
      CHECK(o >= 0 && o < W && split_begin(T, W, o) <= t && t < split_begin(T, W, o + 1));
    }
  }
  // sequences of tiles and of tokens, with empty ones among them
  for (int it = 0; it < 2000; ++it) {
    const int B = 1 + (int)(r() % 70);
    std::vector<long long> P(B + 1, 0);
    for (int b = 0; b < B; ++b) P[b + 1] = P[b] + (r() % 3 == 0 ? 0 : (long long)(r() % 9));
    for (long long x = 0; x < P[B]; ++x) {
      const int b = split_sequence(P.data(), B, x);
      CHECK(b >= 0 && b < B && P[b] <= x && x < P[b + 1]);
    }
    for (long long x = -2; x < P[B] + 3; ++x) {
      int b = -1;
      const bool in = token_sequence(P.data(), B, x, b);
      CHECK(b >= 0 && b < B);
      CHECK(in == (x >= 0 && x < P[B]));
      if (in) CHECK(P[b] <= x && x < P[b + 1]);
    }
  }
  std::printf("ok\n");
  return 0;
}
