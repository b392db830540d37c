// The tile of an 8-bit product, and the CTAs that share a tile's depth.
#pragma once

namespace nncv_b200 {
namespace e4m3 {

struct Tile { int m, n; double block, more, round, launch; };
// 128 x 64, 128 x 128, and on CTA pairs 256 x 128, 256 x 256.
constexpr int kTiles = 4, kSingle = 2;   // the first two on single CTAs, which a cluster may share
inline const Tile& tile(int i) {
  static const Tile t[kTiles] = {{128, 64, 0.16, 0.11, 0.75, 1.7}, {128, 128, 0.17, 0.20, 1.0, 1.8}, {256, 128, 0.27, 0.0, 1.1, 2.2}, {256, 256, 0.42, 0.0, 2.5, 2.0}};
  return t[i];
}
struct Choice { int tile, splits; };
// Clusters of 1, 2, 4 and 8 CTAs that run at once, by size, for either single tile.
struct Room { const int* of[kSingle]; int sms; };

inline long long items(int i, int M, int N) { return ((long long)M + tile(i).m - 1) / tile(i).m * (((long long)N + tile(i).n - 1) / tile(i).n); }
inline long long slots(int i, int s, const Room& r) { return i >= kSingle ? r.sms / 2 : s == 1 ? r.sms : r.of[i][s]; }
// A cluster has one tile, and each of its CTAs at least one block of the KB.
inline bool fits(int i, int s, int M, int N, int KB, const Room& r) {
  if (i < 0 || i >= kTiles || (s != 1 && s != 2 && s != 4 && s != 8)) return false;
  return s == 1 || (i < kSingle && items(i, M, N) <= slots(i, s, r) && KB >= s);
}

// The least of a model's times, in us: rounds x (blocks x time of one + end of a tile) + launch (+ exchange of partial sums).  A block of 128
// takes longer with more rows of A, up to a whole tile.  The constants are fitted to 90 shapes (M and N 1 .. 8192, K 16 .. 8192), each
// timed with every tile and split that fits: the choice is 0.5 % above the fastest on average, 9 % at worst (1024^3: 128 x 64 6.0 us,
// 256 x 128 on pairs 5.5).
inline Choice choose(int M, int N, int KB, const Room& r) {
  const double rows = (M < 128 ? M : 128) / 128.0;
  Choice best{0, 1};
  double least = 1e30;
  for (int i = 0; i < kTiles; ++i) {
    const Tile& t = tile(i);
    const long long n = items(i, M, N);
    for (int s = 1; s <= 8; s *= 2) {
      if (!fits(i, s, M, N, KB, r)) break;
      const long long at_once = slots(i, s, r);
      double us = (double)((n + at_once - 1) / at_once) * ((KB + s - 1) / s * (t.block + t.more * rows) + t.round) + t.launch;
      if (s > 1) us += 0.8 + 1.8 * rows * (i + 1);
      if (us < least) { least = us; best = {i, s}; }
    }
  }
  return best;
}

}  // namespace e4m3
}  // namespace nncv_b200
