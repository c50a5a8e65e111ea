// Which tile shape a 16-bit product runs on, into how many slices of k it is cut, and whether a
// symmetric one computes its lower half or all of it.  Plain arithmetic without device state, so
// it also compiles for the host alone.
//
// Every candidate is priced by a model of its launch and the cheapest is taken.  Fitted to
// launches of 16 .. 2048 tiles with 16 .. 128 panels (64 elements of k) on 256 CUs, in us:
//   256 x 256   8 + 1.25 a panel, per round of one tile a CU
//   128 x 128   4.3 per round of two, and a panel 0.44 per tile of a CU, 0.5 at least
//    64 x 64    3.7 per round of four, and a panel 0.175 per tile of a CU, 0.3 at least
//   slices      3 for the second launch, and their bytes, written and read once, at 4 MB/us
//   the mirrored half of a symmetric product: 7 (narrow stores), 3 when slices are joined
// Examples (us, chosen / whole tiles of the other shapes): 4096 x 2048 x 2048 128: 33 / 64: 52, 256: 44;
// 2048 x 3584 x 4096 128: 57 / 64: 85, 256: 78; 1024^3 64: 6.7 / 128: 10, 256: 25; 768 x 768 x 8192 in
// slices 22 / 64: 28, 128: 45, 256: 144.
#pragma once
#include <stddef.h>

namespace rtat_native {

constexpr int PANEL16 = 64;       // elements of k in a panel
constexpr int SLICE_PANELS16 = 4; // a slice has at least this many

struct Plan16 {
  int tile;    // 256, 128 or 64
  int slices;  // 1: not cut
  int tri;     // 1: only the tiles on and below the diagonal are computed
};

// Floats between the columns of a slice's sums.
inline long slice_ld16(int m) { return ((long)m + 7) / 8 * 8; }

// Whether a product with both operands contiguous along k goes to the kernel for few columns, which
// cuts k across the waves of a workgroup only: a workgroup reads its sixteen rows at 0.63 us per 1024
// of k, whatever their number.  Few rows of a long k have too few workgroups to fill memory's pipe; slices
// of tiles, where there is scratch for them, have 64 times as many.  us, few columns / slices:
//   rows   k = 16384   20480     24576     32768     65536     1048576
//     16     13 / 14   15 / 14   18 / 13   23 / 14   44 / 16   682 / 60
//   1024     14 / 15   17 / 18   19 / 17   24 / 19   45 / 27
//   2048     16 / 20   17 / 22   20 / 24   25 / 29   49 / 44
//   4096     25 / 27   27 / 33   30 / 35   39 / 47  103 / 124
// (one column; where few columns are taken, the slices' time is that of 17).  Sixteen columns take
// up to 70 % longer here from 2048 x 65536 on, slices of them do not.
constexpr int FEW_COLS = 16;
constexpr int FEW_ROWS = 1 << 27;  // 2^23 workgroups of 256: a launch holds fewer than 2^32 threads
inline bool few_columns16(int m, int n, int k, size_t scratch) {
  if (n > FEW_COLS || m > FEW_ROWS || k % 8 != 0 || k == 0) return false;
  return scratch == 0 || m > 2048 || k <= (m <= 1024 ? 20480 : 32768);
}

inline double price16(int tile, long tiles, long panels, long cus) {
  const long w = (tiles + cus - 1) / cus;  // tiles of the busiest CU
  const double p = (double)panels;
  if (tile == 256) return (double)w * (8.0 + 1.25 * p);
  const double per = tile == 128 ? 0.44 : 0.175, least = tile == 128 ? 0.5 : 0.3;
  const double fixed = tile == 128 ? 4.3 * (double)((w + 1) / 2) : 3.7 * (double)((w + 3) / 4);
  const double panel = per * (double)w > least ? per * (double)w : least;
  return fixed + panel * p;
}

// `symmetric`: m == n and half of the product would do.  `large`: the 256 x 256 shape may be used.
// `scratch`: bytes that slices may take.
inline Plan16 plan16(int m, int n, int k, int batch, bool symmetric, bool large, size_t scratch,
                     long cus) {
  const long panels = ((long)k + PANEL16 - 1) / PANEL16;
  const double each = (double)slice_ld16(m) * (double)n * 4.0;
  Plan16 best = {64, 1, 0};
  double least = -1.0;
  const int shapes[3] = {256, 128, 64};
  for (int s = large ? 0 : 1; s < 3; ++s)
    for (int tri = symmetric ? 1 : 0; tri >= 0; --tri) {
      const int b = shapes[s];
      const long tm = ((long)m + b - 1) / b, tn = ((long)n + b - 1) / b;
      const long tiles = (tri ? tm * (tm + 1) / 2 : tm * tn) * batch;
      // The slices of a half are joined in blocks of the 128 x 128 tile.
      long most = batch == 1 && (!tri || b == 128) ? panels / SLICE_PANELS16 : 1;
      if (most > 64) most = 64;
      if (n > 65535 * 16) most = 1;  // the join's grid
      for (long cut = 1; cut <= (most > 1 ? most : 1); ++cut) {
        if (cut > 1 && (double)cut * each > (double)scratch) break;
        double us = price16(b, tiles * cut, (panels + cut - 1) / cut, cus);
        if (cut > 1) us += 3.0 + 2.0 * (double)cut * each * (tri ? 0.5 : 1.0) / 4e6;
        if (tri) us += cut > 1 ? 3.0 : 7.0;
        if (least < 0.0 || us < least) {
          least = us;
          best = {b, (int)cut, tri};
        }
      }
    }
  return best;
}

}  // namespace rtat_native
