// How the two passes of a prompt's attention weights are split over workgroups.  Host code, and the
// sizes of the kernels' tiles.
#pragma once
#include <stdint.h>

#define WG_COLS 256                // columns of a workgroup of the first pass, to a multiple of which they are padded
#define WG_SUM_COLS 128            // and of the second
#define WG_TILE 64                 // rows of a streamed tile
#define WG_ROWS 4096               // keys of a split at most

struct WeighPlan { int cols_pad, S, rows, S2, rows2, per, supers; bool joined, wide; };
static inline int weigh_up(int64_t n, int to) { return (int)((n + to - 1) / to * to); }
// Keys of a split, at least a tile: as many workgroups as run at a time, two to a compute unit in the first pass and three in the second.
// In the first one to a unit where two would have less than 1024 keys (one query, 32 heads, 8000 keys 16.5 us, with two 20.0; with more
// keys two even out unequal lengths, 24 of up to 8340 keys, 516 columns 73 us, with one 78).
// The second pass takes one block of columns to a workgroup, whose sums are a part of the result (8192 queries and keys, 32 heads:
// parts of 67 MB; two blocks to each, added up in LDS, 381 us instead of 334), and more of them where the parts would pass 256 MB.  Two blocks are one
// workgroup's of twice the waves (`wide`): they need not be added up by a launch of their own (256 columns, 8 heads: 2048 keys, 16
// sequences 46.6 us, apart 50.0; 32768 keys 48 and 52; 131072 169 and 176).  Up to 32 splits are joined by whoever needs them, more by a
// launch of their own (256 columns, 8 heads, 4096 keys: 16.4 us, with the launch 17.4; 64 splits of 8192 keys, four heads, 21.3 and 19.3).
static inline WeighPlan weigh_plan(int64_t groups, int cols, int T) {
  WeighPlan p;
  p.cols_pad = weigh_up(cols, WG_COLS);
  const auto split = [&](int64_t workgroups, int at_a_time, int least, int* rows, int* S) {
    int64_t want = (T * workgroups + at_a_time - 1) / at_a_time;
    if (want < least) want = 2 * want < least ? 2 * want : least;
    *rows = weigh_up(want < WG_TILE ? WG_TILE : want > WG_ROWS ? WG_ROWS : want, WG_TILE);
    *S = (T + *rows - 1) / *rows;
  };
  split(groups * (p.cols_pad / WG_COLS), 512, 1024, &p.rows, &p.S);
  const int64_t blocks = weigh_up(cols, WG_SUM_COLS) / WG_SUM_COLS;
  const int64_t per = (groups * blocks * T * (int64_t)sizeof(float) + (1 << 28) - 1) >> 28;
  p.wide = blocks == 2;
  p.per = p.wide ? 1 : (int)(per < blocks ? per : blocks);
  p.supers = p.wide ? 1 : (int)((blocks + p.per - 1) / p.per);
  split(groups * p.supers, p.wide ? 256 : 768, 0, &p.rows2, &p.S2);
  p.joined = p.S > 32;
  return p;
}
