// How the rows of a paged attention are shared over workgroups.  The rules are the host's and the kernels' alike (constant
// expressions may be called from either).
#pragma once
#include <stdint.h>

#define PG_WAVES 8             // waves of an attending workgroup

// The rows of all groups, (sequence, key-value head) pairs in order, are one run of chunks of 16, of which workgroup i takes a
// share of `each`, whatever the lengths: places [i each, (i + 1) each).  A group that has rows begins with PG_LEAD places without
// any, about what its query, its merge and its part cost (a workgroup with a dozen short groups was what all others waited for).
// What workgroup i has of group g is part i + g: along the run either i or g moves on, so no two are the same.
#define PG_SHARE 8    // places of a share at least
#define PG_WORKGROUPS 512   // that share the rows at most: parts of a group
#define PG_LEAD 32

// Workgroups that share so many places: as many as run at a time, two to a compute unit, where that leaves each four chunks to a wave;
// below that one to a compute unit at most, of a chunk to a wave and more (one and a half to a unit, and some units have twice the others'
// work: 8 groups of 16384 rows in 264 of them 23.8 us, in 256 19.2).
static constexpr int pg_workgroups(int64_t places, int most) {
  return places >= 32 * PG_WORKGROUPS || most < PG_WORKGROUPS / 2 ? most : PG_WORKGROUPS / 2;
}
// Places of a workgroup's share of a run of `total`, with `most` workgroups there.
static constexpr int64_t pg_each(int64_t total, int most) {
  const int64_t share = (total + pg_workgroups(total, most) - 1) / pg_workgroups(total, most);
  return share < PG_SHARE ? PG_SHARE : share;
}

// Workgroups that share the rows of up to max_len.  None, one to each group, where that leaves no unit empty that a split would fill:
// no shares to find, nothing to join, but the longest group sets the time, so up to 512 rows, and of many groups up to 2048.  Groups of four heads, us,
// equal lengths | random ones | one long sequence among short ones; shared, then one to each group:
//   8 x 513: 10.3; 8.6     8 x 1024: 10.2; 12.8     128 x 1024: 20.2 | 15.8 | 11.7; 16.1 | 15.0 | 12.9     256 x 2048: 55 | 34 | 18; 44 | 29 | 24
//   512 x 2048: 100 | 61 | 20; 84 | 59 | 25     64 x 1024: 14.4 | 12.4 | 10.5; 15.4 | 14.3 | 12.9     256 x 4096: 93 | 57 | 20; 83 | 58 | 43
// With scores the join is launched anyway, and the gain halves (256 x 1024 29.3 | 22.1 | 15.3; 28.3 | 21.0 | 17.0); the rule is the same,
// so that an output does not depend on whether scores are asked for.
static inline int paged_workgroups(int64_t groups, int max_len) {
  if (max_len <= 512 || (max_len <= 2048 && max_len <= groups * 6)) return 0;
  const int64_t places = groups * ((max_len + 15) / 16 + 1 + PG_LEAD), shares = (places + PG_SHARE - 1) / PG_SHARE;
  return pg_workgroups(places, shares < PG_WORKGROUPS ? (int)shares : PG_WORKGROUPS);
}
