// Layout of a row grouping (flm_group_rows) and the pieces the adapter kernels share.
#pragma once
#include "flm_common.h"

namespace flm {

// Sorted rows are taken in tiles of this many, each inside one group.
#define FLM_ROW_TILE 32

// The int32 buffer of a grouping of n rows into E groups:
//   order [n]      row numbers, stably sorted by group, rows without a group last
//   key [n]        the group of order[i], E for none
//   offsets [E+1]  first position of each group; offsets[E] = rows that have one
//   first_tile [E+1]  first tile of each group; first_tile[E] = number of tiles
//   tiles [2*cap]  (first position, group | rows << 16) of every tile, rows = 0 behind the last
struct RowGroups {
  const int *order, *key, *offsets, *first_tile;
  const int2* tiles;
  int cap;
};

inline long row_tiles_cap(long n, long E) { return (n + FLM_ROW_TILE - 1) / FLM_ROW_TILE + (n < E ? n : E); }
inline long row_groups_pad(long n) { return (n + 3) & ~3L; }
inline long row_groups_ints(long n, long E) {
  return 2 * row_groups_pad(n) + 2 * row_groups_pad(E + 1) + 2 * row_tiles_cap(n, E);
}
inline RowGroups row_groups(const int32_t* buf, long n, long E) {
  RowGroups g;
  g.order = buf;
  g.key = buf + row_groups_pad(n);
  g.offsets = g.key + row_groups_pad(n);
  g.first_tile = g.offsets + row_groups_pad(E + 1);
  g.tiles = reinterpret_cast<const int2*>(g.first_tile + row_groups_pad(E + 1));
  g.cap = (int)row_tiles_cap(n, E);
  return g;
}

}  // namespace flm
