// tile_edge.h -- where the pieces of a tile's line are read when the line ends inside the tile.  For the fp32 tiles of
// linear.hip; nothing of HIP in here, so that a host program can hold every place against the matrix.
#pragma once

#ifndef EDGE_QUAL
#define EDGE_QUAL static inline
#endif

// A tile's line holds `left` (>= 1) values of the matrix, whose own lines are V values long at least.  The piece of V values at
// place c of the line is read from place at - back (below 0: in front of the tile, in the same line of the matrix) and then
// moved forward by back values, zeros behind them.  Pieces that lie wholly behind the end are the line's first one: their sums
// are not stored, but no value from outside the matrix may reach even those.
struct EdgePiece {
  int at, back;
};
EDGE_QUAL EdgePiece edge_piece(int c, int left, int V) {
  EdgePiece e;
  e.at = c < left ? c : 0;
  e.back = e.at + V > left ? e.at + V - left : 0;
  return e;
}
