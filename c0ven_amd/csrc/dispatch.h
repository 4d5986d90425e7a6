// Assignments sorted by expert, and the sums of their rows by token: what the dispatch's entry points and the experts share.
#pragma once

#include "../../include/c0ven_moe_tile.h"
#include "mx4.h"
#include "ops.h"

namespace c0ven {

// Where the sorted assignments go: order (A: position to assignment, -1 past the last), places (A: assignment to position, -1
// without one), offsets (E + 1) and, unless null, the MoeTiles of at most `rows` positions of an expert each, and their number.
struct SortOut {
  int32_t *order, *places;
  uint32_t *offsets;
  MoeTile *tiles;
  uint32_t *n_tiles, rows;
};
// Bytes of work the sort of A ids takes, and the sort, on the current device.
uint64_t sort_bytes(uint32_t A, uint32_t E);
void sort_launch(const int32_t *ids, uint32_t A, uint32_t E, const SortOut &out, void *work, void *stream);
// Its last launch alone: the slices' counts, if there are several, are in work.
void sort_place_launch(const int32_t *ids, uint32_t A, uint32_t E, const SortOut &out, void *work, void *stream);

// y[t] = sum over t's ranks of w o[place], in rank order in fp32, rounded once to y_type: `cols` values a row from y on, rows
// of o (of type, o_stride apart); a place outside 0 .. A - 1 adds nothing; w null: ones.
void combine_launch(uint32_t type, const void *o, uint64_t o_stride, uint32_t ntok, uint32_t K, uint32_t cols,
                    const int32_t *places, const float *w, uint32_t y_type, void *y, uint64_t y_stride, void *stream);

}  // namespace c0ven
