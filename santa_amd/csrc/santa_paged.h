// santa_paged.h -- what the planner (santa_paged_plan.cpp) and the kernels
// (santa_paged.hip) of the paged attention agree on.
#pragma once

namespace santa {
namespace paged {

constexpr int kTile = 64;        // tokens per tile
constexpr int kBlockRows = 256;  // rows per workgroup: 32 for each of its 8 waves

enum ItemFlags {
  kFromList = 1,  // tok0 indexes the plan's list of tokens; no row is before the item's end
  kDirect = 2     // the item is all its rows attend to: it writes the output
};

// What one workgroup per KV head does: rows r < rows, row r being query head
// r % GH of token tok0 + r / GH, over the tokens begin .. end - 1 (begin a
// multiple of the tile) of a block table row.  Token i attends to positions
// <= pos0 + i.  Workgroup w starts with item w; rows == 0: nothing to do.
struct Item {
  int flags, row, begin, end, tok0, rows, pos0;
  int base;  // record of row 0 at KV head 0; KV head h's are h * rows further
  int next;  // the workgroup's next item, or -1
  int unused[7];
};
constexpr int kItemInts = 16;
static_assert(sizeof(Item) == kItemInts * sizeof(int), "packed");

}  // namespace paged
}  // namespace santa
