// santa_paged.h -- what the planner (santa_paged_plan.cpp) and the kernels
// (santa_paged.hip, santa_rotary.hip) of the paged attention agree on.
#pragma once

#include "santa_amd.h"

namespace santa {
namespace paged {

constexpr int kTile = 64;        // tokens per tile
constexpr int kBlockRows = 256;  // rows per workgroup: 32 for each of its 8 waves

enum ItemFlags {
  kFromList = 1,  // tok0 indexes the plan's list of tokens; no row is before the item's end
  kDirect = 2,    // the item is all its rows attend to: it writes the output
  kTree = 4,      // what token i attends to from position tree0 on is in its record
  kTwoParts = 8   // in a plan of kByItem: its probabilities are in two parts
};

// How the probabilities of a plan's items enter the second product
// (santa_paged_plan_info.rounded).
enum Rounded { kNever = 0, kAlways = 1, kByItem = 2 };

// A token's record in a plan with trees: the context tokens that it attends to,
// its position (-1: not in use), and one bit for each position from the last
// multiple of 64 up to the context's end on: whether it attends to that token.
// Records of the plan's other tokens say the same (no bits beyond the context).
constexpr int kTreeWords = 2;  // where the bits begin
constexpr int kMostDrafts = 8192;

// What one workgroup per KV head does: rows r < rows, row r being query head
// r % GH of token tok0 + r / GH, over the tokens begin .. end - 1 (begin a
// multiple of the tile) of a block table row.  Token i attends to positions
// <= pos0 + i.  Workgroup w starts with item w; rows == 0: nothing to do.
struct Item {
  int flags, row, begin, end, tok0, rows, pos0;
  int base;  // record of row 0 at KV head 0; KV head h's are h * rows further
  int next;  // the workgroup's next item, or -1
  int tree0;
  int unused[6];
};
constexpr int kItemInts = 16;
static_assert(sizeof(Item) == kItemInts * sizeof(int), "packed");

// Strides in elements of a pool: pages, rows, heads.
struct PoolStrides {
  long long page, row, head;
};

struct Pages {
  const int* table;
  long long stride;  // entries per row
  int shift, num_pages;
};

// A block table, pools and plan that belong together.
int check_paged(const void* q, const void* k, const void* v, const void* out, int dtype, int num_pages, int page_size,
                const long long* strides, int n_strides, const int* table, long long table_stride, int table_rows,
                const santa_paged_plan_info* info, const int* plan, const char* what, Pages* pg);

}  // namespace paged
}  // namespace santa
