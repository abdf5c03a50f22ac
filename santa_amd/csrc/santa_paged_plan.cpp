// santa_paged_plan.cpp -- how the work of the paged attention
// (santa_paged.hip) is cut into workgroups.
#include <algorithm>
#include <climits>
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <exception>
#include <vector>

#include "santa_amd.h"
#include "santa_internal.h"
#include "santa_paged.h"

namespace santa {
namespace paged {
namespace {

// The kernel's 32-bit positions run past a sequence's end by up to 64 tiles.
constexpr int kMaxLen = 1 << 30;

// Rows (token, query head of one KV head) that pass over the same tokens
// together: those of the tokens tok0 .. tok0 + ntok - 1 of the batch, or of
// the list.
struct Block {
  int flags, row, begin, end, tok0, ntok, pos0;
  int tiles() const { return (end - begin + kTile - 1) / kTile; }
};

// What a tile costs a workgroup, by the rows of its block, and what a piece does
// besides (its first loads, its output), in units of about 0.25 us.  With 64 or
// fewer rows a tile takes as long as its 32 KiB do from HBM, with 256 as long as
// its products, a third more with probabilities in two parts.  All tiles alike and
// a piece like one: 122 us for 64 sequences behind 32k tokens and 232 for 32 behind
// 128k (113 and 219 with these, both rounded); in two parts 115 and 267, and with
// the costs of rounded ones 121 and 272.
constexpr int kPieceCost = 20;
int tile_cost(int rows, bool rounded) { return rows > 128 ? (rounded ? 10 : 13) : rows > 64 ? 7 : 6; }
// Whether a sequence's new tokens have the batch's probabilities rounded for the
// second product (santa_paged_plan_info.rounded, the default): several tokens, as
// in a prefill, whose second products would cost more than they do behind HBM.
// 8 sequences of 3000 to 16000 tokens, GH 4, D 128, rounded and in two parts: 8
// tokens (32 rows) 76.8 and 77.5 us, 9 77.6 and 84.2, 32 90.9 and 102.9; a prefill
// of 1300 tokens 313 and 410.  A single token is never rounded: what it attends to
// must not depend on how many others read the same pages.
bool rounds(int new_tokens, int GH) { return new_tokens > 1 && static_cast<long long>(new_tokens) * GH > 32; }
// The fewest tiles that a block is cut off after.
constexpr int kLeastCut = 2;

// Workgroups that are resident at once, one per compute unit (their LDS).
int resident() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  return cus;
}

struct Input {
  const int *lens, *new_tokens, *rows;
  int B;
  const int *group, *shared;
  int n_groups, heads, kv_heads, fixed;
};

int build(const Input& in, santa_paged_plan_info* info, int* plan, long long plan_ints) {
  const int GH = in.heads / in.kv_heads;
  const int block_tokens = std::max(1, kBlockRows / GH);
  *info = santa_paged_plan_info{};
  info->heads = in.heads;
  info->kv_heads = in.kv_heads;
  info->max_row = -1;
  long long tokens = 0;
  std::vector<int> first(static_cast<size_t>(in.B));       // first token of each sequence
  std::vector<int> prefix(static_cast<size_t>(in.B), 0);   // tokens read with the group
  std::vector<int> lead(static_cast<size_t>(in.n_groups), -1), members(static_cast<size_t>(in.n_groups), 0);
  for (int b = 0; b < in.B; ++b) {
    const int n = in.lens[b], t = in.new_tokens[b], row = in.rows ? in.rows[b] : b;
    if (n < 0 || t < 0) return set_error(SANTA_ERR_INVALID, "a sequence has 0 or more tokens and new tokens");
    if (row < 0) return set_error(SANTA_ERR_INVALID, "bad block table row %d", row);
    if (n > kMaxLen || t > kMaxLen)
      return set_error(SANTA_ERR_UNSUPPORTED, "the paged attention takes up to %d tokens per sequence. Got %d", kMaxLen,
                       std::max(n, t));
    first[b] = static_cast<int>(tokens);
    tokens += t;
    if (tokens > (1 << 26) / GH) return set_error(SANTA_ERR_INVALID, "too many new tokens");
    info->max_len = std::max(info->max_len, n);
    info->max_row = std::max(info->max_row, row);
    if (rounds(t, GH)) info->rounded = 1;
    const int g = in.group ? in.group[b] : -1;
    if (g < 0) continue;
    if (g >= in.n_groups) return set_error(SANTA_ERR_INVALID, "sequence %d names group %d of %d", b, g, in.n_groups);
    if (in.shared[g] < 0 || in.shared[g] > std::max(0, n - t))
      return set_error(SANTA_ERR_INVALID, "%d tokens are not common to sequence %d: %d precede its new tokens",
                       in.shared[g], b, std::max(0, n - t));
    if (t == 0 || static_cast<long long>(t) * GH >= kBlockRows) continue;  // fills workgroups by itself
    if (lead[g] < 0) lead[g] = row;
    ++members[g];
  }
  info->tokens = static_cast<int>(tokens);

  // the passes: whole tiles of each group's common tokens for all its rows, and
  // the rest of each sequence for its own
  std::vector<Block> blocks;
  std::vector<int> list;
  std::vector<int> token_pos(static_cast<size_t>(tokens)), token_row(static_cast<size_t>(tokens));
  std::vector<int> group_list(static_cast<size_t>(in.n_groups), 0);
  for (int g = 0; g < in.n_groups; ++g) {
    const int common = in.shared[g] / kTile * kTile;
    if (members[g] < 2 || common == 0) {
      members[g] = 0;
      continue;
    }
    group_list[g] = static_cast<int>(list.size());
    for (int b = 0; b < in.B; ++b)
      if (in.group[b] == g && static_cast<long long>(in.new_tokens[b]) * GH < kBlockRows) {
        prefix[b] = common;
        for (int i = 0; i < in.new_tokens[b]; ++i) list.push_back(first[b] + i);
      }
    const int n = static_cast<int>(list.size()) - group_list[g];
    for (int i = 0; i < n; i += block_tokens)
      blocks.push_back({kFromList, lead[g], 0, common, group_list[g] + i, std::min(block_tokens, n - i), kMaxLen});
  }
  for (int b = 0; b < in.B; ++b) {
    const int n = in.lens[b], t = in.new_tokens[b], row = in.rows ? in.rows[b] : b;
    for (int i = 0; i < t; ++i) {
      token_pos[first[b] + i] = n - t + i;
      token_row[first[b] + i] = row;
    }
    for (int i = 0; i < t; i += block_tokens) {
      const int k = std::min(block_tokens, t - i);
      const int end = std::max(prefix[b], std::min(n, n - t + i + k));
      blocks.push_back({0, row, prefix[b], end, first[b] + i, k, n - t + i});
    }
  }

  // one resident round of workgroups, each with a run of whole tiles of about
  // the same cost: the least with which they hold everything
  const int slots = std::max(1, resident() / in.kv_heads);
  struct Piece {
    int block, t0, t1, slot;
  };
  std::vector<Piece> pieces;
  auto pack = [&](long long budget, bool keep) {
    int slot = 0;
    long long left = budget;
    for (size_t i = 0; i < blocks.size(); ++i) {
      const int tiles = blocks[i].tiles(), cost = tile_cost(blocks[i].ntok * GH, info->rounded);
      for (int t = 0; t < tiles || t == 0;) {
        long long k = std::min<long long>(tiles - t, (left - kPieceCost) / cost);
        if (left < budget && (k < 1 ? tiles > 0 || left < kPieceCost : k < tiles - t && k < kLeastCut)) {
          if (++slot == slots) return false;
          left = budget;
          continue;
        }
        k = std::max<long long>(k, std::min(1, tiles));
        if (keep) pieces.push_back({static_cast<int>(i), t, t + static_cast<int>(k), slot});
        left -= kPieceCost + cost * k;
        t += std::max(1, static_cast<int>(k));
      }
    }
    return true;
  };
  long long total = 0;
  for (const Block& k : blocks) total += kPieceCost + static_cast<long long>(tile_cost(k.ntok * GH, info->rounded)) * k.tiles();
  long long lo = std::max<long long>(total / slots, kPieceCost + tile_cost(1, true) * kLeastCut), hi = lo;
  while (!pack(hi, false)) lo = hi + 1, hi += std::max(1LL, hi / 4);
  while (lo < hi) {
    const long long mid = lo + (hi - lo) / 2;
    if (pack(mid, false)) hi = mid;
    else lo = mid + 1;
  }
  pack(hi, true);
  const long long used = pieces.empty() ? 0 : pieces.back().slot + 1;
  const long long max_items = static_cast<long long>(blocks.size()) + slots;
  if (max_items > (1 << 26)) return set_error(SANTA_ERR_INVALID, "too many sequences");

  struct Parts {
    int base = 0, rows = 0, local = 0, splits = 0;
  };
  std::vector<Parts> common_parts(static_cast<size_t>(tokens)), own_parts(static_cast<size_t>(tokens));
  std::vector<int> base(pieces.size());
  std::vector<char> direct(pieces.size());
  long long records = 0, most_rows = 0;
  for (size_t i = 0; i < pieces.size();) {
    const Block& k = blocks[pieces[i].block];
    size_t end = i;
    while (end < pieces.size() && pieces[end].block == pieces[i].block) ++end;
    const int rows = k.ntok * GH;
    const bool from_list = (k.flags & kFromList) != 0;
    const bool whole = end - i == 1 && !from_list && k.begin == 0;
    most_rows = std::max<long long>(most_rows, rows);
    for (int j = 0; j < k.ntok && !whole; ++j)
      (from_list ? common_parts[list[k.tok0 + j]] : own_parts[k.tok0 + j]) = {static_cast<int>(records), rows, j * GH,
                                                                              static_cast<int>(end - i)};
    for (; i < end; ++i) {
      base[i] = static_cast<int>(records);
      direct[i] = whole;
      if (!whole) records += static_cast<long long>(rows) * in.kv_heads;
      if (records > INT_MAX) return set_error(SANTA_ERR_INVALID, "too many new tokens");
    }
  }

  info->groups = static_cast<int>(in.fixed ? slots : used);
  info->items = static_cast<int>(in.fixed ? max_items : static_cast<long long>(pieces.size()));
  info->records = in.fixed ? max_items * most_rows * in.kv_heads : records;
  if (info->records > INT_MAX) return set_error(SANTA_ERR_INVALID, "too many new tokens");
  std::vector<int> joined;
  for (long long t = 0; t < tokens; ++t)
    if (own_parts[t].splits > 0) joined.push_back(static_cast<int>(t));
  info->merge_tokens = in.fixed ? info->tokens : static_cast<int>(joined.size());
  info->pos_at = static_cast<long long>(info->items) * kItemInts;
  info->parts_at = info->pos_at + 2 * tokens + (tokens & 1) * 2;
  info->merge_at = info->parts_at + 8 * tokens;
  info->list_at = info->merge_at + info->merge_tokens;
  info->ints = info->list_at + static_cast<long long>(list.size());
  if (!plan) return clear_error();
  if (plan_ints < info->ints) return set_error(SANTA_ERR_INVALID, "the plan does not fit its buffer");

  std::memset(plan, 0, static_cast<size_t>(info->ints) * sizeof(int));
  for (int i = 0; i < info->items; ++i)
    plan[static_cast<size_t>(i) * kItemInts + offsetof(Item, next) / sizeof(int)] = -1;
  // a slot's first piece at the slot's number, the others behind them
  int more = static_cast<int>(used), last = -1;
  for (size_t i = 0; i < pieces.size(); ++i) {
    const Piece& p = pieces[i];
    const Block& k = blocks[p.block];
    Item it{};
    it.flags = k.flags | (direct[i] ? kDirect : 0);
    it.row = k.row;
    it.begin = k.begin + kTile * p.t0;
    it.end = std::min(k.end, k.begin + kTile * p.t1);
    it.tok0 = k.tok0;
    it.rows = k.ntok * GH;
    it.pos0 = k.pos0;
    it.base = base[i];
    it.next = -1;
    const bool first = i == 0 || pieces[i - 1].slot != p.slot;
    const int at = first ? p.slot : more++;
    if (!first) plan[static_cast<size_t>(last) * kItemInts + offsetof(Item, next) / sizeof(int)] = at;
    std::memcpy(plan + static_cast<size_t>(at) * kItemInts, &it, sizeof it);
    last = at;
  }
  int* pos = plan + info->pos_at;
  int* parts = plan + info->parts_at;
  for (long long t = 0; t < tokens; ++t) {
    pos[2 * t] = token_pos[t];
    pos[2 * t + 1] = token_row[t];
    const Parts &a = common_parts[t], &b = own_parts[t];
    const int v[8] = {a.base, a.rows, a.local, a.splits, b.base, b.rows, b.local, b.splits};
    std::memcpy(parts + 8 * t, v, sizeof v);
  }
  for (int t = 0; t < info->merge_tokens; ++t)
    plan[info->merge_at + t] = t < static_cast<int>(joined.size()) ? joined[t] : -1;
  std::copy(list.begin(), list.end(), plan + info->list_at);
  return clear_error();
}

}  // namespace
}  // namespace paged
}  // namespace santa

extern "C" int santa_paged_plan(const int* lens, const int* new_tokens, const int* rows, int B, const int* group,
                                const int* shared, int n_groups, int heads, int kv_heads, int fixed,
                                santa_paged_plan_info* info, int* plan, long long plan_ints) {
  using namespace santa;
  if (!info || B < 0 || (B > 0 && (!lens || !new_tokens)) || n_groups < 0 || (n_groups > 0 && (!group || !shared)))
    return set_error(SANTA_ERR_INVALID, "bad santa_paged_plan arguments");
  if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0)
    return set_error(SANTA_ERR_INVALID, "H must be divisible by KVH. Got H=%d KVH=%d", heads, kv_heads);
  if (heads > 1 << 16) return set_error(SANTA_ERR_UNSUPPORTED, "too many heads");
  if (heads / kv_heads > paged::kBlockRows)
    return set_error(SANTA_ERR_UNSUPPORTED, "the paged attention takes up to %d query heads per KV head. Got %d",
                     paged::kBlockRows, heads / kv_heads);
  try {
    return paged::build({lens, new_tokens, rows, B, n_groups > 0 ? group : nullptr, shared, n_groups, heads, kv_heads,
                         fixed},
                        info, plan, plan_ints);
  } catch (const std::exception&) {  // vectors that do not fit
    return set_error(SANTA_ERR_INVALID, "out of host memory");
  }
}
