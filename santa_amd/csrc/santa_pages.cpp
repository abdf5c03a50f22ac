// santa_pages.cpp -- host bookkeeping of a paged KV cache: which pages each
// sequence holds, how many sequences hold a page, and which pages are free.
// No counterpart in the reference, whose caches are contiguous
// (tutorial_code/runtime_common.py:340-397).
//
// The bookkeeping is exact and on the host, so that a request that does not
// fit fails in the call that makes it, with nothing changed; what it asks of the
// device (page copies, edits of the block table) is left in lists that
// santa_pages_apply turns into kernel launches.
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <exception>
#include <new>
#include <vector>

#include "santa_amd.h"
#include "santa_internal.h"

struct santa_pages {
  struct Seq {
    int len = -1;  // -1: the row is free
    std::vector<int> pages;
  };
  int page_size = 0, row_pages = 0;
  std::vector<int> refs;        // sequences holding each page
  std::vector<uint64_t> open;   // bit p: page p is free
  size_t hint = 0;              // no word of `open` below this one has a bit set
  int used = 0;
  std::vector<Seq> seqs;
  std::vector<char> mark;       // scratch: one per sequence, all 0 between calls
  // what the last operation asks of the device
  std::vector<santa::PageCopy> copies;
  std::vector<santa::TableEdit> edits;
  bool remap = false;

  int num_pages() const { return static_cast<int>(refs.size()); }
  int pages_for(int tokens) const {
    return static_cast<int>((static_cast<int64_t>(tokens) + page_size - 1) / page_size);
  }
  // The free page of the lowest number (there is one).
  int take() {
    while (!open[hint]) ++hint;
    const int p = static_cast<int>(hint * 64) + __builtin_ctzll(open[hint]);
    open[hint] &= open[hint] - 1;
    refs[p] = 1;
    ++used;
    return p;
  }
  void drop(int p, int n = 1) {
    if ((refs[p] -= n) > 0) return;
    open[p >> 6] |= 1ull << (p & 63);
    hint = std::min(hint, static_cast<size_t>(p >> 6));
    --used;
  }
  // Entry `col` of a row is now `page`: part of the last edit where it continues it.
  void edit(int row, int col, int page) {
    if (!edits.empty()) {
      santa::TableEdit& e = edits.back();
      if (e.row == row && e.value >= 0 && e.col + e.count == col && e.value + e.count == page) {
        ++e.count;
        return;
      }
    }
    edits.push_back({row, col, 1, page});
  }
  void begin() {
    copies.clear();
    edits.clear();
    remap = false;
  }
  bool alive(int s) const { return s >= 0 && s < static_cast<int>(seqs.size()) && seqs[s].len >= 0; }
};

namespace {
using santa::set_error;
using santa::clear_error;

// How many of the first n pages of two rows are the same (memcmp passes over
// them several times as fast as a loop).
size_t common_pages(const std::vector<int>& a, const std::vector<int>& b, size_t n) {
  constexpr size_t kBlock = 256;
  size_t i = 0;
  while (i + kBlock <= n && std::memcmp(a.data() + i, b.data() + i, kBlock * sizeof(int)) == 0) i += kBlock;
  while (i < n && a[i] == b[i]) ++i;
  return i;
}

// Runs f; an allocation that fails becomes an error code.
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::exception&) {
    return set_error(SANTA_ERR_INVALID, "out of host memory");
  }
}

// Checks that seqs names sequences in use, each once.
int check_seqs(santa_pages* p, const int* seqs, int n) {
  if (n < 0 || (n > 0 && !seqs)) return set_error(SANTA_ERR_INVALID, "bad list of sequences");
  int rc = SANTA_OK, i = 0;
  for (; i < n && rc == SANTA_OK; ++i) {
    if (!p->alive(seqs[i])) {
      rc = set_error(SANTA_ERR_INVALID, "no sequence %d in the cache", seqs[i]);
      break;
    }
    if (p->mark[seqs[i]]) rc = set_error(SANTA_ERR_INVALID, "sequence %d is named twice", seqs[i]);
    p->mark[seqs[i]] = 1;
  }
  for (int j = 0; j < i; ++j) p->mark[seqs[j]] = 0;
  return rc;
}

// Lengthens the sequences, whose rows exist; all or nothing.
int extend(santa_pages* p, const int* seqs, const int* tokens, int n) {
  int64_t need = 0;
  int rc = SANTA_OK, i = 0;
  std::vector<int> dropped;  // shared last pages given up so far
  dropped.reserve(static_cast<size_t>(n));
  for (; i < n; ++i) {
    const santa_pages::Seq& s = p->seqs[seqs[i]];
    if (tokens[i] < 0) {
      rc = set_error(SANTA_ERR_INVALID, "a sequence grows by at least 0 tokens; got %d", tokens[i]);
      break;
    }
    const int64_t len = static_cast<int64_t>(s.len) + tokens[i];
    if (len > static_cast<int64_t>(p->row_pages) * p->page_size) {
      rc = set_error(SANTA_ERR_INVALID, "sequence %d would hold %lld tokens; the block table has room for %lld",
                     seqs[i], static_cast<long long>(len), static_cast<long long>(p->row_pages) * p->page_size);
      break;
    }
    need += p->pages_for(static_cast<int>(len)) - static_cast<int>(s.pages.size());
    if (tokens[i] > 0 && s.len % p->page_size != 0 && p->refs[s.pages.back()] > 1) {
      --p->refs[s.pages.back()];
      dropped.push_back(i);
      ++need;
    }
  }
  if (rc == SANTA_OK && need > p->num_pages() - p->used)
    rc = set_error(SANTA_ERR_INVALID, "out of pages: %lld needed, %d free", static_cast<long long>(need),
                   p->num_pages() - p->used);
  if (rc == SANTA_OK) {  // everything that can throw, before anything changes
    try {
      p->edits.reserve(static_cast<size_t>(need));
      p->copies.reserve(dropped.size());
      for (int j = 0; j < n; ++j) {
        std::vector<int>& pages = p->seqs[seqs[j]].pages;
        const size_t want = static_cast<size_t>(p->pages_for(p->seqs[seqs[j]].len + tokens[j]));
        // twice as many as there were, or a sequence that grows by single pages copies its list each time
        if (want > pages.capacity()) pages.reserve(std::max(want, 2 * pages.capacity()));
      }
    } catch (const std::bad_alloc&) {
      rc = set_error(SANTA_ERR_INVALID, "out of host memory");
    }
  }
  if (rc != SANTA_OK) {
    for (const int j : dropped) ++p->refs[p->seqs[seqs[j]].pages.back()];
    return rc;
  }
  size_t d = 0;
  for (int j = 0; j < n; ++j) {
    santa_pages::Seq& s = p->seqs[seqs[j]];
    if (d < dropped.size() && dropped[d] == j) {
      ++d;
      const int to = p->take();
      p->copies.push_back({s.pages.back(), to});
      s.pages.back() = to;
      p->edit(seqs[j], static_cast<int>(s.pages.size()) - 1, to);
    }
    s.len += tokens[j];
    const size_t pages = static_cast<size_t>(p->pages_for(s.len));
    while (s.pages.size() < pages) {
      const int to = p->take();
      p->edit(seqs[j], static_cast<int>(s.pages.size()), to);
      s.pages.push_back(to);
    }
  }
  return SANTA_OK;
}

// The n free rows of the lowest numbers, as empty sequences.
int new_rows(santa_pages* p, int n, int* out) {
  int got = 0;
  for (size_t s = 0; s < p->seqs.size() && got < n; ++s)
    if (p->seqs[s].len < 0) out[got++] = static_cast<int>(s);
  if (got < n)
    return set_error(SANTA_ERR_INVALID, "out of sequences: %d wanted, %d of %d free", n, got,
                     static_cast<int>(p->seqs.size()));
  for (int i = 0; i < n; ++i) p->seqs[out[i]].len = 0;
  return SANTA_OK;
}
void drop_rows(santa_pages* p, const int* rows, int n) {
  for (int i = 0; i < n; ++i) p->seqs[rows[i]].len = -1;
}
}  // namespace

extern "C" int santa_pages_create(int num_pages, int page_size, int max_seqs, int row_pages, santa_pages** out) {
  if (!out) return set_error(SANTA_ERR_INVALID, "null pointer argument");
  *out = nullptr;
  const int rc = santa::check_page_size(page_size);
  if (rc != SANTA_OK) return rc;
  if (num_pages <= 0 || max_seqs <= 0 || row_pages <= 0)
    return set_error(SANTA_ERR_INVALID, "a cache needs pages, sequences and room in its block table");
  if (static_cast<int64_t>(row_pages) * page_size > INT32_MAX)
    return set_error(SANTA_ERR_INVALID, "a sequence's pages hold at most 2^31 - 1 tokens");
  return guarded([&] {
    santa_pages* p = new santa_pages;
    try {
      p->page_size = page_size;
      p->row_pages = row_pages;
      p->refs.assign(static_cast<size_t>(num_pages), 0);
      p->open.assign((static_cast<size_t>(num_pages) + 63) / 64, ~0ull);
      if (num_pages % 64) p->open.back() = (1ull << (num_pages % 64)) - 1;
      p->seqs.resize(static_cast<size_t>(max_seqs));
      p->mark.assign(static_cast<size_t>(max_seqs), 0);
    } catch (...) {
      delete p;
      throw;
    }
    *out = p;
    return clear_error();
  });
}

extern "C" void santa_pages_destroy(santa_pages* p) { delete p; }

extern "C" int santa_pages_add(santa_pages* p, const int* lengths, int n, int* seqs) {
  if (!p || n < 0 || (n > 0 && (!lengths || !seqs)))
    return set_error(SANTA_ERR_INVALID, "bad santa_pages_add arguments");
  return guarded([&] {
    p->begin();
    int rc = new_rows(p, n, seqs);
    if (rc != SANTA_OK) return rc;
    try {
      rc = extend(p, seqs, lengths, n);
    } catch (...) {
      drop_rows(p, seqs, n);
      throw;
    }
    if (rc != SANTA_OK) {
      drop_rows(p, seqs, n);
      return rc;
    }
    return clear_error();
  });
}

extern "C" int santa_pages_extend(santa_pages* p, const int* seqs, const int* tokens, int n) {
  if (!p || (n > 0 && !tokens)) return set_error(SANTA_ERR_INVALID, "bad santa_pages_extend arguments");
  return guarded([&] {
    p->begin();
    int rc = check_seqs(p, seqs, n);
    if (rc == SANTA_OK) rc = extend(p, seqs, tokens, n);
    return rc == SANTA_OK ? clear_error() : rc;
  });
}

extern "C" int santa_pages_shrink(santa_pages* p, const int* seqs, const int* tokens, int n) {
  if (!p || (n > 0 && !tokens)) return set_error(SANTA_ERR_INVALID, "bad santa_pages_shrink arguments");
  p->begin();
  const int rc = check_seqs(p, seqs, n);
  if (rc != SANTA_OK) return rc;
  for (int i = 0; i < n; ++i)
    if (tokens[i] < 0 || tokens[i] > p->seqs[seqs[i]].len)
      return set_error(SANTA_ERR_INVALID, "%d tokens cannot leave sequence %d, which holds %d", tokens[i], seqs[i],
                       p->seqs[seqs[i]].len);
  for (int i = 0; i < n; ++i) {
    santa_pages::Seq& s = p->seqs[seqs[i]];
    s.len -= tokens[i];
    for (const size_t pages = static_cast<size_t>(p->pages_for(s.len)); s.pages.size() > pages; s.pages.pop_back())
      p->drop(s.pages.back());
  }
  return clear_error();
}

extern "C" int santa_pages_fork(santa_pages* p, int seq, int n, int* seqs) {
  if (!p || n < 0 || (n > 0 && !seqs)) return set_error(SANTA_ERR_INVALID, "bad santa_pages_fork arguments");
  return guarded([&] {
    p->begin();
    if (!p->alive(seq)) return set_error(SANTA_ERR_INVALID, "no sequence %d in the cache", seq);
    const santa_pages::Seq& from = p->seqs[seq];
    const int rc = new_rows(p, n, seqs);
    if (rc != SANTA_OK) return rc;
    try {
      p->edits.reserve(static_cast<size_t>(n));
      for (int i = 0; i < n; ++i) p->seqs[seqs[i]].pages = from.pages;
    } catch (...) {
      for (int i = 0; i < n; ++i) p->seqs[seqs[i]].pages.clear();
      drop_rows(p, seqs, n);
      throw;
    }
    for (int i = 0; i < n; ++i) {
      p->seqs[seqs[i]].len = from.len;
      if (!from.pages.empty()) p->edits.push_back({seqs[i], 0, static_cast<int>(from.pages.size()), -1 - seq});
    }
    for (const int page : from.pages) p->refs[page] += n;
    return clear_error();
  });
}

extern "C" int santa_pages_free(santa_pages* p, const int* seqs, int n) {
  if (!p) return set_error(SANTA_ERR_INVALID, "bad santa_pages_free arguments");
  p->begin();
  const int rc = check_seqs(p, seqs, n);
  if (rc != SANTA_OK) return rc;
  // Forks of one sequence mostly follow one another here.  The pages that a run
  // of them has in common are given up once for all (64 forks of 2048 pages: 47
  // us page by page, most of the call's time; comparing the rows takes 6).
  for (int i = 0; i < n;) {
    const std::vector<int>& lead = p->seqs[seqs[i]].pages;
    size_t common = lead.size();
    int j = i + 1;
    for (; j < n; ++j) {
      const std::vector<int>& row = p->seqs[seqs[j]].pages;
      const size_t c = common_pages(lead, row, std::min(common, row.size()));
      if (2 * c < lead.size()) break;
      common = c;
    }
    for (size_t k = 0; k < common; ++k) p->drop(lead[k], j - i);
    for (int m = i; m < j; ++m) {
      santa_pages::Seq& s = p->seqs[seqs[m]];
      for (size_t k = common; k < s.pages.size(); ++k) p->drop(s.pages[k]);
      s.len = -1;
    }
    for (; i < j; ++i) p->seqs[seqs[i]].pages.clear();
  }
  return clear_error();
}

extern "C" int santa_pages_compact(santa_pages* p) {
  if (!p) return set_error(SANTA_ERR_INVALID, "bad santa_pages_compact arguments");
  return guarded([&] {
    p->begin();
    const int n = p->used;
    std::vector<int> to(static_cast<size_t>(p->num_pages() - n));  // of page n + i
    int hole = 0;
    for (int page = n; page < p->num_pages(); ++page) {
      if (p->refs[page] == 0) continue;
      while (p->refs[hole] != 0) ++hole;
      to[page - n] = hole;
      p->copies.push_back({page, hole++});  // throws before anything has changed
    }
    for (const santa::PageCopy& c : p->copies) {
      p->refs[c.dst] = p->refs[c.src];
      p->refs[c.src] = 0;
      p->open[c.dst >> 6] &= ~(1ull << (c.dst & 63));
      p->open[c.src >> 6] |= 1ull << (c.src & 63);
    }
    p->hint = static_cast<size_t>(n >> 6) < p->open.size() ? static_cast<size_t>(n >> 6) : 0;
    for (santa_pages::Seq& s : p->seqs)
      for (int& page : s.pages)
        if (page >= n) page = to[page - n];
    p->remap = !p->copies.empty();
    return clear_error();
  });
}

extern "C" int santa_pages_length(const santa_pages* p, int seq) { return p && p->alive(seq) ? p->seqs[seq].len : -1; }

extern "C" int santa_pages_used(const santa_pages* p) { return p ? p->used : -1; }

extern "C" int santa_pages_row(const santa_pages* p, int seq, const int** pages) {
  if (!p || !pages || !p->alive(seq)) return -1;
  *pages = p->seqs[seq].pages.data();
  return static_cast<int>(p->seqs[seq].pages.size());
}

extern "C" int santa_pages_changes(const santa_pages* p, const int** copies, int* n_copies, const int** edits,
                                   int* n_edits, int* remap) {
  static_assert(sizeof(santa::PageCopy) == 2 * sizeof(int) && sizeof(santa::TableEdit) == 4 * sizeof(int), "packed");
  if (!p || !copies || !n_copies || !edits || !n_edits || !remap)
    return set_error(SANTA_ERR_INVALID, "null pointer argument");
  *copies = reinterpret_cast<const int*>(p->copies.data());
  *n_copies = static_cast<int>(p->copies.size());
  *edits = reinterpret_cast<const int*>(p->edits.data());
  *n_edits = static_cast<int>(p->edits.size());
  *remap = p->remap ? 1 : 0;
  return clear_error();
}

// Tokens that the sequences have in common from the start on, found in their
// pages: out[i] names the group of sequence i (-1: none), group g being
// shared[g] tokens (whole pages) long.  Sequences are grouped by their first
// page; a group whose members part at different pages keeps the length that
// saves the most reading, and the members that part earlier look for a group
// among themselves.
extern "C" int santa_pages_shared(const santa_pages* p, const int* seqs, const int* own, int n, int* group, int* shared,
                                  int* n_groups) {
  if (!p || n < 0 || (n > 0 && (!seqs || !own || !group || !shared)) || !n_groups)
    return set_error(SANTA_ERR_INVALID, "bad santa_pages_shared arguments");
  return guarded([&] {
    for (int i = 0; i < n; ++i) {
      if (!p->alive(seqs[i])) return set_error(SANTA_ERR_INVALID, "no sequence %d in the cache", seqs[i]);
      if (own[i] < 0) return set_error(SANTA_ERR_INVALID, "a sequence has 0 or more new tokens; got %d", own[i]);
    }
    *n_groups = 0;
    // whole pages before the sequence's own tokens
    std::vector<int> limit(static_cast<size_t>(n)), common(static_cast<size_t>(n));
    std::vector<std::pair<int, int>> order;  // (first page, index)
    order.reserve(static_cast<size_t>(n));
    for (int i = 0; i < n; ++i) {
      group[i] = -1;
      limit[i] = std::max(0, p->seqs[seqs[i]].len - own[i]) / p->page_size;
      if (limit[i] > 0) order.emplace_back(p->seqs[seqs[i]].pages[0], i);
    }
    std::sort(order.begin(), order.end());
    std::vector<int> members, rest, lengths;
    for (size_t a = 0; a < order.size();) {
      size_t b = a;
      members.clear();
      while (b < order.size() && order[b].first == order[a].first) members.push_back(order[b++].second);
      a = b;
      while (members.size() > 1) {
        // pages in common with the member that has the most of them
        int lead = members[0];
        for (const int m : members)
          if (limit[m] > limit[lead]) lead = m;
        const std::vector<int>& row = p->seqs[seqs[lead]].pages;
        lengths.clear();
        for (const int m : members) {
          const std::vector<int>& other = p->seqs[seqs[m]].pages;
          common[m] = static_cast<int>(common_pages(row, other, static_cast<size_t>(std::min(limit[m], limit[lead]))));
          lengths.push_back(common[m]);
        }
        std::sort(lengths.begin(), lengths.end());
        int64_t best = 0;
        int pages = 0;
        for (size_t i = 0; i + 1 < lengths.size(); ++i) {
          const int64_t saved = static_cast<int64_t>(lengths.size() - 1 - i) * lengths[i];
          if (saved > best) best = saved, pages = lengths[i];
        }
        rest.clear();
        const int g = pages > 0 ? (*n_groups)++ : -1;
        if (g >= 0) shared[g] = pages * p->page_size;
        for (const int m : members) {
          if (g >= 0 && common[m] >= pages) group[m] = g;
          else if (m != lead) rest.push_back(m);  // shares nothing with the lead: a group without it
        }
        members.swap(rest);
      }
    }
    return clear_error();
  });
}
