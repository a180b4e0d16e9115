// The paged kernels' integer arithmetic (ramvamp_amd/csrc/rv_pages.hpp) on the
// host: how a batch's units are dealt, where a row lies, and what is refused.
// Prints nothing and exits 0 when all holds; else names what does not.
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <random>
#include <vector>

#include "../ramvamp_amd/csrc/rv_pages.hpp"

#define CHECK(c, ...)               \
  do {                              \
    if (!(c)) {                     \
      printf("%s: ", #c);           \
      printf(__VA_ARGS__);          \
      printf("\n");                 \
      exit(1);                      \
    }                               \
  } while (0)

using namespace rv;

// Every unit is visited once, a range keeps at most one piece in each of its two
// partials, and the join finds an item's pieces where they were kept.
static void deal(const std::vector<long>& rows, long items, long ranges) {
  std::vector<long> before(rows.size() + 1, 0);
  for (size_t s = 0; s < rows.size(); ++s) before[s + 1] = before[s] + units_of(rows[s]) * items;
  const long total = before.back(), per = std::max((total + ranges - 1) / ranges, 1l);
  CHECK(per * ranges >= total, "units left over");
  std::vector<int> seen(total, 0);
  std::map<std::pair<long, int>, std::pair<size_t, long>> kept;  // (range, partial) -> (sequence, item)
  for (long r = 0; r < ranges; ++r) {
    const long start = r * per, end = std::min(total, start + per);
    if (start >= end) continue;
    size_t s = 0;
    while (!(start >= before[s] && start < before[s + 1])) ++s;
    walk_units((uint32_t)s, start - before[s], start, end, items, [&](uint32_t i) { return rows[i]; },
               [&](uint32_t i) {
                 while (units_of(rows[i]) == 0) ++i;
                 return i;
               },
               [&](uint32_t i, long n, long item, long u0, long u1, long at) {
                 CHECK(n == rows[i] && item >= 0 && item < items, "sequence %u item %ld", i, item);
                 CHECK(u0 < u1 && u1 <= units_of(n), "units %ld..%ld", u0, u1);
                 CHECK(at == before[i] + item * units_of(n) + u0, "unit %ld", at);
                 for (long u = u0; u < u1; ++u) ++seen[at + u - u0];
                 const bool whole = u0 == 0 && u1 == units_of(n);
                 if (whole) return;
                 const auto key = std::make_pair(r, partial_of(r, per, at));
                 CHECK(!kept.count(key), "range %ld keeps two pieces in partial %d", r, key.second);
                 kept[key] = {i, item};
               });
  }
  for (long u = 0; u < total; ++u) CHECK(seen[u] == 1, "unit %ld visited %d times", u, seen[u]);
  size_t joined = 0;
  for (size_t s = 0; s < rows.size(); ++s)
    for (long item = 0; item < items && units_of(rows[s]); ++item) {
      const long start = before[s] + item * units_of(rows[s]), end = start + units_of(rows[s]);
      const long w0 = start / per, w1 = (end - 1) / per;
      if (w0 == w1) continue;
      for (long i = w0; i <= w1; ++i) {
        const auto it = kept.find({i, partial_of(i, per, start)});
        CHECK(it != kept.end() && it->second == std::make_pair(s, item), "range %ld of sequence %zu", i, s);
        ++joined;
      }
    }
  CHECK(joined == kept.size(), "%zu pieces of %zu joined", joined, kept.size());
}

// The joins within and across groups: every piece is kept where its group's last
// workgroup, or the item's, looks for it, and no place is used twice.
static void join_groups(const std::vector<uint32_t>& units, int log_slots, int most, int few) {
  uint32_t total = 0;
  for (uint32_t u : units) total += u;
  const Cut cut = cut_units(total, most, few, log_slots);
  const uint32_t slots = 1u << log_slots, per = cut.per, in_slot = cut.in_slot, ranges = slots * in_slot;
  CHECK(ranges <= std::max(1u << most, slots), "%u ranges", ranges);
  CHECK((uint64_t)per * ranges >= total, "units left over");
  std::vector<int> dealt(ranges, 0);
  for (uint32_t b = 0; b < ranges; ++b) {
    const uint32_t r = range_of(b, log_slots, in_slot);
    CHECK(r < ranges && r / in_slot == b % slots && slot_of(b, log_slots) == b % slots, "workgroup %u", b);
    const Group g = group_of(r, b % slots, in_slot);
    CHECK(g.lo <= r && r <= g.hi && g.hi - g.lo < kGroup && g.hi / in_slot == b % slots, "group of %u", r);
    CHECK(r == 0 || g.id == group_of(r - 1, (r - 1) / in_slot, in_slot).id + (r == g.lo ? 1 : 0), "number of %u's", r);
    ++dealt[r];
  }
  for (int d : dealt) CHECK(d == 1, "a range dealt %d times", d);
  std::map<uint32_t, int> pieces_at, groups_at;  // partial -> item
  uint32_t first = 0;
  for (size_t item = 0; item < units.size(); first += units[item++]) {
    const uint32_t w0 = first / per, w1 = (first + units[item] - 1) / per;
    if (!units[item] || w0 == w1) continue;
    uint32_t seen = 0, seen_groups = 0, group0 = 0;
    for (uint32_t r = w0; r <= w1; ++r) {
      const Group g = group_of(r, r / in_slot, in_slot);
      const Pieces p = pieces_of(g, w0, w1, first, per, in_slot);
      CHECK(p.first <= r && r < p.first + p.count && p.count <= kGroup && p.w0 == w0 && p.all == w1 - w0 + 1, "range %u", r);
      const uint32_t at = std::max(first, r * per), mine = 2 * r + partial_of(r, per, at);
      const uint32_t of_group = group_partial(g, first, per);
      // Where the group's join, and one of all pieces, look for this piece.
      const uint32_t looked = r == p.first ? 2 * p.first + partial_of(p.first, per, first)
                                           : 2 * (p.first + 1) + 2 * (r - p.first - 1);
      const uint32_t flat = r == w0 ? 2 * w0 + partial_of(w0, per, first) : 2 * (w0 + 1) + 2 * (r - w0 - 1);
      CHECK(looked == mine && flat == mine, "range %u's piece", r);
      CHECK(!pieces_at.count(mine), "partial %u twice", mine);
      pieces_at[mine] = (int)item;
      if (r == w0) group0 = of_group;
      CHECK(p.group0 == group0, "first group");
      if (r == p.first) {
        if (p.groups > 1) {
          CHECK(of_group == (seen_groups ? (group0 & ~1u) + 2 + 2 * (seen_groups - 1) : group0), "group %u", g.id);
          CHECK(of_group < 2 * 32 && !groups_at.count(of_group), "group partial %u twice", of_group);
          groups_at[of_group] = (int)item;
        }
        ++seen_groups;
        seen += p.count;
      }
    }
    const Pieces p = pieces_of(group_of(w0, w0 / in_slot, in_slot), w0, w1, first, per, in_slot);
    CHECK(seen == p.all && seen_groups == p.groups, "%u pieces, %u groups", seen, seen_groups);
  }
}

int main() {
  std::mt19937 g(7);
  for (int i = 0; i < 4000; ++i) {
    std::vector<uint32_t> units(1 + g() % 60);
    const uint32_t most = 1 + (i % 2 ? g() % 40 : g() % 2000);
    for (auto& u : units) u = g() % (most + 1);
    if (i % 7 == 0) units.resize(1);
    const int slots = i % 5 ? 3 : 0, cut = slots + (int)(g() % 7);
    join_groups(units, slots, cut, cut && i % 3 ? cut - 1 : cut);
  }
  // Quotients by a reciprocal two steps off either way.
  for (int i = 0; i < 2000000; ++i) {
    const uint32_t y = 1 + (g() >> (g() % 32)), q = g() % (1u << (g() % 21));
    const uint64_t x = (uint64_t)q * y + (i % 3 == 0 ? 0 : i % 3 == 1 ? y - 1 : g() % y);
    if (x >= 0x80000000u || y >= 0x80000000u) continue;
    const float rcp = (float)(1.0 / y) * (1.f + ((int)(g() % 5) - 2) * 5.96e-8f);
    CHECK(quotient((uint32_t)x, y, rcp) == q, "%u / %u", (uint32_t)x, y);
  }
  deal({1}, 1, 512);
  deal({0, 0, 0}, 4, 512);
  deal({131000}, 4, 512);
  deal(std::vector<long>(700, 129), 4, 512);
  for (int i = 0; i < 3000; ++i) {
    std::vector<long> rows(1 + g() % 70);
    const long most = 1 + (long)(g() % (i % 3 == 0 ? 300 : i % 3 == 1 ? 4000 : 60000));
    for (auto& n : rows) n = g() % 5 == 0 ? 0 : (long)(g() % (most + 1)) - (g() % 9 == 0);  // (-1: refused)
    deal(rows, 1 + g() % 9, 1 + g() % 2048);
  }

  // Lengths that shrink under the walk: it ends.
  int visits = 0;
  walk_units(0u, 0l, 0l, 10l, 1l, [](uint32_t) { return 100l; },
             [](uint32_t s) { return s < 3 ? s : kNoMore; }, [&](uint32_t, long, long, long, long, long) { ++visits; });
  CHECK(visits == 3, "%d visits", visits);

  const int32_t ids[3 * 5] = {4, 0, -1, 9, 9, 7, 6, 5, 9, 9, 8, INT32_MIN, INT32_MAX, 9, 9};  // 3 of 5 entries a row
  const Pages t{ids, 5, 3, 3, 9, 4};
  uint32_t page = 99, row = 99, got = 99;
  CHECK(place_of(t, 0, 0, page, row, got) == kHere && page == 4 && row == 0, "first row");
  CHECK(place_of(t, 31, 0, page, row, got) == kHere && page == 0 && row == 15, "last row of a page");
  CHECK(place_of(t, 47, 1, page, row, got) == kHere && page == 5 && row == 15, "last row of a table row");
  CHECK(place_of(t, -1, 77, page, row, got) == kPadding, "padding comes first");
  CHECK(place_of(t, INT32_MIN, 0, page, row, got) == kPadding, "any negative position");
  CHECK(place_of(t, 48, 0, page, row, got) == kNoPosition && got == 48, "past the table row");
  CHECK(place_of(t, INT32_MAX, 2, page, row, got) == kNoPosition, "far past it");
  CHECK(place_of(t, 0, 3, page, row, got) == kNoSequence && got == 3, "past the table");
  CHECK(place_of(t, 0, -1, page, row, got) == kNoSequence, "a negative sequence");
  CHECK(place_of(t, 32, 0, page, row, got) == kNoPage && got == 0xFFFFFFFFu, "page -1");
  CHECK(place_of(t, 16, 2, page, row, got) == kNoPage, "page INT32_MIN");
  CHECK(place_of(t, 32, 2, page, row, got) == kNoPage, "page INT32_MAX");
  const Pages none{nullptr, 0, 2, 0, 9, 4};
  CHECK(place_of(none, 0, 1, page, row, got) == kNoPosition, "a table of no pages");

  CHECK(table_rows(t) == 48, "rows of a table row");
  CHECK(attended_rows(t, 48, false) == 48 && attended_rows(t, 49, false) == -1, "the longest");
  CHECK(attended_rows(t, -1, false) == -1 && attended_rows(t, 0, false) == 0, "lengths");
  CHECK(attended_rows(t, 47, true) == 48 && attended_rows(t, 48, true) == -1, "a step's last position");
  CHECK(attended_rows(t, -1, true) == 0 && attended_rows(t, INT32_MAX, true) == -1, "a step's padding");
  const Pages big{ids, 0x7FFFFFFF, 1, 0x7FFFFFFF, 9, 10};
  CHECK(table_rows(big) == 0x7FFFFFFFl << 10 && attended_rows(big, INT32_MAX, true) == 0x80000000l, "64 bits");
  return 0;
}
