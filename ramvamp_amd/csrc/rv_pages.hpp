// rv_pages.hpp — where a row of a paged cache lies, and how the attention over
// ragged lengths is dealt to workgroups: the integer arithmetic of the paged
// kernels, free of device code so that it also runs on the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#define RV_HD __host__ __device__ __forceinline__

namespace rv {

// A batch's page tables (rv_page_table) and the pool they name pages of.
struct Pages {
  const int32_t* ids;
  long stride;
  uint32_t n_seqs, pages;  // of the table
  uint32_t n_pages;        // of the pool
  int shift;               // log2 of a page's rows
};

enum Place { kHere, kPadding, kNoSequence, kNoPosition, kNoPage };

// Row `pos` of sequence `seq`: its page and the row inside it. `got` is what was
// refused: the sequence, the position or the page id.
RV_HD Place place_of(const Pages& t, int pos, int seq, uint32_t& page, uint32_t& row, uint32_t& got) {
  if (pos < 0) return kPadding;
  if ((uint32_t)seq >= t.n_seqs) {
    got = (uint32_t)seq;
    return kNoSequence;
  }
  const uint32_t p = (uint32_t)pos >> t.shift;
  if (p >= t.pages) {
    got = (uint32_t)pos;
    return kNoPosition;
  }
  page = (uint32_t)t.ids[(long)seq * t.stride + p];
  if (page >= t.n_pages) {
    got = page;
    return kNoPage;
  }
  row = (uint32_t)pos & ((1u << t.shift) - 1);
  return kHere;
}

RV_HD long table_rows(const Pages& t) { return (long)t.pages << t.shift; }

// Rows attended by a sequence of length `len`, or at position `len` with the row
// there (step); -1: refused.
RV_HD long attended_rows(const Pages& t, int len, bool step) {
  const long rows = step ? (len < 0 ? 0 : (long)len + 1) : (long)len;
  return rows >= 0 && rows <= table_rows(t) ? rows : -1;
}

// The work of a batch is a line of units, one for every kUnitRows rows of every
// item (a kv head, or a part of its query heads) of every sequence in order. It is
// cut into ranges of `per` units, one a workgroup.
constexpr int kUnitRows = 128;

template <typename I>
RV_HD I units_of(I rows) {
  return rows > 0 ? (rows + (kUnitRows - 1)) / kUnitRows : 0;
}

// x / y for a quotient below 2^21, by a float reciprocal of y that is off by at
// most 2^-22 of itself (x and y round by 2^-24, the product by 2^-24: the estimate
// is less than one off).
RV_HD uint32_t quotient(uint32_t x, uint32_t y, float reciprocal_y) {
  uint32_t q = (uint32_t)((float)x * reciprocal_y);
  const uint32_t r = x - q * y;
  if ((int32_t)r < 0)
    --q;
  else if (r >= y)
    ++q;
  return q;
}

// Which of its range's two partials a cut item's piece is kept in: the first when
// it opens the range (the item may have begun before), else the second (it runs on
// past the range's end).
template <typename I>
RV_HD int partial_of(I range, I per, I item_start) {
  return item_start > range * per ? 1 : 0;
}

// Floats of a partial: `cols` rows of hd values, then (maximum, sum) of each column, in
// whole lines of the caches. Two partials have different writers, and a CU that reads
// one may keep its lines: none of them may hold a part of another that is still to come.
constexpr uint32_t kLineFloats = 32;

RV_HD uint32_t partial_floats(uint32_t cols, uint32_t hd) {
  return (cols * (hd + 2) + kLineFloats - 1) / kLineFloats * kLineFloats;
}

struct PlainQuotient {
  template <typename I>
  RV_HD I operator()(I x, I y) const {
    return x / y;
  }
};

// Walks the units [start, end), the first of which is unit `off` of sequence s:
// visit(sequence, its rows, item, first unit, last unit + 1 of the item, the first
// unit's place in the line). next_of(s): the first sequence from s on that has rows, or
// kNoMore, where the walk ends (the lengths have been changed under it).
constexpr uint32_t kNoMore = 0xFFFFFFFFu;

template <typename I, typename Rows, typename Next, typename Visit, typename Quotient = PlainQuotient>
RV_HD void walk_units(uint32_t s, I off, I start, I end, I items, Rows rows_of, Next next_of, Visit visit,
                      Quotient divide = Quotient()) {
  for (I at = start; at < end;) {
    const I rows = rows_of(s), units = units_of(rows);
    if (off >= units * items) {
      off -= units * items;
      s = next_of(s + 1);
      if (s == kNoMore) return;
      continue;
    }
    const I item = divide(off, units), u0 = off - item * units;
    const I u1 = units < u0 + (end - at) ? units : u0 + (end - at);
    visit(s, rows, item, u0, u1, at);
    off += u1 - u0;
    at += u1 - u0;
  }
}

// Workgroups are dealt to the XCDs in turn, so with 2^slots of them, in_slot ranges to
// each, workgroup b takes a range such that consecutive ones share an XCD: range r is
// of slot r / in_slot. A slot's ranges make groups of kGroup. An item's pieces (ranges
// w0 .. w1) are joined by whoever leaves the last of them, or, where they are many and
// of several groups, first within each group, then across groups.
constexpr uint32_t kGroup = 16;

RV_HD uint32_t slot_of(uint32_t b, int slots) { return b & ((1u << slots) - 1); }

RV_HD uint32_t range_of(uint32_t b, int slots, uint32_t in_slot) { return slot_of(b, slots) * in_slot + (b >> slots); }

struct Group {
  uint32_t id, lo, hi;  // its number, first and last range
};

RV_HD Group group_of(uint32_t r, uint32_t slot, uint32_t in_slot) {
  const uint32_t k = (r - slot * in_slot) / kGroup, last = slot * in_slot + in_slot - 1;
  Group g;
  g.id = slot * ((in_slot + kGroup - 1) / kGroup) + k;
  g.lo = slot * in_slot + k * kGroup;
  g.hi = g.lo + kGroup - 1 < last ? g.lo + kGroup - 1 : last;
  return g;
}

// Of the two partials a group keeps for items that other groups have ranges of too:
// the first is the item's that is there from the group's first unit on.
RV_HD uint32_t group_partial(const Group& g, uint32_t item_start, uint32_t per) {
  return 2 * g.id + (item_start > g.lo * per ? 1 : 0);
}

struct Pieces {
  uint32_t first, count;    // of the group: its ranges of the item
  uint32_t w0, all;         // of the item: its first range, and how many
  uint32_t group0, groups;  // and its first group's partial, and how many groups
};

template <typename Quotient = PlainQuotient>
RV_HD Pieces pieces_of(const Group& g, uint32_t w0, uint32_t w1, uint32_t item_start, uint32_t per, uint32_t in_slot,
                       Quotient divide = Quotient()) {
  Pieces p;
  p.first = w0 > g.lo ? w0 : g.lo;
  p.count = (w1 < g.hi ? w1 : g.hi) - p.first + 1;
  p.w0 = w0;
  p.all = w1 - w0 + 1;
  const Group a = w0 >= g.lo ? g : group_of(w0, divide(w0, in_slot), in_slot);
  const Group z = w1 <= g.hi ? g : group_of(w1, divide(w1, in_slot), in_slot);
  p.group0 = group_partial(a, item_start, per);
  p.groups = z.id - a.id + 1;
  return p;
}

// Pieces are counted by tickets, an item's and a group's as they are left. There are two
// sets, which take turns by the launch: one counts, the one of the launch before is
// cleared. So a launch finds zeros whatever was left of earlier ones, also of one whose
// lengths were changed while it ran, and whose workgroups did not agree on the pieces.
// Whose turn it is each workgroup reads from a word of its own, which it alone writes
// in the launch: kTurns words are shared out evenly over the launch's grid (a power of
// two). All are equal between launches.
constexpr uint32_t kTurns = 512;

struct Turn {
  uint32_t set, used;  // the set that counts, and the tickets of the other to be cleared
};

RV_HD uint32_t own_turn(uint32_t block, uint32_t grid) { return block * (kTurns / grid); }

RV_HD size_t set_words(size_t tickets) { return (tickets + kLineFloats - 1) / kLineFloats * kLineFloats; }

// Lane `lane` of `lanes` of workgroup `block` ends its launch's turn: pass(word, turn)
// for the next launch, of `tickets` this one may have drawn; clear(ticket of the other set).
template <typename Pass, typename Clear>
RV_HD void end_turn(Turn t, uint32_t block, uint32_t grid, uint32_t lane, uint32_t lanes, uint32_t tickets, Pass pass,
                    Clear clear) {
  for (uint32_t c = lane; c < kTurns / grid; c += lanes) pass(own_turn(block, grid) + c, Turn{1 - t.set, tickets});
  for (size_t i = (size_t)block * lanes + lane; i < t.used; i += (size_t)grid * lanes) clear(i);
}

// How `total` units are cut: units a range, and the ranges of a slot (so that every
// slot has as many to do). At most 2^most ranges; 2^few where that makes two units or
// more a range.
struct Cut {
  uint32_t per, in_slot;
};

template <typename Quotient = PlainQuotient>
RV_HD Cut cut_units(uint32_t total, int most, int few, int slots, Quotient divide = Quotient()) {
  const int n = total >> (few + 1) ? few : most;
  Cut c;
  c.per = (total + (1u << n) - 1) >> n;
  if (c.per < 1) c.per = 1;
  const uint32_t used = c.per == 1 ? total : divide(total + c.per - 1, c.per);
  c.in_slot = (used + (1u << slots) - 1) >> slots;
  if (c.in_slot < 1) c.in_slot = 1;
  return c;
}

}  // namespace rv
