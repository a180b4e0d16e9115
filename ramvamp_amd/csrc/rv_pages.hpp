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

template <typename I>
RV_HD I units_per_range(I total, I ranges) {
  const I per = (total + ranges - 1) / ranges;
  return per > 1 ? per : 1;
}

// Which of its range's two partials a cut item's piece is kept in: the first when
// it opens the range (the item may have begun before), else the second (it runs on
// past the range's end).
template <typename I>
RV_HD int partial_of(I range, I per, I item_start) {
  return item_start > range * per ? 1 : 0;
}

// Walks the units [start, end), the first of which is unit `off` of sequence s:
// visit(sequence, its rows, item, first unit, last unit + 1 of the item, the first
// unit's place in the line).
template <typename I, typename Rows, typename Visit>
RV_HD void walk_units(uint32_t s, I off, I start, I end, I items, Rows rows_of, Visit visit) {
  for (I at = start; at < end;) {
    const I rows = rows_of(s), units = units_of(rows);
    if (off >= units * items) {
      off -= units * items;
      ++s;
      continue;
    }
    const I item = off / units, u0 = off - item * units;
    const I u1 = units < u0 + (end - at) ? units : u0 + (end - at);
    visit(s, rows, item, u0, u1, at);
    off += u1 - u0;
    at += u1 - u0;
  }
}

// The partials of an item cut into `pieces` are joined by whoever leaves the last
// of them; past kFlat pieces first in groups of kGroup, whose partials the last of
// a group replaces by one.
constexpr int kFlat = 32, kGroup = 16;

RV_HD uint32_t groups_of(uint32_t pieces) {
  return pieces > (uint32_t)kFlat ? (pieces + kGroup - 1) / kGroup : 1;
}

}  // namespace rv
