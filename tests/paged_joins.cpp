// What the joins of paged attention rest on (ramvamp_amd/csrc/rv_pages.hpp), on the
// host. Prints nothing and exits 0 when all holds; else names what does not.
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
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

// A partial's line that a CU has read holds nothing of a partial that another
// workgroup writes later.
static void lines() {
  constexpr uint32_t kLine = 128;  // bytes, of L1 and L2
  for (uint32_t cols = 1; cols <= 16; ++cols)
    for (uint32_t hd = 1; hd <= 512; ++hd) {
      const uint32_t bytes = partial_floats(cols, hd) * 4, need = cols * (hd + 2) * 4;
      CHECK(bytes >= need && bytes < need + kLine, "%u x %u: %u of %u", cols, hd, bytes, need);
      for (uint32_t i = 0; i < 3; ++i)
        CHECK((i * bytes + need - 1) / kLine < (i + 1) * bytes / kLine, "%u x %u shares a line", cols, hd);
    }
}

// A launch finds its tickets zero, whatever an earlier one left: workgroups come in any
// order, draw in any number (as where the lengths change under them and they do not
// agree on the pieces), and launches differ in grid and in tickets.
static void turns() {
  std::mt19937 g(11);
  for (int run = 0; run < 300; ++run) {
    const size_t words = set_words(1 + g() % 3000);
    CHECK(words % kLineFloats == 0, "%zu words", words);
    std::vector<Turn> turn(kTurns, Turn{0, 0});
    std::vector<uint32_t> tickets(2 * words, 0);
    for (int launch = 0; launch < 12; ++launch) {
      const uint32_t grid = 8u << (g() % 7), n = 1 + g() % words;
      const uint32_t lanes = 1u << (g() % 7);
      const bool agree = g() % 2;
      const uint32_t set = turn[0].set;
      for (size_t i = 0; i < words; ++i) CHECK(tickets[set * words + i] == 0, "run %d launch %d: ticket %zu", run, launch, i);
      std::vector<uint32_t> order(grid);
      for (uint32_t b = 0; b < grid; ++b) order[b] = b;
      std::shuffle(order.begin(), order.end(), g);
      uint32_t last = 0;
      for (uint32_t b : order) {
        const Turn t = turn[own_turn(b, grid)];
        CHECK(t.set == set && t.used <= words, "run %d launch %d: workgroup %u's turn", run, launch, b);
        if (agree)
          last += tickets[t.set * words]++ == grid - 1;  // one item of all workgroups
        else
          for (int k = 0; k < 3; ++k) tickets[t.set * words + g() % n] += g() % 3;
        for (uint32_t lane = 0; lane < lanes; ++lane)
          end_turn(t, b, grid, lane, lanes, n, [&](uint32_t c, Turn next) { turn.at(c) = next; },
                   [&](size_t i) { tickets.at((1 - t.set) * words + i) = 0; });
      }
      CHECK(!agree || last == 1, "run %d launch %d: %u last", run, launch, last);
    }
  }
}

int main() {
  lines();
  turns();
  return 0;
}
