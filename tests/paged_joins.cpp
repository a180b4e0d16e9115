// What the joins of paged attention rest on (ramvamp_amd/csrc/rv_pages.hpp), on the
// host. Prints nothing and exits 0 when all holds; else names what does not.
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>

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

int main() {
  lines();
  return 0;
}
