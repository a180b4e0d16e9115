// A cache's hand-over from stream to stream (ramvamp_amd/csrc/rv_order.hpp) on the host:
// streams are sets of the work that has to end before what is queued next on them.
// Prints nothing and exits 0 when all holds; else names what does not.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <set>

#include "../ramvamp_amd/csrc/rv_order.hpp"

#define CHECK(c, ...)               \
  do {                              \
    if (!(c)) {                     \
      printf("%s: ", #c);           \
      printf(__VA_ARGS__);          \
      printf("\n");                 \
      exit(1);                      \
    }                               \
  } while (0)

typedef std::set<int> Work;

// Streams 0 .. 4; 0 is the null stream, which waits for stream 1 (a blocking one) and so
// takes no event while that is captured.
static Work on[5], event;
static bool captured[5];
static int run, step_no;

struct Streams {
  typedef int Stream;
  typedef int Error;
  static constexpr int kUnsupported = 7;
  static bool capturing(int s) { return captured[s]; }
  static bool recordable(int s) { return !captured[s] && !(s == 0 && captured[1]); }
  static int record(int s) {
    CHECK(!captured[s], "run %d step %d: an event recorded into the capture of %d", run, step_no, s);
    event = on[s];
    return s == 0 && captured[1] ? 9 : 0;
  }
  static int wait(int s) {
    CHECK(!captured[s], "run %d step %d: the capture of %d waits for what is outside", run, step_no, s);
    on[s].insert(event.begin(), event.end());
    return 0;
  }
};

int main() {
  std::mt19937 g(3);
  long queued = 0, refused = 0;
  for (run = 0; run < 20000; ++run) {
    for (int s = 0; s < 5; ++s) on[s].clear(), captured[s] = false;
    event.clear();
    rv::StreamOrder<Streams> order;
    Work all;
    for (step_no = 0; step_no < 40; ++step_no) {
      const int s = (int)(g() % 5);
      switch (g() % 4) {
        case 0:  // a capture begins or ends (never of the null stream)
          if (s) captured[s] = !captured[s];
          break;
        case 1: {
          const int e = order.move_to(s);
          // (Refused: the work to wait for is on a stream that cannot be asked now.)
          CHECK(e == 0 || e == 9 || !Streams::recordable(order.behind), "run %d step %d: %d", run, step_no, e);
          CHECK(e != 9 || captured[1], "run %d step %d", run, step_no);
          CHECK(e ? order.stream != s : order.stream == s, "run %d step %d", run, step_no);
          break;
        }
        default: {  // a call, as C makes it: on the stream that was set last
          const int e = order.settle();
          CHECK(e == 0 || !Streams::recordable(order.behind), "run %d step %d: %d", run, step_no, e);
          refused += e != 0;
          if (e || captured[order.stream]) break;
          for (int w : all) CHECK(on[order.stream].count(w), "run %d step %d: stream %d does not wait for call %d", run, step_no, order.stream, w);
          all.insert((int)all.size());
          on[order.stream] = all;
          ++queued;
        }
      }
    }
  }
  CHECK(queued > 50000 && refused < queued / 20, "%ld queued, %ld refused", queued, refused);
  return 0;
}
