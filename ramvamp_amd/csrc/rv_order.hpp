// rv_order.hpp — the stream a cache's calls are queued on, moved from one to another so
// that what is queued on the new one runs behind what the earlier ones hold, also where
// calls were captured on one in between: a captured call waits for nothing outside its
// graph, so what came before the capture is remembered for the first uncaptured call
// after it. Free of HIP's own calls so that it also runs on the host.
#pragma once

namespace rv {

// Api: Stream; Error, zero where all is well; capturing(stream); recordable(stream), whether
// an event can be recorded on it now; record(stream) into the one event there is;
// wait(stream) for that event; kUnsupported.
template <typename Api>
struct StreamOrder {
  typedef typename Api::Stream Stream;
  typedef typename Api::Error Error;

  Api api;
  Stream stream{};
  bool holds = true;      // uncaptured calls, or waits for those of other streams
  Stream behind{};        // where `pending`: what it held has still to be waited for
  bool pending = false;
  bool recorded = false;  // the event stands for that

  // A call is about to be queued on the stream (a captured one waits for nothing).
  Error settle() {
    if ((holds && !pending) || api.capturing(stream)) return Error{};
    const Error e = pending ? settle(stream) : Error{};
    if (e == Error{}) holds = true;
    return e;
  }

  Error move_to(Stream next) {
    if (next == stream) return Error{};
    const bool from = api.capturing(stream), to = api.capturing(next);
    Error e{};
    if (!from && (e = settle()) != Error{}) return e;
    if (holds) {
      // (Not of a stream that is captured, nor of the null stream while one that it
      // waits for is: for them the event is left until it is needed.)
      const bool now = !from && (!to || api.recordable(stream));
      if (now && (e = api.record(stream)) != Error{}) return e;
      behind = stream;
      recorded = now;
      pending = true;
    }
    if (!to && pending && (e = settle(next)) != Error{}) return e;
    stream = next;
    holds = !to;
    return Error{};
  }

 private:
  Error settle(Stream s) {
    if (behind != s) {
      Error e{};
      if (!recorded) {
        if (!api.recordable(behind)) return Api::kUnsupported;
        if ((e = api.record(behind)) != Error{}) return e;
        recorded = true;
      }
      if ((e = api.wait(s)) != Error{}) return e;
    }
    pending = false;
    return Error{};
  }
};

}  // namespace rv
