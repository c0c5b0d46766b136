// scratch_order.h -- the order between uses of one scratch buffer on several streams.
//
// A use follows an event behind the last one, unless both are on one stream.  A handle does not name
// a stream for good: it may be destroyed with work pending and its handle given to the next, and
// cudaStreamPerThread is another stream in each thread; the streams' ids tell them apart.
//
// Plain C++ on purpose: the calls are given, so the same code runs against fakes in a host-only test.
#pragma once

namespace af2 {

struct ScratchUse {
  const void *stream = nullptr;   // NULL: none yet
  unsigned long long id = 0;      // not asked for where the stream is lasting
  bool lasting = false;           // lives as long as the buffer: its event is recorded when it is needed
  bool operator==(const ScratchUse &o) const { return stream == o.stream && id == o.id; }
};

// Orders `next` behind `last`.  grow: the buffer is about to be replaced, so the host waits.  record(stream)
// puts the event there, wait() makes next's stream wait for it, synchronize() the host; each returns a
// status, 0 when it is done.
template <typename Record, typename Wait, typename Synchronize>
auto order_scratch(const ScratchUse &last, const ScratchUse &next, bool grow, Record &&record, Wait &&wait,
                   Synchronize &&synchronize) -> decltype(wait()) {
  if (!last.stream || (!grow && last == next)) return {};
  if (last.lasting)
    if (auto status = record(last.stream); status != decltype(wait()){}) return status;
  return grow ? synchronize() : wait();
}

}  // namespace af2
