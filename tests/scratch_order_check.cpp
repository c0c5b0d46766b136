// Host-only check of the order between uses of the learned layers' scratch (csrc/scratch_order.h)
// against a fake of the runtime's calls.  Built and run by tests/test_layers_scratch.py with g++;
// prints "ok" on success.
#include <cstdio>
#include <string>

#include "scratch_order.h"

using namespace af2;

static int failures = 0;

static int a, b, context_stream;

// What the calls for `next` after `last` are: r(ecord), w(ait) and s(ynchronize).
static void expect(const char *what, ScratchUse last, ScratchUse next, bool grow, const char *want) {
  std::string calls;
  const int status = order_scratch(
      last, next, grow,
      [&](const void *stream) {
        calls += stream == last.stream ? "r" : "?";
        return 0;
      },
      [&] { return calls += "w", 0; }, [&] { return calls += "s", 0; });
  if (status == 0 && calls == want) return;
  std::printf("FAILED %s: calls \"%s\", expected \"%s\"\n", what, calls.c_str(), want);
  ++failures;
}

int main() {
  const ScratchUse none, on_a{&a, 7, false}, on_b{&b, 8, false}, context{&context_stream, 0, true};
  expect("first use", none, on_a, false, "");
  expect("first use that grows", none, on_a, true, "");
  expect("same stream", on_a, on_a, false, "");
  expect("same stream, grows", on_a, on_a, true, "s");
  expect("another stream", on_a, on_b, false, "w");
  expect("another stream, grows", on_a, on_b, true, "s");
  expect("a new stream with a destroyed one's handle", on_a, {&a, 9, false}, false, "w");
  expect("the same per-thread handle in two threads", {&b, 8, false}, {&b, 10, false}, false, "w");
  expect("the context's stream twice", context, context, false, "");
  expect("the context's stream twice, grows", context, context, true, "rs");
  expect("after the context's stream", context, on_a, false, "rw");
  expect("before the context's stream", on_a, context, false, "w");
  // a call that fails ends it
  int later = 0;
  const int status = order_scratch(context, on_a, false, [](const void *) { return 5; }, [&] { return ++later; },
                                   [&] { return ++later; });
  if (status != 5 || later) std::printf("FAILED a failing record: status %d\n", status), ++failures;
  if (failures) return 1;
  std::printf("ok\n");
  return 0;
}
