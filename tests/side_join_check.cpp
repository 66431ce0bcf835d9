// Host check of csrc/side_join.cuh: the caller's stream waits for every forked
// stream when a call returns early, and nothing is added to one that joined them.
#include <cstdio>
#include <string>

#include "side_join.cuh"

static std::string trace;
static bool fail_record = false;

struct Fake {
  using Stream = char;
  using Event = char;
  static bool record(char ev, char s) {
    trace += std::string("record ") + ev + " on " + s + "; ";
    return !fail_record;
  }
  static bool wait(char s, char ev) {
    trace += std::string(1, s) + " waits for " + ev + "; ";
    return true;
  }
  static void synchronize(char s) { trace += std::string("synchronize ") + s + "; "; }
};

// A call with launches at steps 0 .. 4, the streams a and b forked after steps 0 and 1;
// the launch of step `bad` fails.
static int call(int bad) {
  cce::SideJoin<Fake> join('m', 'e');
  if (bad == 0) return 1;
  join.forked('a');
  if (bad == 1) return 1;
  join.forked('b');
  for (int step = 2; step < 5; ++step)
    if (bad == step) return 1;
  join.joined();
  return 0;
}

static bool check(int bad, const char* want) {
  trace.clear();
  const int rc = call(bad);
  if (rc == (bad < 5) && trace == want) return true;
  std::printf("step %d: rc %d, \"%s\", expected \"%s\"\n", bad, rc, trace.c_str(), want);
  return false;
}

int main() {
  const char* a = "record e on a; m waits for e; ";
  const char* ab = "record e on a; m waits for e; record e on b; m waits for e; ";
  bool ok = check(0, "") && check(1, a) && check(2, ab) && check(3, ab) && check(4, ab) && check(5, "");
  fail_record = true;
  ok = ok && check(3, "record e on a; synchronize a; record e on b; synchronize b; ");
  std::puts(ok ? "SIDE_JOIN_OK" : "FAILED");
  return ok ? 0 : 1;
}
