// Two host threads that ask for a kernel's shared memory at the same time, against the runtime
// of fake_runtime.cpp: the one whose launch is large is held in its first call until the other
// is through, as the scheduler may.  Whoever comes out of `room` finds the limit large enough.
#include <cstdio>
#include <condition_variable>
#include <mutex>
#include <thread>

#include "dense.cuh"

constexpr int kOptIn = 232448, kFixed = 1024, kLarge = 131072;
extern std::mutex m;
extern std::condition_variable changed;
extern int limit;                        // what the kernel may take
extern bool first_in, second_done;

static void kernel(int) {}

static void ask() { eps_b200::dense::room<kernel>(0); }
static int limit_now() { std::lock_guard<std::mutex> l(m); return limit; }

int main() {
  std::thread large([] { ask(); });
  {
    std::unique_lock<std::mutex> l(m);
    changed.wait(l, [] { return first_in; });
  }
  std::thread small([] {
    ask();
    { std::lock_guard<std::mutex> l(m); second_done = true; }
    changed.notify_all();
  });
  large.join();
  const int then = limit_now();          // the large launch comes now
  small.join();
  ask();                           // and every later one
  const int later = limit_now();
  std::printf("%d %d\n", then, later);
  return then >= kLarge && later >= kLarge && later <= kOptIn - kFixed ? 0 : 1;
}
