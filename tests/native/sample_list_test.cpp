// The list of sample.hip on host threads: filled twice in a row, every thread
// gets both counts, however late it reads them.

#include "../../vx_amd/csrc/kernels/sample_list.h"

#include <atomic>
#include <chrono>
#include <cstdio>
#include <pthread.h>
#include <thread>
#include <vector>

namespace {

constexpr int kThreads = 8;

struct Workgroup {
  pthread_barrier_t barrier;
  Workgroup() { pthread_barrier_init(&barrier, nullptr, kThreads); }
  ~Workgroup() { pthread_barrier_destroy(&barrier); }
};

struct Group {
  Workgroup *wg;
  int id;
  int late; // the thread that leaves each barrier after the others
  int thread() const { return id; }
  void sync() const {
    pthread_barrier_wait(&wg->barrier);
    if (id == late) {
      std::this_thread::sleep_for(std::chrono::milliseconds(5));
    }
  }
  static uint32_t add(uint32_t &n) { return __atomic_fetch_add(&n, 1u, __ATOMIC_RELAXED); }
};

std::atomic<int> failures{0};

void expect(bool ok, const char *what, int thread, int late, int got) {
  if (!ok) {
    fprintf(stderr, "%s: thread %d, late %d: %d\n", what, thread, late, got);
    ++failures;
  }
}

} // namespace

int main() {
  for (int late = 0; late < kThreads; ++late) {
    Workgroup wg;
    uint32_t count = 77;
    unsigned long long list[16];
    std::vector<std::thread> threads;
    for (int t = 0; t < kThreads; ++t) {
      threads.emplace_back([&, t] {
        const Group group{&wg, t, late};
        auto entries = [&](int n) {
          return [t, n](auto take) {
            for (int e = 0; e < n; ++e) {
              take((unsigned long long)(t * n + e));
            }
          };
        };
        // more than the list holds, then fewer
        const int first = vxk::fill_list(group, count, list, entries(4));
        const int second = vxk::fill_list(group, count, list, entries(1));
        expect(first == 4 * kThreads, "first count", t, late, first);
        expect(second == kThreads, "second count", t, late, second);
      });
    }
    for (auto &t : threads) {
      t.join();
    }
    unsigned seen = 0;
    for (int e = 0; e < kThreads; ++e) {
      seen |= 1u << list[e];
    }
    expect(seen == (1u << kThreads) - 1, "entries", -1, late, (int)seen);
  }
  if (!failures) {
    puts("ok");
  }
  return failures != 0;
}
