// Threads that make the first calls of all devices at once: each device is prepared exactly once, a failure is tried
// again, and whoever gets 0 reads what the successful preparation wrote.  Built with the thread sanitizer.
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#include "once.h"

int main() {
  using nvfp4::kMaxDevices;
  static nvfp4::OncePerDevice once;
  static int fits[kMaxDevices][4], tries[kMaxDevices];      // plain, as the library's are
  std::atomic<int> wrong{0}, go{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&, t] {
      go.fetch_add(1);
      while (go.load() < 8) {}
      for (int i = 0; i < kMaxDevices; ++i) {
        const int dev = (i + t) % kMaxDevices;
        int status;
        do {
          status = once.run(dev, [&] {
            if (tries[dev]++ == 0) return 3;                // the first try of each device fails
            for (int s = 0; s < 4; ++s) fits[dev][s] = dev * 4 + s + 1;
            return 0;
          });
          if (status != 0 && status != 3) ++wrong;
        } while (status);
        for (int s = 0; s < 4; ++s)
          if (fits[dev][s] != dev * 4 + s + 1) ++wrong;
      }
    });
  for (auto& t : threads) t.join();
  for (int dev = 0; dev < kMaxDevices; ++dev)
    if (tries[dev] != 2) ++wrong;
  int calls = 0;
  for (int i = 0; i < 3; ++i) once.run(-1, [&] { return ++calls, 0; });
  if (calls != 3) ++wrong;
  std::printf("wrong %d\n", wrong.load());
  return wrong.load() != 0;
}
