// shards.h -- one call's work on the devices of a handle.
#pragma once
#include <exception>
#include <functional>
#include <thread>
#include <vector>

namespace mfb200 {

// Runs work(0) .. work(n - 1) and returns when all have ended: on the calling
// thread where there is one, else each on a thread of its own, so that the
// caller's current device stays what it is. Where a thread cannot be started
// (an exception that must not leave a C entry, nor end the process by way of the
// threads that were), here(i) runs what is left on the calling thread.
template <class Work, class Here>
void run_shards(int n, const Work &work, const Here &here) {
  if (n == 1) {
    work(0);
    return;
  }
  std::vector<std::thread> threads;
  int started = 0;
  try {
    threads.reserve(n);
    for (; started < n; ++started) threads.emplace_back(std::cref(work), started);
  } catch (const std::exception &) {
  }
  for (int i = started; i < n; ++i) here(i);
  for (auto &t : threads) t.join();
}

}  // namespace mfb200
