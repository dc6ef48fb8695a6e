// PerDeviceOnce against a stand-in for the CUDA runtime (no GPU): whoever finds a device not yet done runs the
// action before going on, also while another thread is still at it, and an action that throws leaves it undone.
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <stdexcept>
#include <thread>

#include "common.cuh"

namespace {
thread_local int device = 0;
bool no_device = false;
}  // namespace

extern "C" cudaError_t cudaGetDevice(int* d) {
  *d = device;
  return no_device ? cudaErrorNoDevice : cudaSuccess;
}
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }

#define CHECK(cond)                                              \
  do {                                                           \
    if (!(cond)) {                                               \
      std::fprintf(stderr, "line %d: %s\n", __LINE__, #cond);    \
      return 1;                                                  \
    }                                                            \
  } while (0)

int main() {
  {  // once per device
    static rb200::PerDeviceOnce once;
    int runs[3] = {};
    for (int i = 0; i < 5; ++i) {
      device = i % 2;
      once.run([&] { ++runs[device]; });
    }
    CHECK(runs[0] == 1 && runs[1] == 1);
    device = rb200::PerDeviceOnce::kMaxDevices;  // not remembered
    for (int i = 0; i < 2; ++i) once.run([&] { ++runs[2]; });
    device = 0, no_device = true;
    once.run([&] { ++runs[2]; });
    no_device = false;
    CHECK(runs[2] == 3);
  }
  {  // an action that throws is tried again
    static rb200::PerDeviceOnce once;
    bool threw = false;
    try {
      once.run([] { throw std::runtime_error("attribute"); });
    } catch (const std::runtime_error&) {
      threw = true;
    }
    int runs = 0;
    for (int i = 0; i < 2; ++i) once.run([&] { ++runs; });
    CHECK(threw && runs == 1);
  }
  {  // a second thread that comes while the first is still at it has the action behind it, too, when it goes on
    static rb200::PerDeviceOnce once;
    std::mutex lock;
    std::condition_variable changed;
    bool started = false, finish = false;
    std::thread first([&] {
      once.run([&] {
        std::unique_lock<std::mutex> l(lock);
        started = true;
        changed.notify_all();
        changed.wait(l, [&] { return finish; });
      });
    });
    {
      std::unique_lock<std::mutex> l(lock);
      changed.wait(l, [&] { return started; });
    }
    bool ran = false;
    once.run([&] { ran = true; });
    {
      std::lock_guard<std::mutex> l(lock);
      finish = true;
      changed.notify_all();
    }
    first.join();
    CHECK(ran);
    bool again = false;
    once.run([&] { again = true; });
    CHECK(!again);
  }
  std::puts("ok");
  return 0;
}
