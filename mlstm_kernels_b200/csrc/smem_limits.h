// How much dynamic shared memory kernels may be launched with (host compilers too).
#pragma once
#include <cstddef>
#include <map>
#include <mutex>
#include <utility>

namespace mlstm {

// A kernel's limit belongs to the process, its launches to the threads that make them.  A kernel whose need depends on the call's sizes
// must not have its limit lowered for a smaller call: between another thread's setting and its launch that would make the launch fail.
// So limits only rise.
class SmemLimits {
 public:
  // set(): raises the limit of `kernel` on `device` to `bytes`, 0 on success; called where no call before has asked for as much
  template <class Set> int allow(int device, const void* kernel, size_t bytes, Set set) {
    std::lock_guard<std::mutex> lock(mu_);
    size_t& have = limits_[{device, kernel}];
    if (bytes <= have) return 0;
    const int rc = set();
    if (rc == 0) have = bytes;
    return rc;
  }

 private:
  std::mutex mu_;
  std::map<std::pair<int, const void*>, size_t> limits_;
};

}  // namespace mlstm
