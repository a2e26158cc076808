// What each stream has been told of waits that gave up in kernels without a handle (b2_lm_sync). The kernels of a device count them in words
// that are never cleared, so that one caller's question does not take the answer from another; a kernel in a graph does not know the
// stream that it is launched on, so a count is all that it can leave.
#pragma once

#include <map>
#include <mutex>
#include <utility>

namespace b2 {

class WaitReports {
 public:
  // Whether `count` waits given up on a device are other than what this stream was last told (none, at first). It is told now.
  bool news(int device, unsigned long long stream, unsigned int count) {
    std::lock_guard<std::mutex> lock(mutex_);
    const auto key = std::make_pair(device, stream);
    if (count == 0 && told_.find(key) == told_.end()) return false;  // nothing is kept for streams while nothing has gone wrong
    unsigned int& told = told_[key];
    const bool other = told != count;
    told = count;
    return other;
  }

 private:
  std::mutex mutex_;
  std::map<std::pair<int, unsigned long long>, unsigned int> told_;
};

}  // namespace b2
