// A fact that is found once and kept (host code).  A search that fails is not kept: the next call tries again, so one
// transient error does not refuse every later call of the process.
#pragma once
#include <mutex>

namespace dfl_host {
template <class T>
class FoundOnce {
 public:
  // find(T*) returns 0 on success.  *value is what the first successful search found; the return value is this search's.
  template <class Find>
  int get(T* value, Find find) {
    std::lock_guard<std::mutex> hold(mutex_);
    if (!found_) {
      T fresh{};
      const int rc = find(&fresh);
      if (rc) return rc;
      value_ = fresh;
      found_ = true;
    }
    *value = value_;
    return 0;
  }

 private:
  std::mutex mutex_;
  bool found_ = false;
  T value_{};
};
}  // namespace dfl_host
