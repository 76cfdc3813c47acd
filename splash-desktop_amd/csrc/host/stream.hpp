// What the operators between the projections share when they launch.
#pragma once
#include <string>

#include "ops.hpp"

namespace sq::ops {

inline void launched(hipError_t e, const char *what) {
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

// Launches go to the stream's device, whichever is current; the current one is put back.
class OnStreamDevice {
 public:
  explicit OnStreamDevice(hipStream_t stream) {
    hipDevice_t device = 0;
    int current = 0;
    if (!stream) return;
    launched(hipStreamGetDevice(stream, &device), "stream device");
    launched(hipGetDevice(&current), "current device");
    if (current == device) return;
    launched(hipSetDevice(device), "stream device");
    before_ = current;
  }
  ~OnStreamDevice() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
  OnStreamDevice(const OnStreamDevice &) = delete;
  OnStreamDevice &operator=(const OnStreamDevice &) = delete;

 private:
  int before_ = -1;
};

inline bool aligned(const Buffer &b, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(b.ptr) % bytes == 0; }

}  // namespace sq::ops
