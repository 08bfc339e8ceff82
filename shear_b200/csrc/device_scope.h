// The calling thread's current device, put back at the end of a call.
#pragma once

namespace tessa {

// Api: get(int* device) and set(int device), each 0 or an error.
template <class Api>
class DeviceScope {
 public:
  DeviceScope() = default;
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  ~DeviceScope() {
    if (before_ >= 0) Api::set(before_);
  }
  // Makes `device` current until the scope ends.
  int enter(int device) {
    int now = -1;
    int e = Api::get(&now);
    if (e == 0) e = Api::set(device);
    if (e == 0 && now != device) before_ = now;
    return e;
  }

 private:
  int before_ = -1;
};

}  // namespace tessa
