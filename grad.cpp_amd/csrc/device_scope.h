// The device that a call's memory is on is the current one while the call runs.
#pragma once

#include "api_error.h"

namespace gh {

struct DeviceScope {
    int before = 0;
    explicit DeviceScope(int device) {
        HIP_CHECK(hipGetDevice(&before));
        if (before != device) HIP_CHECK(hipSetDevice(device));
        now = device;
    }
    ~DeviceScope() {
        if (before != now) (void)hipSetDevice(before);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    int now = 0;
};

}  // namespace gh
