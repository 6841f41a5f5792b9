// What the entry points of the serving operators share (fortai_hip_serving.hip,
// fortai_hip_step.hip).
#pragma once

#include "fortai_hip_context.h"

#include <hip/hip_runtime.h>

namespace fortai_hip {

// The context's device for the length of a call; the caller's own device is
// current again after it.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        if (before_ != device) (void)hipSetDevice(device);
        device_ = device;
    }
    ~DeviceScope() {
        if (before_ != device_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;

private:
    int before_ = 0, device_ = 0;
};

// Making a handle is no work of a graph: its copy or clearing would wait for a replay.
inline const char *check_no_capture(fortai_hip_q8_context *c) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(c->stream, &status) == hipSuccess && status == hipStreamCaptureStatusNone) return nullptr;
    return "handles are created before a capture begins";
}

}  // namespace fortai_hip
