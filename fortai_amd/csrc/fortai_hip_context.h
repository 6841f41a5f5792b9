// The device context behind the C ABI's handles, and the error and allocation
// helpers of the entry points (shared by the files that define entry points).
#pragma once

#include "../../include/fortai_hip_backend.h"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <cstdio>

struct fortai_hip_q8_context {
    int device = 0;
    hipStream_t stream = nullptr;
    hipEvent_t start = nullptr, stop = nullptr;
    int *position = nullptr;    // device: current token position
    int64_t *token = nullptr;   // device: current token id
    int8_t *scratch_act = nullptr;
    size_t scratch_act_bytes = 0;
    float *scratch_out = nullptr;
    size_t scratch_out_bytes = 0;
    float *scratch_aux = nullptr;
    size_t scratch_aux_bytes = 0;
    float *argmax_value = nullptr;
    int32_t *argmax_index = nullptr;
    void *scratch_q8l = nullptr;  // quantized FFN hidden of the ABI FFN paths
    size_t scratch_q8l_bytes = 0;
    void *noalloc_scratch = nullptr;  // device address of this GPU's `scratch` array (set at create)
    hipEvent_t noalloc_done = nullptr;  // recorded after this context's last use of that array
    hipGraph_t graph = nullptr;
    hipGraphExec_t graph_exec = nullptr;
    char error[256] = {};
};

namespace fortai_hip {

inline int fail(fortai_hip_q8_context *ctx, int code, const char *op, hipError_t err = hipSuccess) {
    if (ctx) {
        if (err == hipSuccess) std::snprintf(ctx->error, sizeof(ctx->error), "%s", op);
        else std::snprintf(ctx->error, sizeof(ctx->error), "%s: %s", op, hipGetErrorString(err));
    }
    return code;
}

inline int done(fortai_hip_q8_context *ctx, hipError_t err, const char *op) {
    return err == hipSuccess ? FORTAI_HIP_OK : fail(ctx, FORTAI_HIP_RUNTIME_ERROR, op, err);
}

template <typename T>
hipError_t alloc(T **ptr, size_t count) {
    *ptr = nullptr;
    if (count == 0) return hipSuccess;
    return hipMalloc(reinterpret_cast<void **>(ptr), count * sizeof(T));
}

template <typename T>
void release(T *&ptr) {
    if (ptr) (void)hipFree(ptr);
    ptr = nullptr;
}

}  // namespace fortai_hip
