// Entry points of the serving operators (include/fortai_hip_backend.h): rotary
// positions, the 8-bit paged cache with its attention and page copies, and draft
// verification.  Argument checks and launches only; the kernels are in rope.hip,
// kv8_cache.hip, kv8_attention.hip and verify.hip.
#include "fortai_hip_context.h"
#include "serving_checks.h"
#include "serving_kernels.h"

#include <new>
#include <vector>

using namespace fortai_hip;

namespace {

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

}  // namespace

struct fortai_hip_rope {
    fortai_hip_q8_context *context = nullptr;
    int device = 0;
    int rotary = 0;
    bool interleaved = false;
    float attention = 1.0f;
    double *turns = nullptr;
};

extern "C" {

// ---------------------------------------------------------- rotary positions
int fortai_hip_rope_create(fortai_hip_q8_context *c, int rope_dimension, int interleaved, double base, int scaling,
    double factor, int original_context, double beta_fast, double beta_slow, double attention_factor,
    fortai_hip_rope **rope) {
    if (!c || !rope) return FORTAI_HIP_INVALID;
    *rope = nullptr;
    if (const char *wrong = check_rope_create(rope_dimension, base, scaling, factor, original_context, beta_fast,
            beta_slow, attention_factor))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    double turns[128];
    rope_turns(rope_dimension, base, scaling, factor, original_context, beta_fast, beta_slow, turns);
    const int pairs = rope_dimension / 2;
    auto *h = new (std::nothrow) fortai_hip_rope;
    if (!h) return fail(c, FORTAI_HIP_RUNTIME_ERROR, "rope: out of host memory");
    h->context = c;
    h->device = c->device;
    h->rotary = rope_dimension;
    h->interleaved = interleaved != 0;
    h->attention = static_cast<float>(attention_factor);
    const DeviceScope scope(c->device);
    hipError_t e = alloc(&h->turns, pairs);
    if (e == hipSuccess) e = hipMemcpyAsync(h->turns, turns, pairs * sizeof(double), hipMemcpyHostToDevice, c->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
    if (e != hipSuccess) {
        release(h->turns);
        delete h;
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "rope create", e);
    }
    *rope = h;
    return FORTAI_HIP_OK;
}

int fortai_hip_rope_destroy(fortai_hip_rope *h) {
    if (!h) return FORTAI_HIP_OK;
    const DeviceScope scope(h->device);
    release(h->turns);
    delete h;
    return FORTAI_HIP_OK;
}

int fortai_hip_rope_device(fortai_hip_rope *h, int dtype, const void *input, int64_t input_row_pitch,
    int64_t input_head_pitch, int rows, int heads, int head_size, const void *positions, const void *norm,
    float epsilon, void *output, int64_t output_row_pitch, int64_t output_head_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    fortai_hip_q8_context *c = h->context;
    if (const char *wrong = check_rope(h->rotary, dtype, input, input_row_pitch, input_head_pitch, rows, heads,
            head_size, positions, norm, epsilon, output, output_row_pitch, output_head_pitch))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    if (rows == 0) return FORTAI_HIP_OK;
    RopeParams p;
    p.x = input;
    p.out = output;
    p.positions = static_cast<const int32_t *>(positions);
    p.norm = static_cast<const float *>(norm);
    p.turns = h->turns;
    p.attention = h->attention;
    p.eps = epsilon;
    p.rows = rows;
    p.heads = heads;
    p.head = head_size;
    p.rotary = h->rotary;
    p.x_row = input_row_pitch;
    p.x_head = input_head_pitch;
    p.out_row = output_row_pitch;
    p.out_head = output_head_pitch;
    p.interleaved = h->interleaved;
    p.half4 = (h->rotary / 2) % 4 == 0;
    const bool vec = vector4_ok(input, dtype, input_row_pitch, input_head_pitch) &&
        vector4_ok(output, dtype, output_row_pitch, output_head_pitch);
    const DeviceScope scope(c->device);
    return done(c, launch_rope(p, static_cast<Dtype>(dtype), vec, c->stream), "rotary positions");
}

}  // extern "C"
