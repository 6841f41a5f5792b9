// Entry points of the operators around a step's products (include/fortai_hip_backend.h):
// norm into 8-bit tokens, rules on logits, the delta rule over a batch's rows.  Argument
// checks and launches only; the kernels are in norm_tokens.hip, logit_rules.hip,
// gdn_rows.hip and gdn_chunks.hip.
#include "fortai_hip_context.h"
#include "fortai_hip_kernels.h"
#include "serving_kernels.h"
#include "serving_scope.h"
#include "step_checks.h"
#include "step_kernels.h"

#include <mutex>
#include <new>

using namespace fortai_hip;

struct fortai_hip_gdn_cache {
    fortai_hip_q8_context *context = nullptr;
    int device = 0, max_rows = 0;
    GdnShape shape;
    float *storage = nullptr;
    bool owned = false;
    // made with the cache and never again, so that a captured call keeps their addresses
    int *arrivals = nullptr, *stands = nullptr;
    _Float16 *asks = nullptr, *keys_by_dim = nullptr, *through = nullptr, *inner = nullptr;
    float *values = nullptr, *chunk_gates = nullptr, *decay = nullptr, *rate = nullptr;
    uint32_t *columns = nullptr;
    int *faint = nullptr;
    std::mutex launches;  // a call's launches follow each other on the stream, without another's between them

    GdnView layer(int index) const {
        GdnView v;
        float *planes[6], *at = storage;
        for (int i = 0; i < 6; ++i) {
            const size_t layer_floats = shape.plane(i) * shape.slots;
            planes[i] = at + index * layer_floats;
            at += shape.layers * layer_floats;
        }
        v.states = planes[0];
        v.inputs = planes[1];
        v.keys = planes[2];
        v.updates = planes[3];
        v.decays = planes[4];
        v.counts = reinterpret_cast<int *>(planes[5]);
        v.slots = shape.slots;
        v.key_heads = shape.key_heads;
        v.value_heads = shape.value_heads;
        v.head = shape.head;
        v.taps = shape.taps;
        v.pending = shape.pending;
        return v;
    }
    void release_all() {
        if (owned) release(storage);
        release(arrivals);
        release(stands);
        release(asks);
        release(keys_by_dim);
        release(through);
        release(inner);
        release(values);
        release(chunk_gates);
        release(columns);
        release(faint);
        release(decay);
        release(rate);
    }
};

namespace {

GdnShape gdn_shape(int layers, int slots, int key_heads, int value_heads, int head_size, int conv_kernel, int pending) {
    GdnShape s;
    s.layers = layers;
    s.slots = slots;
    s.key_heads = key_heads;
    s.value_heads = value_heads;
    s.head = head_size;
    s.taps = conv_kernel;
    s.pending = pending;
    return s;
}

}  // namespace

extern "C" {

// ------------------------------------------- norm into 8-bit tokens, and back
int fortai_hip_norm_tokens_device(fortai_hip_q8_context *c, int dtype, const void *x, int64_t x_pitch, const void *residual,
    int64_t residual_pitch, void *sum, int64_t sum_pitch, const void *norm, int group, float epsilon, const void *gate,
    int64_t gate_pitch, int rows, int width, void *output, int64_t output_pitch, void *tokens) {
    if (!c) return FORTAI_HIP_INVALID;
    const NormTokensArrays arrays = {x, residual, sum, norm, gate, output, tokens, x_pitch, residual_pitch, sum_pitch, gate_pitch,
        output_pitch};
    if (const char *wrong = check_norm_tokens(dtype, rows, width, group, epsilon, arrays)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (rows == 0) return FORTAI_HIP_OK;
    NormTokensParams p;
    p.x = x;
    p.residual = residual;
    p.gate = gate;
    p.sum = sum;
    p.out = output;
    p.norm = static_cast<const float *>(norm);
    p.x_row = x_pitch;
    p.residual_row = residual_pitch;
    p.gate_row = gate_pitch;
    p.sum_row = sum_pitch;
    p.out_row = output_pitch;
    p.rows = rows;
    p.width = width;
    p.group = group;
    p.eps = epsilon;
    p.ld = q8_tokens_ld(rows);
    p.blocks_pad = (width / 32 + 3) / 4 * 4;
    p.codes = static_cast<int8_t *>(tokens);
    p.scales = tokens ? reinterpret_cast<float *>(p.codes + static_cast<size_t>(p.ld) * p.blocks_pad * 32) : nullptr;
    const bool vec = vector4_ok(x, dtype, x_pitch, 0) && vector4_ok(residual, dtype, residual ? residual_pitch : 0, 0) &&
        vector4_ok(gate, dtype, gate ? gate_pitch : 0, 0) && vector4_ok(sum, dtype, sum ? sum_pitch : 0, 0) &&
        vector4_ok(output, dtype, output ? output_pitch : 0, 0);
    const DeviceScope scope(c->device);
    return done(c, launch_norm_tokens(p, static_cast<Dtype>(dtype), vec, c->stream), "norm into tokens");
}

int fortai_hip_q8_tokens_read_device(fortai_hip_q8_context *c, int dtype, const void *tokens, int rows, int width, void *output,
    int64_t output_pitch) {
    if (!c) return FORTAI_HIP_INVALID;
    if (const char *wrong = check_tokens_read(dtype, rows, width, tokens, output, output_pitch)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (rows == 0) return FORTAI_HIP_OK;
    const int ld = q8_tokens_ld(rows);
    const int8_t *codes = static_cast<const int8_t *>(tokens);
    const float *scales = reinterpret_cast<const float *>(codes + static_cast<size_t>(ld) * ((width / 32 + 3) / 4 * 4) * 32);
    const DeviceScope scope(c->device);
    return done(c, launch_tokens_read(codes, scales, ld, rows, width, output, output_pitch, static_cast<Dtype>(dtype),
        vector4_ok(output, dtype, output_pitch, 0), c->stream), "tokens read");
}

// ------------------------------------------------------------- logits' rules
int fortai_hip_logits_adjust_device(fortai_hip_q8_context *c, int dtype, const void *logits, int64_t logits_pitch, int rows,
    int vocab, int sequences, const void *row_starts, const fortai_hip_logit_rules *rules, void *output, int64_t output_pitch) {
    if (!c) return FORTAI_HIP_INVALID;
    if (!rules) return fail(c, FORTAI_HIP_INVALID, "logits: no rules");
    const LogitRulesArrays arrays = {logits, row_starts, rules->device_tokens, rules->device_history, rules->device_history_lengths,
        rules->device_penalties, rules->device_bias, rules->device_masks, rules->device_mask_of, output, logits_pitch,
        rules->history_pitch, rules->bias_pitch, rules->mask_pitch, output_pitch};
    if (const char *wrong = check_logit_rules(dtype, rows, vocab, sequences, rules->window, rules->mask_count, arrays))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    if (rows == 0 || sequences == 0) return FORTAI_HIP_OK;
    LogitRulesParams p;
    p.logits = logits;
    p.out = output;
    p.row_starts = static_cast<const int32_t *>(row_starts);
    p.tokens = static_cast<const int64_t *>(rules->device_tokens);
    p.history = static_cast<const int64_t *>(rules->device_history);
    p.history_lengths = static_cast<const int32_t *>(rules->device_history_lengths);
    p.penalties = static_cast<const float *>(rules->device_penalties);
    p.bias = static_cast<const float *>(rules->device_bias);
    p.masks = static_cast<const uint32_t *>(rules->device_masks);
    p.mask_of = static_cast<const int32_t *>(rules->device_mask_of);
    p.logits_row = logits_pitch;
    p.out_row = output_pitch;
    p.bias_pitch = rules->bias_pitch;
    p.mask_pitch = rules->mask_pitch;
    p.history_pitch = rules->history_pitch;
    p.rows = rows;
    p.vocab = vocab;
    p.sequences = sequences;
    p.window = rules->window;
    p.mask_count = rules->mask_count;
    const bool vec = vocab % 4 == 0 && vector4_ok(logits, dtype, logits_pitch, 0) && vector4_ok(output, dtype, output_pitch, 0) &&
        vector4_ok(rules->device_bias, FORTAI_HIP_DTYPE_F32, rules->device_bias ? rules->bias_pitch : 0, 0);
    const DeviceScope scope(c->device);
    return done(c, launch_logit_rules(p, static_cast<Dtype>(dtype), vec, c->stream), "logits' rules");
}

// ------------------------------------------------------------ the delta rule
size_t fortai_hip_gdn_bytes(int layers, int slots, int key_heads, int value_heads, int head_size, int conv_kernel, int pending) {
    return gdn_bytes(gdn_shape(layers, slots, key_heads, value_heads, head_size, conv_kernel, pending));
}

int fortai_hip_gdn_create(fortai_hip_q8_context *c, int layers, int slots, int key_heads, int value_heads, int head_size,
    int conv_kernel, int pending, int max_rows, void *device_storage, size_t storage_bytes, fortai_hip_gdn_cache **cache) {
    if (!c || !cache) return FORTAI_HIP_INVALID;
    *cache = nullptr;
    const GdnShape s = gdn_shape(layers, slots, key_heads, value_heads, head_size, conv_kernel, pending);
    if (const char *wrong = check_gdn_shape(s)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (const char *wrong = check_gdn_rows(max_rows)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (const char *wrong = check_no_capture(c)) return fail(c, FORTAI_HIP_INVALID, wrong);
    const size_t bytes = gdn_bytes(s);
    if (bytes == 0) return fail(c, FORTAI_HIP_INVALID, "gdn: the cache is larger than any memory");
    if (device_storage && (storage_bytes < bytes || !aligned(device_storage, 16)))
        return fail(c, FORTAI_HIP_INVALID, "gdn: storage smaller than fortai_hip_gdn_bytes, or not aligned to 16 bytes");
    auto *h = new (std::nothrow) fortai_hip_gdn_cache;
    if (!h) return fail(c, FORTAI_HIP_RUNTIME_ERROR, "gdn: out of host memory");
    h->context = c;
    h->device = c->device;
    h->max_rows = max_rows;
    h->shape = s;
    h->storage = static_cast<float *>(device_storage);
    const DeviceScope scope(c->device);
    hipError_t e = hipSuccess;
    if (!device_storage) {
        e = alloc(&h->storage, bytes / sizeof(float));
        h->owned = e == hipSuccess;
        if (e == hipSuccess) e = launch_kv8_clear(h->storage, bytes, c->stream);
    }
    const size_t counters = static_cast<size_t>(kGdnMaxSequences) * (key_heads + 1), rows = max_rows;
    if (e == hipSuccess) e = alloc(&h->arrivals, counters);
    if (e == hipSuccess) e = launch_kv8_clear(h->arrivals, counters * sizeof(int), c->stream);
    if (max_rows > kGdnFewRows) {
        if (e == hipSuccess) e = alloc(&h->stands, static_cast<size_t>(kGdnMaxSequences));
        const size_t runs = gdn_runs(rows) * kGdnRun;  // rows of whole runs
        if (e == hipSuccess) e = alloc(&h->asks, runs * 2 * key_heads * 2 * head_size);
        if (e == hipSuccess) e = alloc(&h->keys_by_dim, runs * key_heads * 2 * head_size);
        if (e == hipSuccess) e = alloc(&h->through, runs * value_heads * 2 * head_size);
        if (e == hipSuccess) e = alloc(&h->inner, runs * value_heads * 2 * kGdnChunk);
        if (e == hipSuccess) e = alloc(&h->values, runs * value_heads * head_size);
        if (e == hipSuccess) e = alloc(&h->chunk_gates, runs * value_heads * 2);
        if (e == hipSuccess) e = alloc(&h->columns, gdn_runs(rows) * value_heads * head_size);
        if (e == hipSuccess) e = alloc(&h->faint, gdn_runs(rows) * value_heads * head_size);
        if (e == hipSuccess) e = alloc(&h->decay, rows * value_heads);
        if (e == hipSuccess) e = alloc(&h->rate, rows * value_heads);
    }
    if (e != hipSuccess) {
        (void)hipStreamSynchronize(c->stream);  // a clearing may be under way
        h->release_all();
        delete h;
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "gdn create", e);
    }
    *cache = h;
    return FORTAI_HIP_OK;
}

int fortai_hip_gdn_destroy(fortai_hip_gdn_cache *h) {
    if (!h) return FORTAI_HIP_OK;
    const DeviceScope scope(h->device);
    h->release_all();
    delete h;
    return FORTAI_HIP_OK;
}

int fortai_hip_gdn_run_device(fortai_hip_gdn_cache *h, int layer, const fortai_hip_gdn_batch *batch, int dtype, const void *qkv,
    int64_t qkv_pitch, const void *alpha, int64_t alpha_pitch, const void *beta, int64_t beta_pitch, const void *conv,
    const void *ssm_a, const void *ssm_dt, float epsilon, void *output, int64_t output_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    fortai_hip_q8_context *c = h->context;
    if (!batch) return fail(c, FORTAI_HIP_INVALID, "gdn: no batch");
    if (const char *wrong = check_gdn_batch(batch->sequences, batch->rows, batch->max_rows, h->max_rows, batch->device_row_starts,
            batch->device_slots, batch->device_standing))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    if (batch->sequences == 0 || batch->rows == 0 || batch->max_rows == 0) return FORTAI_HIP_OK;
    const GdnArrays arrays = {qkv, alpha, beta, conv, ssm_a, ssm_dt, output, qkv_pitch, alpha_pitch, beta_pitch, output_pitch};
    if (const char *wrong = check_gdn_run(h->shape, layer, dtype, batch->rows, epsilon, arrays)) return fail(c, FORTAI_HIP_INVALID, wrong);
    GdnRowsParams p;
    p.cache = h->layer(layer);
    p.batch.starts = static_cast<const int32_t *>(batch->device_row_starts);
    p.batch.slots = static_cast<const int32_t *>(batch->device_slots);
    p.batch.standing = static_cast<const int32_t *>(batch->device_standing);
    p.batch.sequences = batch->sequences;
    p.batch.rows = batch->rows;
    p.batch.max_rows = batch->max_rows;
    p.qkv = qkv;
    p.alpha = alpha;
    p.beta = beta;
    p.out = output;
    p.conv = static_cast<const float *>(conv);
    p.ssm_a = static_cast<const float *>(ssm_a);
    p.ssm_dt = static_cast<const float *>(ssm_dt);
    p.qkv_row = qkv_pitch;
    p.alpha_row = alpha_pitch;
    p.beta_row = beta_pitch;
    p.out_row = output_pitch;
    p.eps = epsilon;
    p.arrivals = h->arrivals;
    p.pairs = aligned(qkv, 2 * dtype_bytes(dtype)) && qkv_pitch % 2 == 0;
    p.asks = h->asks;
    p.keys_by_dim = h->keys_by_dim;
    p.through = h->through;
    p.inner = h->inner;
    p.values = h->values;
    p.chunk_gates = h->chunk_gates;
    p.columns = h->columns;
    p.faint = h->faint;
    p.decay = h->decay;
    p.rate = h->rate;
    p.stands = h->stands;
    const Dtype type = static_cast<Dtype>(dtype);
    const DeviceScope scope(c->device);
    const std::lock_guard<std::mutex> lock(h->launches);
    const bool many = batch->max_rows > kGdnFewRows;
    // one sequence that may have many rows, none of them to wait: through chunks whatever their
    // number, which saves a launch (5 us) that would most often find nothing to do
    if (many && batch->sequences == 1 && h->shape.pending == 0) p.few = 0;
    hipError_t e = p.few > 0 ? launch_gdn_few(p, type, c->stream) : hipSuccess;
    if (e == hipSuccess && many) e = launch_gdn_many(p, type, c->stream);
    return done(c, e, "delta rule");
}

int fortai_hip_gdn_copy_slots(fortai_hip_gdn_cache *h, const int32_t *from, const int32_t *to, int count) {
    if (!h || count < 0) return FORTAI_HIP_INVALID;
    if (count == 0) return FORTAI_HIP_OK;
    fortai_hip_q8_context *c = h->context;
    if (!from || !to) return fail(c, FORTAI_HIP_INVALID, "gdn copy: null array");
    try {
        if (const char *wrong = check_slot_pairs(from, to, count, h->shape.slots)) return fail(c, FORTAI_HIP_INVALID, wrong);
    } catch (...) {
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "gdn copy: out of host memory");
    }
    const DeviceScope scope(c->device);
    const std::lock_guard<std::mutex> lock(h->launches);
    return done(c, launch_gdn_copy_slots(h->layer(0), h->shape.layers, from, to, count, c->stream), "gdn copy slots");
}

}  // extern "C"
