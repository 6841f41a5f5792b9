// Entry points of the serving operators (include/fortai_hip_backend.h): rotary
// positions, the 8-bit paged cache with its attention and page copies, and draft
// verification.  Argument checks and launches only; the kernels are in rope.hip,
// kv8_cache.hip, kv8_attention.hip and verify.hip.
#include "fortai_hip_context.h"
#include "serving_checks.h"
#include "serving_kernels.h"
#include "serving_scope.h"

#include <mutex>
#include <new>

using namespace fortai_hip;

struct fortai_hip_rope {
    fortai_hip_q8_context *context = nullptr;
    int device = 0;
    int rotary = 0;
    bool interleaved = false;
    float attention = 1.0f;
    double *turns = nullptr;
};

struct fortai_hip_kv8_cache {
    fortai_hip_q8_context *context = nullptr;
    int device = 0;
    Kv8Shape shape;
    uint8_t *storage = nullptr;
    bool owned = false;
    // partial results of split attention calls, [kKv8SharedRows][head + 4]: made
    // with the cache and never again, so that a captured call keeps its address
    float *partial = nullptr;
    std::mutex launches;  // a call's two launches follow each other on the stream

    Kv8View layer(int index) const {
        Kv8View v;
        const size_t at = static_cast<size_t>(index);
        v.keys = reinterpret_cast<int8_t *>(storage) + at * shape.layer_codes();
        v.values = v.keys + shape.codes();
        v.key_max = reinterpret_cast<float *>(storage + 2 * shape.codes()) + at * shape.layer_tops();
        v.value_max = v.key_max + shape.layers * shape.layer_tops();
        v.pages = shape.pages;
        v.page_tokens = shape.page_tokens;
        v.kv_heads = shape.kv_heads;
        v.head = shape.head;
        return v;
    }
};

struct fortai_hip_verifier {
    fortai_hip_q8_context *context = nullptr;
    int device = 0;
    int max_rows = 0, max_sequences = 0, vocab = 0, chunk = 0, chunks = 0;
    // made with the verifier and never again, so that a captured call keeps their addresses
    VerifyPart *parts = nullptr;
    double *weights = nullptr;
    VerifyDecision *decisions = nullptr;
    VerifyRow *row_stats = nullptr;
    std::mutex launches;  // a call's launches follow each other on the stream
};

namespace {

Kv8Rows batch_rows(const fortai_hip_kv8_batch *b) {
    Kv8Rows r;
    r.starts = static_cast<const int32_t *>(b->device_row_starts);
    r.lengths = static_cast<const int32_t *>(b->device_lengths);
    r.tables = static_cast<const int32_t *>(b->device_tables);
    r.sequences = b->sequences;
    r.rows = b->rows;
    r.max_rows = b->max_rows;
    r.pitch = b->table_pitch;
    return r;
}

const char *check_batch(const fortai_hip_kv8_batch *b) {
    if (!b) return "kv8: no batch";
    return check_kv8_batch(b->sequences, b->rows, b->max_rows, b->table_pitch, b->device_row_starts, b->device_lengths,
        b->device_tables);
}

bool empty(const fortai_hip_kv8_batch *b) { return b->sequences == 0 || b->rows == 0 || b->max_rows == 0; }

// Attention of a batch's rows, over tokens that sequences share (sharing: may be null) and their own.
int attend(fortai_hip_kv8_cache *h, int layer, const fortai_hip_kv8_batch *batch, const fortai_hip_kv8_groups *sharing, int dtype,
    const void *query, int64_t query_pitch, int64_t query_head_pitch, const void *gate, int heads, float scale, int max_length,
    int max_shared, void *output, int64_t output_pitch) {
    fortai_hip_q8_context *c = h->context;
    if (const char *wrong = check_batch(batch)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (sharing)
        if (const char *wrong = check_kv8_groups(sharing->groups, sharing->max_rows, batch->rows, batch->sequences, max_shared,
                sharing->device_starts, sharing->device_shared, sharing->device_group_of))
            return fail(c, FORTAI_HIP_INVALID, wrong);
    if (empty(batch)) return FORTAI_HIP_OK;
    if (const char *wrong = check_kv8_attention(h->shape, layer, dtype, batch->rows, batch->max_rows, query, query_pitch,
            query_head_pitch, gate, heads, scale, max_length, output, output_pitch))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    Kv8AttentionParams p;
    p.cache = h->layer(layer);
    p.batch = batch_rows(batch);
    p.q = query;
    p.gate = gate;
    p.out = output;
    p.q_row = query_pitch;
    p.q_head = query_head_pitch;
    p.out_row = output_pitch;
    p.group = heads / h->shape.kv_heads;
    p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634074 / 127.0);
    p.vec = vector4_ok(query, dtype, query_pitch, query_head_pitch) && vector4_ok(output, dtype, output_pitch, 0) &&
        vector4_ok(gate, dtype, 0, 0);
    p.partial = h->partial;
    p.partial_ml = reinterpret_cast<f32x4_t *>(h->partial + static_cast<size_t>(kKv8SharedRows) * h->shape.head);
    const bool fp32 = dtype == FORTAI_HIP_DTYPE_F32;
    const int head = h->shape.head, kv_heads = h->shape.kv_heads;
    const int64_t rows = static_cast<int64_t>(batch->max_rows) * p.group;
    const DeviceScope scope(c->device);
    const std::lock_guard<std::mutex> lock(h->launches);
    if (sharing && sharing->groups > 0 && sharing->max_rows > 0) {
        const Kv8SharedPlan plan = kv8_shared_plan(fp32, head, batch->sequences, sharing->groups, kv_heads, rows,
            static_cast<int64_t>(sharing->max_rows) * p.group, max_length > max_shared ? max_length - max_shared : 1, max_shared);
        if (plan.shares) {
            p.sharing.starts = static_cast<const int32_t *>(sharing->device_starts);
            p.sharing.shared = static_cast<const int32_t *>(sharing->device_shared);
            p.sharing.group_of = static_cast<const int32_t *>(sharing->device_group_of);
            p.sharing.groups = sharing->groups;
            p.sharing.max_rows = sharing->max_rows;
            return done(c, launch_kv8_shared_attention(p, static_cast<Dtype>(dtype), plan, c->stream), "kv8 shared attention");
        }
    }
    const Kv8Plan plan = kv8_plan(fp32, head, batch->sequences, kv_heads, rows, max_length);
    return done(c, launch_kv8_attention(p, static_cast<Dtype>(dtype), plan, c->stream), "kv8 attention");
}

}  // namespace

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
    if (const char *wrong = check_no_capture(c)) return fail(c, FORTAI_HIP_INVALID, wrong);
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

// --------------------------------------------------------------- 8-bit cache
size_t fortai_hip_kv8_bytes(int layers, int pages, int page_tokens, int kv_heads, int head_size) {
    Kv8Shape s;
    s.layers = layers;
    s.pages = pages;
    s.page_tokens = page_tokens;
    s.kv_heads = kv_heads;
    s.head = head_size;
    return kv8_bytes(s);
}

int fortai_hip_kv8_create(fortai_hip_q8_context *c, int layers, int pages, int page_tokens, int kv_heads, int head_size,
    void *device_storage, size_t storage_bytes, fortai_hip_kv8_cache **cache) {
    if (!c || !cache) return FORTAI_HIP_INVALID;
    *cache = nullptr;
    Kv8Shape s;
    s.layers = layers;
    s.pages = pages;
    s.page_tokens = page_tokens;
    s.kv_heads = kv_heads;
    s.head = head_size;
    if (const char *wrong = check_kv8_shape(s)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (const char *wrong = check_no_capture(c)) return fail(c, FORTAI_HIP_INVALID, wrong);
    const size_t bytes = kv8_bytes(s);
    if (bytes == 0) return fail(c, FORTAI_HIP_INVALID, "kv8: the cache is larger than any memory");
    if (device_storage && (storage_bytes < bytes || !aligned(device_storage, 16)))
        return fail(c, FORTAI_HIP_INVALID, "kv8: storage smaller than fortai_hip_kv8_bytes, or not aligned to 16 bytes");
    auto *h = new (std::nothrow) fortai_hip_kv8_cache;
    if (!h) return fail(c, FORTAI_HIP_RUNTIME_ERROR, "kv8: out of host memory");
    h->context = c;
    h->device = c->device;
    h->shape = s;
    h->storage = static_cast<uint8_t *>(device_storage);
    const DeviceScope scope(c->device);
    hipError_t e = hipSuccess;
    if (!device_storage) {
        e = alloc(&h->storage, bytes);
        h->owned = e == hipSuccess;
        if (e == hipSuccess) e = launch_kv8_clear(h->storage, bytes, c->stream);
    }
    if (e == hipSuccess) e = alloc(&h->partial, static_cast<size_t>(kKv8SharedRows) * (head_size + 4));
    if (e != hipSuccess) {
        if (h->owned) release(h->storage);
        release(h->partial);
        delete h;
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "kv8 create", e);
    }
    *cache = h;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_destroy(fortai_hip_kv8_cache *h) {
    if (!h) return FORTAI_HIP_OK;
    const DeviceScope scope(h->device);
    if (h->owned) release(h->storage);
    release(h->partial);
    delete h;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_append_device(fortai_hip_kv8_cache *h, int layer, const fortai_hip_kv8_batch *batch, int dtype,
    const void *keys, int64_t key_pitch, const void *values, int64_t value_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    fortai_hip_q8_context *c = h->context;
    if (const char *wrong = check_batch(batch)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (empty(batch)) return FORTAI_HIP_OK;
    if (const char *wrong = check_kv8_rows(h->shape, layer, dtype, keys, key_pitch, values, value_pitch, false))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    const bool vec = vector4_ok(keys, dtype, key_pitch, 0) && vector4_ok(values, dtype, value_pitch, 0);
    const DeviceScope scope(c->device);
    return done(c, launch_kv8_append(h->layer(layer), batch_rows(batch), static_cast<Dtype>(dtype), keys, key_pitch,
        values, value_pitch, vec, c->stream), "kv8 append");
}

int fortai_hip_kv8_read_device(fortai_hip_kv8_cache *h, int layer, const fortai_hip_kv8_batch *batch, int dtype,
    void *keys, int64_t key_pitch, void *values, int64_t value_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    fortai_hip_q8_context *c = h->context;
    if (const char *wrong = check_batch(batch)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (empty(batch)) return FORTAI_HIP_OK;
    if (const char *wrong = check_kv8_rows(h->shape, layer, dtype, keys, key_pitch, values, value_pitch, true))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    const bool vec = vector4_ok(keys, dtype, key_pitch, 0) && vector4_ok(values, dtype, value_pitch, 0);
    const DeviceScope scope(c->device);
    return done(c, launch_kv8_read(h->layer(layer), batch_rows(batch), static_cast<Dtype>(dtype), keys, key_pitch,
        values, value_pitch, vec, c->stream), "kv8 read");
}

int fortai_hip_kv8_attention_device(fortai_hip_kv8_cache *h, int layer, const fortai_hip_kv8_batch *batch, int dtype,
    const void *query, int64_t query_pitch, int64_t query_head_pitch, const void *gate, int heads, float scale,
    int max_length, void *output, int64_t output_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    return attend(h, layer, batch, nullptr, dtype, query, query_pitch, query_head_pitch, gate, heads, scale, max_length, 0, output,
        output_pitch);
}

int fortai_hip_kv8_shared_attention_device(fortai_hip_kv8_cache *h, int layer, const fortai_hip_kv8_batch *batch,
    const fortai_hip_kv8_groups *sharing, int dtype, const void *query, int64_t query_pitch, int64_t query_head_pitch,
    const void *gate, int heads, float scale, int max_length, int max_shared, void *output, int64_t output_pitch) {
    if (!h) return FORTAI_HIP_INVALID;
    if (!sharing) return fail(h->context, FORTAI_HIP_INVALID, "kv8: no groups");
    return attend(h, layer, batch, sharing, dtype, query, query_pitch, query_head_pitch, gate, heads, scale, max_length, max_shared,
        output, output_pitch);
}

int fortai_hip_kv8_copy_pages(fortai_hip_kv8_cache *h, const int32_t *from, const int32_t *to, int count) {
    if (!h || count < 0) return FORTAI_HIP_INVALID;
    if (count == 0) return FORTAI_HIP_OK;
    fortai_hip_q8_context *c = h->context;
    if (!from || !to) return fail(c, FORTAI_HIP_INVALID, "kv8 copy: null array");
    try {
        if (const char *wrong = check_page_pairs(from, to, count, h->shape.pages)) return fail(c, FORTAI_HIP_INVALID, wrong);
    } catch (...) {
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "kv8 copy: out of host memory");
    }
    const DeviceScope scope(c->device);
    return done(c, launch_kv8_copy_pages(h->layer(0), h->shape.layer_codes(), h->shape.layer_tops(), h->shape.layers, from,
        to, count, c->stream), "kv8 copy pages");
}

// -------------------------------------------------------- draft verification
int fortai_hip_verifier_create(fortai_hip_q8_context *c, int max_rows, int max_sequences, int vocab,
    fortai_hip_verifier **verifier) {
    if (!c || !verifier) return FORTAI_HIP_INVALID;
    *verifier = nullptr;
    if (const char *wrong = check_verifier(max_rows, max_sequences, vocab)) return fail(c, FORTAI_HIP_INVALID, wrong);
    if (const char *wrong = check_no_capture(c)) return fail(c, FORTAI_HIP_INVALID, wrong);
    auto *h = new (std::nothrow) fortai_hip_verifier;
    if (!h) return fail(c, FORTAI_HIP_RUNTIME_ERROR, "verify: out of host memory");
    h->context = c;
    h->device = c->device;
    h->max_rows = max_rows;
    h->max_sequences = max_sequences;
    h->vocab = vocab;
    h->chunk = verify_chunk(max_rows, vocab);
    h->chunks = (vocab + h->chunk - 1) / h->chunk;
    const DeviceScope scope(c->device);
    hipError_t e = alloc(&h->parts, 2 * static_cast<size_t>(max_rows) * h->chunks);
    if (e == hipSuccess) e = alloc(&h->weights, static_cast<size_t>(max_sequences) * h->chunks);
    if (e == hipSuccess) e = alloc(&h->decisions, static_cast<size_t>(max_sequences));
    if (e == hipSuccess) e = alloc(&h->row_stats, static_cast<size_t>(max_rows));
    if (e != hipSuccess) {
        release(h->parts);
        release(h->weights);
        release(h->decisions);
        release(h->row_stats);
        delete h;
        return fail(c, FORTAI_HIP_RUNTIME_ERROR, "verifier create", e);
    }
    *verifier = h;
    return FORTAI_HIP_OK;
}

int fortai_hip_verifier_destroy(fortai_hip_verifier *h) {
    if (!h) return FORTAI_HIP_OK;
    const DeviceScope scope(h->device);
    release(h->parts);
    release(h->weights);
    release(h->decisions);
    release(h->row_stats);
    delete h;
    return FORTAI_HIP_OK;
}

int fortai_hip_verify_drafts_device(fortai_hip_verifier *h, int dtype, const void *target_logits, int64_t target_pitch,
    const void *draft_logits, int64_t draft_pitch, const void *tokens, const void *uniforms, const void *temperatures,
    int sequences, const void *row_starts, int rows, void *emitted, void *accepted, void *logprobs) {
    if (!h) return FORTAI_HIP_INVALID;
    fortai_hip_q8_context *c = h->context;
    if (const char *wrong = check_verify(h->max_rows, h->max_sequences, h->vocab, dtype, target_logits, target_pitch,
            draft_logits, draft_pitch, tokens, uniforms, temperatures, sequences, row_starts, rows, emitted, accepted, logprobs))
        return fail(c, FORTAI_HIP_INVALID, wrong);
    if (sequences == 0) return FORTAI_HIP_OK;
    VerifyParams p;
    p.target = target_logits;
    p.draft = draft_logits;
    p.target_pitch = target_pitch;
    p.draft_pitch = draft_pitch;
    p.tokens = static_cast<const int64_t *>(tokens);
    p.uniforms = static_cast<const float *>(uniforms);
    p.temperatures = static_cast<const float *>(temperatures);
    p.row_starts = static_cast<const int32_t *>(row_starts);
    p.emitted = static_cast<int64_t *>(emitted);
    p.accepted = static_cast<int32_t *>(accepted);
    p.logprobs = static_cast<float *>(logprobs);
    p.parts = h->parts;
    p.weights = h->weights;
    p.decisions = h->decisions;
    p.row_stats = h->row_stats;
    p.rows = rows;
    p.max_rows = h->max_rows;
    p.sequences = sequences;
    p.vocab = h->vocab;
    p.chunk = h->chunk;
    p.chunks = h->chunks;
    const bool vec = h->vocab % 4 == 0 && vector4_ok(target_logits, dtype, target_pitch, 0) &&
        (!draft_logits || vector4_ok(draft_logits, dtype, draft_pitch, 0));
    const DeviceScope scope(c->device);
    const std::lock_guard<std::mutex> lock(h->launches);
    return done(c, launch_verify(p, static_cast<Dtype>(dtype), vec, c->stream), "draft verification");
}

}  // extern "C"
