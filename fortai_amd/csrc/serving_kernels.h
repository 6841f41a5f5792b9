// Host-side launchers of the serving operators' kernels (rope.hip, kv8_cache.hip,
// kv8_attention.hip, verify.hip).  Every launcher enqueues on the given stream and
// returns hipGetLastError() of the launch; the entry points that call them
// (fortai_hip_serving.hip) have checked the arguments.
#pragma once

#include "element_types.h"
#include "kv8_device.h"

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fortai_hip {

struct RopeParams {
    const void *x = nullptr;
    void *out = nullptr;
    const int32_t *positions = nullptr;  // [rows]
    const float *norm = nullptr;         // [head], or null: no norm
    const double *turns = nullptr;       // [rotary / 2]: theta_i / (2 pi)
    float attention = 1.0f, eps = 0.0f;
    int rows = 0, heads = 0, head = 0, rotary = 0;
    int64_t x_row = 0, x_head = 0, out_row = 0, out_head = 0;  // pitches in elements
    bool interleaved = false;
    bool half4 = false;  // rotary / 2 is a multiple of 4
};
// vec: x and out allow four-element accesses
hipError_t launch_rope(const RopeParams &p, Dtype dtype, bool vec, hipStream_t stream);

// vec: keys and values allow four-element accesses
hipError_t launch_kv8_append(const Kv8View &cache, const Kv8Rows &batch, Dtype dtype, const void *keys, int64_t key_pitch,
    const void *values, int64_t value_pitch, bool vec, hipStream_t stream);
hipError_t launch_kv8_read(const Kv8View &cache, const Kv8Rows &batch, Dtype dtype, void *keys, int64_t key_pitch,
    void *values, int64_t value_pitch, bool vec, hipStream_t stream);
// cache: the first layer; layer_codes, layer_tops: bytes and maxima of a layer's planes; from, to: host arrays
hipError_t launch_kv8_copy_pages(const Kv8View &cache, size_t layer_codes, size_t layer_tops, int layers,
    const int32_t *from, const int32_t *to, int count, hipStream_t stream);

// Sequences that share their first tokens' pages.
struct Kv8Sharing {
    const int32_t *starts = nullptr;    // [groups + 1], sequences
    const int32_t *shared = nullptr;    // [groups], tokens
    const int32_t *group_of = nullptr;  // [sequences]
    int groups = 0, max_rows = 0;       // rows of a group
};

struct Kv8AttentionParams {
    Kv8View cache;
    Kv8Rows batch;
    Kv8Sharing sharing;  // of calls that share
    const void *q = nullptr, *gate = nullptr;  // gate: null, or at q's pitches
    void *out = nullptr;
    int64_t q_row = 0, q_head = 0, out_row = 0;
    int group = 0;            // query heads of a kv head
    float scale_log2 = 0.0f;  // softmax scale * log2(e) / 127
    bool vec = false;         // q, gate and out allow four-element accesses
    float *partial = nullptr;        // [kKv8SharedRows][head]
    f32x4_t *partial_ml = nullptr;   // [kKv8SharedRows]
    int splits = 0, row_tiles = 0;  // set by the launcher; of a call that shares, for each sequence's own tokens
    int shared_splits = 0, shared_row_tiles = 0, shared_rows = 0, own_rows = 0, own_at = 0, first_block = 0;
};
hipError_t launch_kv8_shared_attention(const Kv8AttentionParams &p, Dtype dtype, const Kv8SharedPlan &plan, hipStream_t stream);
hipError_t launch_kv8_attention(const Kv8AttentionParams &p, Dtype dtype, const Kv8Plan &plan, hipStream_t stream);
hipError_t launch_kv8_clear(void *storage, size_t bytes, hipStream_t stream);


// a row's chunk of the vocabulary: its largest logit, the first token that has it, sum of exp((x - top) / T)
struct VerifyPart {
    double sum;
    float top;
    int32_t place;
};

// a row: its largest logit, the first token that has it, sum of exp((x - top) / T)
struct VerifyRow {
    double sum;
    float top;
    int32_t place;
};

// a sequence's rows [begin, end) and the one that decides (-1: it has no rows)
struct VerifyDecision {
    VerifyRow target, draft;  // of that row
    double uniform;           // for the token that is drawn
    int32_t begin, end, row;
    int32_t rejected;         // the draft that was turned down there, -1: none in the vocabulary
    int32_t against_draft;    // whether one was: what p has over q is drawn from
};

struct VerifyParams {
    const void *target = nullptr, *draft = nullptr;  // [rows][vocab]; draft null: drafts without probabilities
    int64_t target_pitch = 0, draft_pitch = 0;
    const int64_t *tokens = nullptr;        // [rows]
    const float *uniforms = nullptr;        // [rows]
    const float *temperatures = nullptr;    // [sequences], or null: 1
    const int32_t *row_starts = nullptr;    // [sequences + 1]
    int64_t *emitted = nullptr;             // [rows]
    int32_t *accepted = nullptr;            // [sequences]
    float *logprobs = nullptr;              // [rows], or null
    VerifyPart *parts = nullptr;            // [2][max_rows][chunks]
    double *weights = nullptr;              // [sequences][chunks]
    VerifyDecision *decisions = nullptr;    // [sequences]
    VerifyRow *row_stats = nullptr;         // [max_rows], of the target's rows up to the deciding one
    int rows = 0, max_rows = 0, sequences = 0, vocab = 0, chunk = 0, chunks = 0;
};
hipError_t launch_verify(const VerifyParams &p, Dtype dtype, bool vec, hipStream_t stream);

}  // namespace fortai_hip
