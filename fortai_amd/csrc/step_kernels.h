// Host-side launchers of the kernels around a step's products (norm_tokens.hip,
// logit_rules.hip, gdn_rows.hip, gdn_chunks.hip).  Every launcher enqueues on the
// given stream and returns hipGetLastError() of the launch; the entry points that
// call them (fortai_hip_step.hip) have checked the arguments.
#pragma once

#include "element_types.h"

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fortai_hip {

struct NormTokensParams {
    const void *x = nullptr, *residual = nullptr, *gate = nullptr;  // residual, gate: or null
    void *sum = nullptr, *out = nullptr;  // or null
    const float *norm = nullptr;          // [group], or null: no norm
    int8_t *codes = nullptr;              // [blocks_pad][ld][32], or null
    float *scales = nullptr;              // [blocks_pad][ld]
    int64_t x_row = 0, residual_row = 0, gate_row = 0, sum_row = 0, out_row = 0;  // pitches in elements
    int rows = 0, width = 0, group = 0, ld = 0, blocks_pad = 0;
    float eps = 0.0f;
};
// vec: all arrays allow four-element accesses
hipError_t launch_norm_tokens(const NormTokensParams &p, Dtype dtype, bool vec, hipStream_t stream);
hipError_t launch_tokens_read(const int8_t *codes, const float *scales, int ld, int rows, int width, void *out,
    int64_t out_row, Dtype dtype, bool vec, hipStream_t stream);

struct LogitRulesParams {
    const void *logits = nullptr;
    void *out = nullptr;                       // may be logits
    const int32_t *row_starts = nullptr;       // [sequences + 1]
    const int64_t *tokens = nullptr;           // [rows], or null
    const int64_t *history = nullptr;          // [sequences][history_pitch], or null
    const int32_t *history_lengths = nullptr;  // [sequences]
    const float *penalties = nullptr;          // [sequences][3], or null: none
    const float *bias = nullptr;               // [vocab] at bias_pitch, or null
    const uint32_t *masks = nullptr;           // [mask_count][mask_pitch], or null
    const int32_t *mask_of = nullptr;          // [rows]
    int64_t logits_row = 0, out_row = 0, bias_pitch = 0, mask_pitch = 0, history_pitch = 0;
    int rows = 0, vocab = 0, sequences = 0, window = 0, mask_count = 0;
};
// vec: logits, out and bias allow four-element accesses
hipError_t launch_logit_rules(const LogitRulesParams &p, Dtype dtype, bool vec, hipStream_t stream);

// ------------------------------------------------- the delta rule over rows
constexpr int kGdnMaxPending = 16;      // rows that may wait for their verdict
constexpr int kGdnFewRows = 16;         // a sequence's rows up to which the recurrent kernel takes them
constexpr int kGdnChunk = 64;           // rows of a chunk otherwise
constexpr int kGdnRun = 16;             // rows whose keys are kept by dims
constexpr int kGdnMaxSequences = 16384;
constexpr int kGdnMaxTaps = 8;

// One layer's planes of the cache, and its shape.
struct GdnView {
    float *states = nullptr;   // [slots][value_heads][head][head]: [value dim][key dim]
    float *inputs = nullptr;   // [slots][taps - 1 + pending][channels], oldest first
    float *keys = nullptr;     // [slots][pending][key_heads][head]
    float *updates = nullptr;  // [slots][pending][value_heads][head]
    float *decays = nullptr;   // [slots][pending][value_heads]
    int *counts = nullptr;     // [slots]: pending rows
    int slots = 0, key_heads = 0, value_heads = 0, head = 0, taps = 0, pending = 0;
    __host__ __device__ int channels() const { return (2 * key_heads + value_heads) * head; }
};

struct GdnRows {
    const int32_t *starts = nullptr;    // [sequences + 1]
    const int32_t *slots = nullptr;     // [sequences]
    const int32_t *standing = nullptr;  // [sequences], or null: every pending row stands
    int sequences = 0, rows = 0, max_rows = 0;
};

struct GdnRowsParams {
    GdnView cache;
    GdnRows batch;
    const void *qkv = nullptr, *alpha = nullptr, *beta = nullptr;
    void *out = nullptr;
    const float *conv = nullptr, *ssm_a = nullptr, *ssm_dt = nullptr;
    int64_t qkv_row = 0, alpha_row = 0, beta_row = 0, out_row = 0;
    float eps = 0.0f;
    int *arrivals = nullptr;  // [kGdnMaxSequences][key_heads + 1], zeros between calls
    bool pairs = false;       // qkv allows two-element accesses
    int few = kGdnFewRows;    // sequences of more rows go through chunks
    // of these, a run of 16 rows and a head at a time (gdn_chunks.hip); numbers as two fp16
    // halves of x 2^15 (weights 2^18):
    _Float16 *asks = nullptr;         // [runs][queries over sqrt(head), keys][key_heads], by rows
    _Float16 *keys_by_dim = nullptr;  // [runs][key_heads], by dims
    _Float16 *through = nullptr;      // [runs][value_heads]: W, by rows
    _Float16 *inner = nullptr;        // [runs][value_heads][4]: weights of the chunk's updates, by rows
    float *values = nullptr;          // [runs][value_heads]: V, then U, by dims
    float *chunk_gates = nullptr;     // [runs][value_heads][2][kGdnRun]: decays since the chunk's start, and to its end
    uint32_t *columns = nullptr;      // [runs][value_heads][head]: of a chunk's value dims, at its first run (gdn_chunks.hip)
    int *faint = nullptr;             // beside them: the last row with too little in its text, -1: none
    float *decay = nullptr;           // [rows][value_heads]: logarithms
    float *rate = nullptr;            // [rows][value_heads]: beta
    int *stands = nullptr;    // [kGdnMaxSequences]
};
// runs of up to `rows` rows (their places: gdn_chunks.hip), and of the rest of the last chunk
inline size_t gdn_runs(size_t rows) { return rows / kGdnRun + rows / (kGdnRun + 1) + 4; }
// few rows of every sequence that has few
hipError_t launch_gdn_few(const GdnRowsParams &p, Dtype dtype, hipStream_t stream);
// the others: convolution, norms and gates; products within chunks; the states through them
hipError_t launch_gdn_many(const GdnRowsParams &p, Dtype dtype, hipStream_t stream);
// slots to[i] become copies of slots from[i], in every layer (host arrays); cache: the first layer
hipError_t launch_gdn_copy_slots(const GdnView &cache, int layers, const int32_t *from, const int32_t *to, int count, hipStream_t stream);

}  // namespace fortai_hip
