// Argument checks and launch rules of the serving operators, free of device
// code so that they also compile for the host alone.  A check returns what is
// wrong with the arguments, or nullptr.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <vector>

namespace fortai_hip {

constexpr int64_t kMaxPitch = int64_t{1} << 31;  // elements: products with int counts stay within 64 bits
constexpr int kMaxRows = 1 << 23;                // a launch's threads stay below 2^32

inline bool dtype_ok(int d) { return d >= 0 && d <= 2; }
inline size_t dtype_bytes(int d) { return d == 0 ? 4 : 2; }
inline bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool pitch_ok(int64_t pitch) { return pitch >= 0 && pitch <= kMaxPitch; }

// Whether rows x heads vectors of `head` elements at these pitches touch no
// element twice (either pitch may be the outer one).
inline bool apart(int64_t rows, int64_t heads, int64_t head, int64_t row_pitch, int64_t head_pitch) {
    const bool by_row = (heads == 1 || head_pitch >= head) &&
        (rows == 1 || row_pitch >= (heads - 1) * (heads == 1 ? 0 : head_pitch) + head);
    const bool by_head = (rows == 1 || row_pitch >= head) &&
        (heads == 1 || head_pitch >= (rows - 1) * (rows == 1 ? 0 : row_pitch) + head);
    return by_row || by_head;
}

// Whether four consecutive elements at this address and at every multiple of
// these pitches are aligned to all four.
inline bool vector4_ok(const void *p, int dtype, int64_t pitch_a, int64_t pitch_b) {
    return aligned(p, 4 * dtype_bytes(dtype)) && pitch_a % 4 == 0 && pitch_b % 4 == 0;
}

// ---------------------------------------------------------- rotary positions
inline const char *check_rope_create(int rope_dimension, double base, int scaling, double factor, int original_context,
    double beta_fast, double beta_slow, double attention_factor) {
    if (rope_dimension < 2 || rope_dimension > 256 || rope_dimension % 2) return "rope: dimension even, 2 to 256";
    if (!(base > 0.0) || !std::isfinite(base)) return "rope: base above 0";
    if (!(attention_factor > 0.0) || !std::isfinite(attention_factor)) return "rope: attention factor above 0";
    if (scaling < 0 || scaling > 2) return "rope: unknown scaling";
    if (scaling != 0 && (!(factor > 0.0) || !std::isfinite(factor))) return "rope: scaling factor above 0";
    if (scaling == 2 && (original_context < 1 || !(base > 1.0) || !(beta_slow > 0.0) || !(beta_fast > beta_slow) ||
        !std::isfinite(beta_fast)))
        return "rope: scaling by parts needs original_context, base > 1 and beta_fast > beta_slow > 0";
    return nullptr;
}

// theta_i / 2 pi of the rope_dimension / 2 pairs
inline void rope_turns(int rope_dimension, double base, int scaling, double factor, int original_context,
    double beta_fast, double beta_slow, double *turns) {
    const double two_pi = 6.283185307179586476925286766559, r = rope_dimension;
    double low = 0.0, high = 0.0;
    if (scaling == 2) {
        // the pair index that makes this many turns within the original context
        const auto pair = [&](double t) { return r * std::log(original_context / (t * two_pi)) / (2.0 * std::log(base)); };
        low = std::fmax(std::floor(pair(beta_fast)), 0.0);
        high = std::fmin(std::ceil(pair(beta_slow)), r - 1.0);
    }
    for (int i = 0; i < rope_dimension / 2; ++i) {
        double theta = std::pow(base, -2.0 * i / r);
        if (scaling == 1) theta /= factor;
        if (scaling == 2) {
            const double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
            theta = theta / factor * ramp + theta * (1.0 - ramp);
        }
        turns[i] = theta / two_pi;
    }
}

inline const char *check_rope(int rotary, int dtype, const void *input, int64_t in_row, int64_t in_head, int rows,
    int heads, int head_size, const void *positions, const void *norm, float epsilon, const void *output,
    int64_t out_row, int64_t out_head) {
    if (!dtype_ok(dtype)) return "rope: unknown dtype";
    if (rows < 0 || rows > kMaxRows || heads < 1 || heads > kMaxRows) return "rope: rows 0 to 2^23, heads 1 to 2^23";
    if (head_size < 4 || head_size > 256 || head_size % 4 || head_size < rotary)
        return "rope: head size a multiple of 4, from the rope dimension to 256";
    if (rows == 0) return nullptr;
    if (!input || !output || !positions) return "rope: null array";
    if (!aligned(input, dtype_bytes(dtype)) || !aligned(output, dtype_bytes(dtype)) || !aligned(positions, 4) ||
        !aligned(norm, 4))
        return "rope: misaligned array";
    if (norm && !(epsilon > 0.0f)) return "rope: the norm needs epsilon > 0";
    if (!pitch_ok(in_row) || !pitch_ok(in_head) || !pitch_ok(out_row) || !pitch_ok(out_head))
        return "rope: pitches 0 to 2^31";
    if (!apart(rows, heads, head_size, out_row, out_head)) return "rope: output vectors overlap";
    if (input == output && ((rows > 1 && in_row != out_row) || (heads > 1 && in_head != out_head)))
        return "rope: in place, both sides have the same pitches";
    return nullptr;
}

// --------------------------------------------------------------- 8-bit cache
struct Kv8Shape {
    int layers = 0, pages = 0, page_tokens = 0, kv_heads = 0, head = 0;
    size_t layer_tops() const { return static_cast<size_t>(pages) * kv_heads; }
    size_t layer_codes() const { return layer_tops() * page_tokens * head; }
    size_t codes() const { return layers * layer_codes(); }  // bytes of the key codes, and of the value codes
    size_t bytes() const { return 2 * codes() + 2 * sizeof(float) * layers * layer_tops(); }
};

inline const char *check_kv8_shape(const Kv8Shape &s) {
    if (s.layers < 1 || s.layers > 4096 || s.kv_heads < 1 || s.kv_heads > 1024) return "kv8: layers 1 to 4096, heads 1 to 1024";
    if (s.pages < 1) return "kv8: no pages";
    if (s.page_tokens != 16 && s.page_tokens != 32 && s.page_tokens != 64) return "kv8: pages of 16, 32 or 64 tokens";
    if (s.head != 64 && s.head != 128 && s.head != 256) return "kv8: heads of 64, 128 or 256";
    return nullptr;  // at most 2^(12 + 10 + 31 + 6 + 8) = 2^67 bytes: kv8_bytes() says which do not fit
}

// 0 where 64 bits do not hold it (no storage is that large)
inline size_t kv8_bytes(const Kv8Shape &s) {
    if (check_kv8_shape(s)) return 0;
    const double about = 2.0 * s.layers * s.pages * s.kv_heads * (static_cast<double>(s.page_tokens) * s.head + 4.0);
    return about < 9.0e15 ? s.bytes() : 0;
}

inline const char *check_kv8_batch(int sequences, int rows, int max_rows, int table_pitch, const void *starts,
    const void *lengths, const void *tables) {
    if (sequences < 0 || sequences > 16384) return "kv8: sequences 0 to 16384";
    if (rows < 0 || rows > kMaxRows || max_rows < 0 || max_rows > rows) return "kv8: rows 0 to 2^23, max_rows 0 to rows";
    if (sequences == 0 || rows == 0 || max_rows == 0) return nullptr;
    if (table_pitch < 1 || table_pitch > (1 << 24)) return "kv8: table pitch 1 to 2^24";
    if (!starts || !lengths || !tables) return "kv8: null array";
    if (!aligned(starts, 4) || !aligned(lengths, 4) || !aligned(tables, 4)) return "kv8: misaligned array";
    return nullptr;
}

// the rows of keys and values that are appended (written == false) or read into
inline const char *check_kv8_rows(const Kv8Shape &s, int layer, int dtype, const void *keys, int64_t key_pitch,
    const void *values, int64_t value_pitch, bool written) {
    const int64_t width = static_cast<int64_t>(s.kv_heads) * s.head;
    if (layer < 0 || layer >= s.layers) return "kv8: no such layer";
    if (!dtype_ok(dtype)) return "kv8: unknown dtype";
    if (!keys || !values) return "kv8: null array";
    if (!aligned(keys, dtype_bytes(dtype)) || !aligned(values, dtype_bytes(dtype))) return "kv8: misaligned array";
    if (!pitch_ok(key_pitch) || !pitch_ok(value_pitch) || (written && (key_pitch < width || value_pitch < width)))
        return written ? "kv8: pitches from kv_heads * head to 2^31" : "kv8: pitches 0 to 2^31";
    return nullptr;
}

inline const char *check_kv8_attention(const Kv8Shape &s, int layer, int dtype, int rows, int max_rows, const void *query,
    int64_t query_pitch, int64_t query_head_pitch, const void *gate, int heads, float scale, int max_length,
    const void *output, int64_t output_pitch) {
    if (layer < 0 || layer >= s.layers) return "kv8: no such layer";
    if (!dtype_ok(dtype)) return "kv8: unknown dtype";
    if (heads < 1 || heads % s.kv_heads || heads > 65535) return "kv8: heads a multiple of the cache's, at most 65535";
    const int64_t group = heads / s.kv_heads;
    if (group * max_rows > kMaxRows || (group * max_rows + 7) / 8 * s.kv_heads > 65535 || 4 * s.kv_heads > 65535)
        return "kv8: more rows in a sequence than a call takes";
    if (!(std::fabs(scale) <= 1e30f)) return "kv8: scale is not a number, or beyond 1e30";
    if (max_length < 0) return "kv8: max_length below 0";
    if (!query || !output) return "kv8: null array";
    const size_t e = dtype_bytes(dtype);
    if (!aligned(query, e) || !aligned(gate, e) || !aligned(output, e)) return "kv8: misaligned array";
    if (!pitch_ok(query_pitch) || !pitch_ok(query_head_pitch)) return "kv8: pitches 0 to 2^31";
    if (!pitch_ok(output_pitch) || (rows > 1 && output_pitch < static_cast<int64_t>(heads) * s.head))
        return "kv8: output pitch from heads * head to 2^31";
    return nullptr;
}

// Pairs that can be copied in any order: ids within the pool, no page written
// twice, none both read and written.  May throw std::bad_alloc.
inline const char *check_page_pairs(const int32_t *from, const int32_t *to, int count, int pages) {
    for (int i = 0; i < count; ++i)
        if (from[i] < 0 || from[i] >= pages || to[i] < 0 || to[i] >= pages) return "kv8 copy: a page outside the pool";
    if (count == 1) return from[0] == to[0] ? "kv8 copy: a page is both read and written" : nullptr;
    std::vector<int32_t> written(to, to + count);
    std::sort(written.begin(), written.end());
    for (int i = 1; i < count; ++i)
        if (written[i] == written[i - 1]) return "kv8 copy: a page is written twice";
    for (int i = 0; i < count; ++i)
        if (std::binary_search(written.begin(), written.end(), from[i])) return "kv8 copy: a page is both read and written";
    return nullptr;
}

// -------------------------------------------------------- draft verification
inline const char *check_verifier(int max_rows, int max_sequences, int vocab) {
    if (max_rows < 1 || max_rows > 65535) return "verify: rows 1 to 65535";
    if (max_sequences < 1 || max_sequences > 65535) return "verify: sequences 1 to 65535";
    if (vocab < 1 || vocab > (1 << 28)) return "verify: vocabulary 1 to 2^28";
    return nullptr;
}

// Tokens a workgroup takes of a row: 4096, or 1024 where that leaves fewer than
// two workgroups a CU.
inline int verify_chunk(int max_rows, int vocab) {
    return static_cast<int64_t>(max_rows) * ((vocab + 4095) / 4096) >= 512 ? 4096 : 1024;
}

inline const char *check_verify(int max_rows, int max_sequences, int vocab, int dtype, const void *target,
    int64_t target_pitch, const void *draft, int64_t draft_pitch, const void *tokens, const void *uniforms,
    const void *temperatures, int sequences, const void *row_starts, int rows, const void *emitted, const void *accepted,
    const void *logprobs) {
    if (!dtype_ok(dtype)) return "verify: unknown dtype";
    if (sequences < 0 || sequences > max_sequences || rows < 0 || rows > max_rows)
        return "verify: more rows or sequences than the verifier was made for";
    if (sequences == 0) return nullptr;
    if (!row_starts || !accepted || (rows > 0 && (!target || !tokens || !uniforms || !emitted))) return "verify: null array";
    const size_t e = dtype_bytes(dtype);
    if (!aligned(target, e) || !aligned(draft, e) || !aligned(tokens, 8) || !aligned(uniforms, 4) ||
        !aligned(temperatures, 4) || !aligned(row_starts, 4) || !aligned(emitted, 8) || !aligned(accepted, 4) ||
        !aligned(logprobs, 4))
        return "verify: misaligned array";
    if (target_pitch < vocab || !pitch_ok(target_pitch) || (draft && (draft_pitch < vocab || !pitch_ok(draft_pitch))))
        return "verify: pitches from the vocabulary to 2^31";
    return nullptr;
}

}  // namespace fortai_hip
