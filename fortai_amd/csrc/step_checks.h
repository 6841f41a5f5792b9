// Argument checks of the operators around a step's products, free of device code
// so that they also compile for the host alone.  A check returns what is wrong
// with the arguments, or nullptr.
#pragma once

#include "serving_checks.h"

namespace fortai_hip {

// ------------------------------------------- norm into 8-bit tokens, and back
struct NormTokensArrays {
    const void *x, *residual, *sum, *norm, *gate, *output, *tokens;
    int64_t x_pitch, residual_pitch, sum_pitch, gate_pitch, output_pitch;
};

inline const char *check_norm_tokens(int dtype, int rows, int width, int group, float epsilon, const NormTokensArrays &a) {
    if (!dtype_ok(dtype)) return "norm tokens: unknown dtype";
    if (rows < 0 || rows > kMaxRows) return "norm tokens: rows 0 to 2^23";
    if (width < 32 || width % 32 || width > (1 << 20)) return "norm tokens: width a multiple of 32, up to 2^20";
    if (group != width && ((group != 32 && group != 64 && group != 128 && group != 256) || width % group))
        return "norm tokens: groups of the whole width, or of 32, 64, 128 or 256 that divide it";
    if (a.norm && !(epsilon > 0.0f)) return "norm tokens: the norm needs epsilon > 0";
    if (rows == 0) return nullptr;
    if (!a.x || (!a.output && !a.tokens)) return "norm tokens: null array";
    const size_t e = dtype_bytes(dtype);
    if (!aligned(a.x, e) || !aligned(a.residual, e) || !aligned(a.sum, e) || !aligned(a.gate, e) || !aligned(a.output, e) ||
        !aligned(a.norm, 4) || !aligned(a.tokens, 16))
        return "norm tokens: misaligned array";
    if (!pitch_ok(a.x_pitch) || !pitch_ok(a.residual_pitch) || !pitch_ok(a.gate_pitch)) return "norm tokens: pitches 0 to 2^31";
    if (!pitch_ok(a.sum_pitch) || !pitch_ok(a.output_pitch) || (rows > 1 && a.sum && a.sum_pitch < width) ||
        (rows > 1 && a.output && a.output_pitch < width))
        return "norm tokens: output pitches from the width to 2^31";
    if ((a.sum && a.sum == a.x && rows > 1 && a.sum_pitch != a.x_pitch) ||
        (a.sum && a.sum == a.residual && rows > 1 && a.sum_pitch != a.residual_pitch))
        return "norm tokens: in place, both sides have the same pitch";
    return nullptr;
}

inline const char *check_tokens_read(int dtype, int rows, int width, const void *tokens, const void *output, int64_t output_pitch) {
    if (!dtype_ok(dtype)) return "tokens read: unknown dtype";
    if (rows < 0 || rows > kMaxRows) return "tokens read: rows 0 to 2^23";
    if (width < 32 || width % 32 || width > (1 << 20)) return "tokens read: width a multiple of 32, up to 2^20";
    if (rows == 0) return nullptr;
    if (!tokens || !output) return "tokens read: null array";
    if (!aligned(tokens, 16) || !aligned(output, dtype_bytes(dtype))) return "tokens read: misaligned array";
    if (!pitch_ok(output_pitch) || (rows > 1 && output_pitch < width)) return "tokens read: output pitch from the width to 2^31";
    return nullptr;
}

// ------------------------------------------------------------- logits' rules
struct LogitRulesArrays {
    const void *logits, *row_starts, *tokens, *history, *history_lengths, *penalties, *bias, *masks, *mask_of, *output;
    int64_t logits_pitch, history_pitch, bias_pitch, mask_pitch, output_pitch;
};

inline const char *check_logit_rules(int dtype, int rows, int vocab, int sequences, int window, int mask_count,
    const LogitRulesArrays &a) {
    if (!dtype_ok(dtype)) return "logits: unknown dtype";
    if (rows < 0 || rows > 65535 || sequences < 0 || sequences > 65535) return "logits: rows and sequences 0 to 65535";
    if (vocab < 1 || vocab > (1 << 28)) return "logits: vocabulary 1 to 2^28";
    if (window < 0) return "logits: window below 0";
    if (rows == 0 || sequences == 0) return nullptr;
    if (!a.logits || !a.output || !a.row_starts) return "logits: null array";
    if (a.history && !a.history_lengths) return "logits: a history has lengths";
    if (a.masks && !a.mask_of) return "logits: masks have an array that says which row has which";
    const size_t e = dtype_bytes(dtype);
    if (!aligned(a.logits, e) || !aligned(a.output, e) || !aligned(a.row_starts, 4) || !aligned(a.tokens, 8) ||
        !aligned(a.history, 8) || !aligned(a.history_lengths, 4) || !aligned(a.penalties, 4) || !aligned(a.bias, 4) ||
        !aligned(a.masks, 4) || !aligned(a.mask_of, 4))
        return "logits: misaligned array";
    if (a.logits_pitch < vocab || !pitch_ok(a.logits_pitch) || a.output_pitch < vocab || !pitch_ok(a.output_pitch))
        return "logits: pitches from the vocabulary to 2^31";
    if (a.history && (a.history_pitch < 0 || a.history_pitch > (1 << 30))) return "logits: history pitch 0 to 2^30";
    if (a.bias && a.bias_pitch != 0 && (a.bias_pitch < vocab || !pitch_ok(a.bias_pitch)))
        return "logits: bias pitch 0, or from the vocabulary to 2^31";
    if (a.masks && (mask_count < 0 || a.mask_pitch < (vocab + 31) / 32 || !pitch_ok(a.mask_pitch)))
        return "logits: mask pitch from the vocabulary's words to 2^31";
    if (a.logits == a.output && rows > 1 && a.logits_pitch != a.output_pitch) return "logits: in place, both sides have the same pitch";
    return nullptr;
}

// ----------------------------------------------------- the delta rule's cache
struct GdnShape {
    int layers = 0, slots = 0, key_heads = 0, value_heads = 0, head = 0, taps = 0, pending = 0;
    size_t channels() const { return (2 * static_cast<size_t>(key_heads) + value_heads) * head; }
    // floats of a slot in the planes states, inputs, keys, updates, decays, counts
    size_t plane(int i) const {
        const size_t d = head, p = pending;
        const size_t floats[6] = {value_heads * d * d, (taps - 1 + p) * channels(), p * key_heads * d, p * value_heads * d,
            p * value_heads, 1};
        return floats[i];
    }
    size_t slot() const {
        size_t n = 0;
        for (int i = 0; i < 6; ++i) n += plane(i);
        return n;
    }
};

inline const char *check_gdn_shape(const GdnShape &s) {
    if (s.layers < 1 || s.layers > 4096 || s.slots < 1) return "gdn: layers 1 to 4096, slots from 1";
    if (s.key_heads < 1 || s.key_heads > 1024 || s.value_heads < 1 || s.value_heads > 1024 || s.value_heads % s.key_heads)
        return "gdn: heads 1 to 1024, value heads a multiple of key heads";
    if (s.head != 64 && s.head != 128) return "gdn: heads of 64 or 128";
    if (s.taps < 2 || s.taps > 8) return "gdn: convolutions of 2 to 8";
    if (s.pending < 0 || s.pending > 16) return "gdn: pending rows 0 to 16";
    return nullptr;  // at most 2^12 layers of 2^31 slots of 2^25 floats: gdn_bytes() says which do not fit
}

// 0 where 64 bits do not hold it (no storage is that large)
inline size_t gdn_bytes(const GdnShape &s) {
    if (check_gdn_shape(s)) return 0;
    const double about = 4.0 * s.layers * s.slots * static_cast<double>(s.slot());
    return about < 9.0e15 ? 4 * static_cast<size_t>(s.layers) * s.slots * s.slot() : 0;
}

inline const char *check_gdn_rows(int max_rows) {
    return max_rows < 1 || max_rows > (1 << 19) ? "gdn: rows 1 to 2^19" : nullptr;
}

inline const char *check_gdn_batch(int sequences, int rows, int max_rows, int most, const void *starts, const void *slots,
    const void *standing) {
    if (sequences < 0 || sequences > 16384) return "gdn: sequences 0 to 16384";
    if (rows < 0 || rows > most) return "gdn: more rows than the cache was made for";
    if (max_rows < 0 || max_rows > rows) return "gdn: max_rows 0 to rows";
    if (sequences == 0 || rows == 0 || max_rows == 0) return nullptr;
    if (!starts || !slots) return "gdn: null array";
    if (!aligned(starts, 4) || !aligned(slots, 4) || !aligned(standing, 4)) return "gdn: misaligned array";
    return nullptr;
}

struct GdnArrays {
    const void *qkv, *alpha, *beta, *conv, *ssm_a, *ssm_dt, *output;
    int64_t qkv_pitch, alpha_pitch, beta_pitch, output_pitch;
};

inline const char *check_gdn_run(const GdnShape &s, int layer, int dtype, int rows, float epsilon, const GdnArrays &a) {
    if (layer < 0 || layer >= s.layers) return "gdn: no such layer";
    if (!dtype_ok(dtype)) return "gdn: unknown dtype";
    if (!(epsilon > 0.0f)) return "gdn: epsilon above 0";
    if (!a.qkv || !a.alpha || !a.beta || !a.conv || !a.ssm_a || !a.ssm_dt || !a.output) return "gdn: null array";
    const size_t e = dtype_bytes(dtype);
    if (!aligned(a.qkv, e) || !aligned(a.alpha, e) || !aligned(a.beta, e) || !aligned(a.output, e) || !aligned(a.conv, 4) ||
        !aligned(a.ssm_a, 4) || !aligned(a.ssm_dt, 4))
        return "gdn: misaligned array";
    if (!pitch_ok(a.qkv_pitch) || !pitch_ok(a.alpha_pitch) || !pitch_ok(a.beta_pitch)) return "gdn: pitches 0 to 2^31";
    if (!pitch_ok(a.output_pitch) || (rows > 1 && a.output_pitch < static_cast<int64_t>(s.value_heads) * s.head))
        return "gdn: output pitch from value_heads * head to 2^31";
    return nullptr;
}

// Pairs that can be copied in any order: ids below `count_of`, none written twice, none
// both read and written.  May throw std::bad_alloc.
inline const char *check_slot_pairs(const int32_t *from, const int32_t *to, int count, int count_of) {
    return check_page_pairs(from, to, count, count_of) ? "gdn copy: a slot outside the cache, written twice, or both read and written"
                                                       : nullptr;
}

}  // namespace fortai_hip
