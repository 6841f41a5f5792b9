// Rules on the logits of a step's rows, before they are verified or drawn from.
//
//   n = how often the token is among the text's last `window` tokens
//   n > 0:  x = x > 0 ? x / repetition : x * repetition;  x -= n frequency + presence
//   x += bias;  tokens that the row's mask leaves out: -infinity
//
// The text of a row is its sequence's history and the step's tokens up to the row.
// A workgroup has a chunk of the vocabulary and a run of one sequence's rows: it
// counts the chunk's tokens in the text once, in LDS by their place in the chunk (no
// hashing, and integer sums, whose order does not matter), and from row to row adds
// the one token that comes and takes away the one that leaves the window, while the
// next row's logits are on their way.
//
// Bound by the bytes of the rows, by the first count of a long text (every chunk's workgroup
// reads it again, from L2) and, for one row, by a launch's latency.  33 rows of 248,320 of
// eight sequences in fp32 (67 MB) behind texts of up to 8000 tokens, with biases and masks:
// 22 us; one row of 16,384 5.0 us.
#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "step_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kRuleThreads = 256;

template <Dtype DT, bool VEC, int CHUNK>
__global__ __launch_bounds__(kRuleThreads) void logit_rules_kernel(LogitRulesParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kFours = CHUNK / (4 * kRuleThreads), kAtOnce = 16;
    __shared__ __align__(16) int counts[CHUNK];
    // the tokens that come and go with a row, from row0 + 1 on, as places in the chunk (-1: elsewhere)
    __shared__ int comes[kRuleThreads], goes[kRuleThreads];
    const int seq = blockIdx.y, first = blockIdx.x * CHUNK, thread = threadIdx.x;
    int begin = read_only(p.row_starts + seq), end = read_only(p.row_starts + seq + 1);
    begin = min(max(begin, 0), p.rows);
    end = min(max(end, begin), p.rows);
    // this workgroup's share of the rows
    const int parts = gridDim.z, part = blockIdx.z, share = (end - begin + parts - 1) / parts;
    const int row0 = begin + part * share, row1 = min(row0 + share, end);
    if (row0 >= row1) return;

    f32x4_t x[kFours];
    const auto load_row = [&](int row) {
        const E *at = static_cast<const E *>(p.logits) + static_cast<int64_t>(row) * p.logits_row + first;
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const int i = 4 * (f * kRuleThreads + thread);
            if (VEC ? first + i < p.vocab : first + i + 3 < p.vocab) {
                x[f] = load4<DT, VEC>(at + i);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[f][k] = first + i + k < p.vocab ? static_cast<float>(at[i + k]) : 0.0f;
            }
        }
    };
    load_row(row0);
    // the chunk's biases, the same for every row, and the next row's mask, whose number is known a row before
    const bool biased = p.bias != nullptr;
    f32x4_t biases[kFours];
    if (biased) {
        const float *at = p.bias + seq * p.bias_pitch + first;
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const int i = 4 * (f * kRuleThreads + thread);
            biases[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (VEC) {
                if (first + i < p.vocab) biases[f] = *reinterpret_cast<const f32x4_t *>(at + i);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (first + i + k < p.vocab) biases[f][k] = at[i + k];
            }
        }
    }
    uint32_t words[kFours];
    const auto mask_number = [&](int row) { return p.masks ? read_only(p.mask_of + min(row, row1 - 1)) : -1; };
    const auto load_words = [&](int number) {
        const bool held = number >= 0 && number < p.mask_count;
        const uint32_t *allowed = p.masks + (held ? number * p.mask_pitch : 0);
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const int i = first + 4 * (f * kRuleThreads + thread);
            words[f] = ~0u;
            if (held && i < p.vocab) words[f] = allowed[i >> 5] >> (i & 31);
        }
    };
    load_words(mask_number(row0));
    int next_number = mask_number(row0 + 1);

    const bool counting = p.penalties != nullptr;
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    int64_t length = 0;  // of the history
    const int64_t *history = nullptr;
    const auto token_at = [&](int64_t place) { return place < length ? history[place] : p.tokens[begin + (place - length)]; };
    // x / repetition where x is positive, by the reciprocal and what is left of x then: the quotient to its last place
    // without a division each (divisions took 2 us of 27)
    float inverse = 1.0f;
    const auto repeated = [&](float x) {
        const float q = x * (x > 0.0f ? inverse : repetition), left = __builtin_fmaf(-q, repetition, x);
        const float quotient = __builtin_fmaf(left, inverse, q);
        return x > 0.0f && fabsf(quotient) < __builtin_inff() ? quotient : q;
    };
    const auto place_of = [&](int64_t token) {
        const int64_t at = token - first;
        return at >= 0 && at < CHUNK && token < p.vocab ? static_cast<int>(at) : -1;
    };
    const auto text_end = [&](int row) { return length + (p.tokens ? row - begin + 1 : 0); };
    // a thread's row of the next kRuleThreads
    const auto note_tokens = [&](int from_row) {
        const int row = from_row + thread;
        comes[thread] = goes[thread] = -1;
        if (!p.tokens || row >= row1) return;
        const int64_t last = text_end(row);
        comes[thread] = place_of(token_at(last - 1));
        if (p.window > 0 && last > p.window) goes[thread] = place_of(token_at(last - 1 - p.window));
    };
    if (counting) {
        repetition = p.penalties[3 * seq];
        inverse = 1.0f / repetition;
        frequency = p.penalties[3 * seq + 1];
        presence = p.penalties[3 * seq + 2];
        if (p.history) {
            length = min(max(static_cast<int64_t>(p.history_lengths[seq]), static_cast<int64_t>(0)), p.history_pitch);
            history = p.history + seq * p.history_pitch;
        }
        const int64_t last = text_end(row0), from = p.window > 0 && last > p.window ? last - p.window : 0;
        int64_t token[kAtOnce];
        const auto load_tokens = [&](int64_t place) {
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) token[k] = place + k * kRuleThreads < last ? token_at(place + k * kRuleThreads) : -1;
        };
        load_tokens(from + thread);
        note_tokens(row0 + 1);
        for (int i = thread; i < CHUNK; i += kRuleThreads) counts[i] = 0;
        lds_barrier();
        for (int64_t place = from + thread; place < last; place += kAtOnce * kRuleThreads) {
            int at[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) at[k] = place_of(token[k]);
            load_tokens(place + kAtOnce * kRuleThreads);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k)
                if (at[k] >= 0) atomicAdd(&counts[at[k]], 1);
        }
        lds_barrier();
    }

#pragma unroll 1
    for (int row = row0; row < row1; ++row) {
        f32x4_t y[kFours];
#pragma unroll
        for (int f = 0; f < kFours; ++f) y[f] = x[f];
        uint32_t bits[kFours];
#pragma unroll
        for (int f = 0; f < kFours; ++f) bits[f] = words[f];
        if (row + 1 < row1) {
            load_row(row + 1);
            load_words(next_number);
            next_number = mask_number(row + 2);
        }
        E *to = static_cast<E *>(p.out) + static_cast<int64_t>(row) * p.out_row + first;
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const int i = 4 * (f * kRuleThreads + thread);
            if (first + i >= p.vocab) continue;
            if (counting) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int n = counts[i + k];
                    const float seen = repeated(y[f][k]) - static_cast<float>(n) * frequency - presence;
                    y[f][k] = n > 0 ? seen : y[f][k];
                }
            }
            const bool four = VEC || first + i + 3 < p.vocab;
            if (biased) y[f] += biases[f];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (!(bits[f] >> k & 1u)) y[f][k] = -__builtin_inff();
            if (four) {
                store4<DT, VEC>(to + i, y[f]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (first + i + k < p.vocab) to[i + k] = static_cast<E>(y[f][k]);
            }
        }
        if (counting && p.tokens && row + 1 < row1) {
            const int ahead = (row - row0) % kRuleThreads;
            lds_barrier();
            if (thread == 0) {
                if (comes[ahead] >= 0) ++counts[comes[ahead]];
                if (goes[ahead] >= 0) --counts[goes[ahead]];
            }
            lds_barrier();
            if (ahead == kRuleThreads - 1) {
                note_tokens(row + 2);
                lds_barrier();
            }
        }
    }
}

template <Dtype DT, bool VEC>
hipError_t rules_typed(const LogitRulesParams &p, hipStream_t stream) {
    // three rows of a sequence stay together, for which the text is counted once and whose rows follow each other:
    // eight sequences of up to five behind 8000 tokens (16) 21.6 us (18.2), five together 22.6 (21.7), two 23.5 (19.9), one
    // 26.0 (20.8)
    const int average = (p.rows + p.sequences - 1) / p.sequences, parts = (average + 2) / 3;
    const int64_t groups = static_cast<int64_t>(p.sequences) * parts;
    // chunks of 4096 where they fill the chip (33 rows of 248,320 21.5 us, of 1024 30.7), otherwise of 1024 (of the same
    // rows, behind as long a text: one 7.3 us against 9.1, four sequences' 9.2 against 9.6)
    if (groups * ((p.vocab + 4095) / 4096) >= 256)
        hipLaunchKernelGGL((logit_rules_kernel<DT, VEC, 4096>), dim3((p.vocab + 4095) / 4096, p.sequences, parts), dim3(kRuleThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((logit_rules_kernel<DT, VEC, 1024>), dim3((p.vocab + 1023) / 1024, p.sequences, parts), dim3(kRuleThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_logit_rules(const LogitRulesParams &p, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) return vec ? rules_typed<Dtype::F32, true>(p, stream) : rules_typed<Dtype::F32, false>(p, stream);
    if (dtype == Dtype::F16) return vec ? rules_typed<Dtype::F16, true>(p, stream) : rules_typed<Dtype::F16, false>(p, stream);
    return vec ? rules_typed<Dtype::BF16, true>(p, stream) : rules_typed<Dtype::BF16, false>(p, stream);
}

}  // namespace fortai_hip
