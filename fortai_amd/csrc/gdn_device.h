// What the kernels of the delta rule over rows share (gdn_rows.hip, gdn_chunks.hip).
// Every number that comes from device memory (row starts, slots, counts) is brought
// into range before it is used.
#pragma once

#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "step_kernels.h"

namespace fortai_hip {

// A sequence's rows [begin, begin + count), its slot (-1: none of the cache's), how
// many of the slot's pending rows stand, and whether it begins anew.
struct GdnSequence {
    int begin, count, slot, stands;
    bool begins;
};

__device__ __forceinline__ GdnSequence gdn_sequence(const GdnRowsParams &p, int seq) {
    GdnSequence s;
    const int32_t *starts = p.batch.starts;
    int b = read_only(starts + seq), e = read_only(starts + seq + 1);
    b = min(max(b, 0), p.batch.rows);
    e = min(max(e, b), p.batch.rows);
    s.begin = b;
    s.count = min(e - b, p.batch.max_rows);
    s.slot = read_only(p.batch.slots + seq);
    if (s.slot < 0 || s.slot >= p.cache.slots) s.slot = -1;
    const int standing = p.batch.standing ? read_only(p.batch.standing + seq) : kGdnMaxPending;
    s.begins = standing < 0;
    s.stands = standing;  // to be brought into [0, pending rows] by the reader of the slot's count
    return s;
}

__device__ __forceinline__ int gdn_stands(const GdnRowsParams &p, const GdnSequence &s) {
    const int pending = min(max(p.cache.counts[s.slot], 0), p.cache.pending);
    return min(max(s.stands, 0), pending);
}

// x / (1 + exp(-x)).  The exponent is off by 2^-24 of x, which moves the result by at most
// 0.3 2^-24 of x: less than the convolution's own rounding of x does.
__device__ __forceinline__ float gdn_silu(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}

// ssm_a softplus(alpha + ssm_dt): the logarithm of a row's decay.  Below -256 the decay is nothing (fp32's last number
// is e^-103), and so it is at -256: sums over a chunk's rows keep every row's own decay behind one that forgets
// everything.  Sum and product are taken in 64 bits, where they stay finite (of numbers that are), and a NaN stays one.
__device__ __forceinline__ float gdn_log_decay(float a, float alpha, float dt) {
    const double x = static_cast<double>(alpha) + static_cast<double>(dt);
    const double log = a * (fmax(x, 0.0) + static_cast<double>(log1pf(expf(-fabsf(static_cast<float>(x))))));
    return log < -256.0 ? -256.0f : static_cast<float>(log);
}

// Whether a sum of squares may have left fp32 where the length has not, or be short of its smallest parts where epsilon is
// smaller still: then the numbers are brought near 1 first.
__device__ __forceinline__ bool gdn_length_is_lost(float sum, float eps) { return !(sum < 0x1p126f) | ((sum < 0x1p-90f) & (eps < 0x1p-44f)); }

__device__ __forceinline__ float gdn_sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// The inputs of a channel that a slot keeps, written by one thread: behind a sequence
// of rows that wait, the taps - 1 inputs before them and theirs; otherwise the last
// taps - 1.  In place, in ascending order, four or eight at a time: what is read lies at or behind
// what is written.
template <typename E, int AT_ONCE>
__device__ __forceinline__ void gdn_keep_some(const GdnRowsParams &p, const GdnSequence &s, float *window, const E *x, int from, int kept) {
    const int channels = p.cache.channels(), before = p.cache.taps - 1;
#pragma unroll 1
    for (int j = 0; j < kept; j += AT_ONCE) {
        float v[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int at = from + min(j + k, kept - 1);
            v[k] = 0.0f;
            if (at >= before) v[k] = static_cast<float>(x[static_cast<int64_t>(at - before) * p.qkv_row]);
            else if (!s.begins) v[k] = window[static_cast<int64_t>(s.stands + at) * channels];
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
            if (j + k < kept) window[static_cast<int64_t>(j + k) * channels] = v[k];
    }
}

template <typename E>
__device__ __forceinline__ void gdn_keep_inputs(const GdnRowsParams &p, const GdnSequence &s, bool waits, int channel) {
    const int before = p.cache.taps - 1;
    float *window = p.cache.inputs + static_cast<int64_t>(s.slot) * (before + p.cache.pending) * p.cache.channels() + channel;
    const E *x = static_cast<const E *>(p.qkv) + static_cast<int64_t>(s.begin) * p.qkv_row + channel;
    const int from = waits ? 0 : s.count, kept = before + (waits ? s.count : 0);
    if (kept <= 4) gdn_keep_some<E, 4>(p, s, window, x, from, kept);
    else gdn_keep_some<E, 8>(p, s, window, x, from, kept);
}

}  // namespace fortai_hip
