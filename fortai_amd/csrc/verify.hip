// Verification of drafted tokens against the target's distribution, from given
// random numbers.
//
// Row i of a sequence has the target's logits after the step's token i, and (i <
// drafts) the distribution that draft x_i = tokens[i + 1] was drawn from.  With
// p = softmax(target / T) and q = softmax(draft / T), x_i stands while
//   u_i q(x_i) < p(x_i).
// At the first row that does not, one token is drawn from max(p - q, 0); if all
// stand, from the last row's p; by inverse CDF: the lowest token whose cumulative
// weight exceeds u times the total.  T <= 0 takes the argmax instead.  The tokens
// that this emits are distributed as the target's own.
//
// Everything that decides is in 64 bits: with 250,000 tokens a cumulative weight
// that is off by 10^-7 would cross a token's border in one of twenty draws.
//
// Three launches, joined at kernel boundaries: (1) each row's maximum, its first
// token and sum of exponentials, by chunks of the vocabulary; (2) for each
// sequence the row that decides, worked out again by every workgroup from the
// chunks' sums, and the weights of that row summed by chunk; (3) the chunk, the
// token and the outputs.  Bound by reading the logits once, and about as much by
// the exponentials in 64 bits: eight sequences of up to five rows of 248,320 tokens
// with their drafts' logits, 58 MB, take 21 + 10 + 8.5 us under a trace, 37 back to back;
// five rows of 16,384 tokens 13.2 us.
#include "fortai_hip_internal.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr float kLargest = 3.402823466e38f;
constexpr float kHottest = 1e9f;  // above it the weight of what is masked would have to be told from 2^-1000

// NaN counts as -infinity, +infinity as the largest number.
__device__ __forceinline__ float logit(float x) { return x != x ? -__builtin_inff() : fminf(x, kLargest); }

// exp((x - top) / T) of a row as 2^(d c), d = x - top exactly (the difference of two
// fp32 numbers), c = log2(e) / T, to 1.9e-14: d c = n + r with |r| <= 1/2, and the
// polynomial of degree 9 that equals 2^r at the ten Chebyshev nodes.  Adding
// 1.5 * 2^52 leaves n in the sum's low bits, from where it goes into the exponent.
struct RowExp {
    double c, top, least;
    __device__ __forceinline__ RowExp(float row_top, double per_t)
        : c(per_t), top(static_cast<double>(row_top)), least(-1000.0 / per_t) {}
    // x <= top, or NaN: 2^-1000 for what lies lower, -infinity and NaN among it
    __device__ __forceinline__ double raw(float x) const {
        const double shift = 6755399441055744.0;
        const double d = fmax(static_cast<double>(x) - top, least);
        const double k = __builtin_fma(d, c, shift);
        const double r = __builtin_fma(d, c, shift - k);
        double y = 0x1.b6571de2f2351p-24;
        y = __builtin_fma(y, r, 0x1.63ef969a64d3cp-20);
        y = __builtin_fma(y, r, 0x1.ffcb76789860fp-17);
        y = __builtin_fma(y, r, 0x1.43088e257f341p-13);
        y = __builtin_fma(y, r, 0x1.5d87fe908f88ap-10);
        y = __builtin_fma(y, r, 0x1.3b2ab72b175eep-7);
        y = __builtin_fma(y, r, 0x1.c6b08d7044119p-5);
        y = __builtin_fma(y, r, 0x1.ebfbdff8149f2p-3);
        y = __builtin_fma(y, r, 0x1.62e42fefa39f7p-1);
        y = __builtin_fma(y, r, 0x1.000000000003dp+0);
        return __builtin_ldexp(y, static_cast<int>(__builtin_bit_cast(uint2, k).x));
    }
    // No weight for what lies lower than 2^-1000, as far as 64 bits tell it from nothing: -infinity, and masks
    // by the type's lowest number, which a draw at u = 0 would otherwise find.
    __device__ __forceinline__ double operator()(float x) const {
        return static_cast<double>(x) - top > least ? raw(x) : 0.0;
    }
};

__device__ __forceinline__ void sequence_rows(const VerifyParams &p, int seq, int *begin, int *end) {
    int b = p.row_starts[seq], e = p.row_starts[seq + 1];
    b = min(max(b, 0), p.rows);
    e = min(max(e, b), p.rows);
    *begin = b;
    *end = e;
}

__device__ __forceinline__ float temperature(const VerifyParams &p, int seq) {
    return p.temperatures ? p.temperatures[seq] : 1.0f;
}
__device__ __forceinline__ double inverse_temperature(float t) {
    return t > 0.0f ? 1.0 / static_cast<double>(fminf(t, kHottest)) : 1.0;
}
constexpr double kLog2e = 1.4426950408889634074;

// the larger value, the lower index among equals
__device__ __forceinline__ void take_larger(float &v, int &i, float w, int j) {
    i = w > v ? j : w == v ? min(i, j) : i;
    v = fmaxf(v, w);
}

__device__ __forceinline__ void wave_larger(float &v, int &i) {
    take_larger(v, i, xor_lane<32>(v), xor_lane<32>(i));
    take_larger(v, i, xor_lane<16>(v), xor_lane<16>(i));
    take_larger(v, i, xor_lane<8>(v), xor_lane<8>(i));
    take_larger(v, i, xor_lane<4>(v), xor_lane<4>(i));
    take_larger(v, i, xor_lane<2>(v), xor_lane<2>(i));
    take_larger(v, i, xor_lane<1>(v), xor_lane<1>(i));
}

__device__ __forceinline__ int wave_least(int v) {
    v = min(v, xor_lane<32>(v));
    v = min(v, xor_lane<16>(v));
    v = min(v, xor_lane<8>(v));
    v = min(v, xor_lane<4>(v));
    v = min(v, xor_lane<2>(v));
    return min(v, xor_lane<1>(v));
}
__device__ __forceinline__ int wave_most(int v) { return -wave_least(-v); }

// ---------------------------------------------------------------- (1) rows
// EACH: groups of four logits a thread holds (chunk = 1024 EACH)
template <Dtype DT, int EACH, bool VEC>
__device__ __forceinline__ void load_chunk(const typename Element<DT>::type *x, int chunk, int vocab, float (&v)[EACH][4]) {
    const float none = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int at = (chunk * EACH + k) * kVerifyThreads * 4 + static_cast<int>(threadIdx.x) * 4;
        if constexpr (VEC) {  // the vocabulary is a multiple of four
            const f32x4_t y = at < vocab ? load4<DT, true>(x + at) : f32x4_t{none, none, none, none};
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = y[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = at + i < vocab ? static_cast<float>(x[at + i]) : none;
        }
    }
}

// A workgroup walks every gridDim.x-th chunk of a row, the next one in flight.
template <Dtype DT, int EACH, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_rows_kernel(VerifyParams p) {
    typedef typename Element<DT>::type E;
    __shared__ int found;
    __shared__ float tops[kVerifyWaves];
    __shared__ int places[kVerifyWaves];
    __shared__ double sums[kVerifyWaves];
    const int row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool draft = blockIdx.z != 0;
    const E *x = static_cast<const E *>(draft ? p.draft : p.target) +
        static_cast<int64_t>(row) * (draft ? p.draft_pitch : p.target_pitch);
    float next[EACH][4];
    load_chunk<DT, EACH, VEC>(x, blockIdx.x, p.vocab, next);
    // the row's sequence: its temperature, and whether it is a row with a draft
    if (threadIdx.x == 0) found = p.sequences;
    __syncthreads();
    for (int s = threadIdx.x; s < p.sequences; s += kVerifyThreads) {
        int begin, end;
        sequence_rows(p, s, &begin, &end);
        if (row >= begin && row < end - (draft ? 1 : 0)) atomicMin(&found, s);
    }
    __syncthreads();
    const int seq = found;
    if (seq >= p.sequences) return;
    const float t = temperature(p, seq);
    const double per_t = inverse_temperature(t) * kLog2e;
#pragma unroll 1
    for (int chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
        float v[EACH][4];
#pragma unroll
        for (int k = 0; k < EACH; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = next[k][i];
        if (chunk + static_cast<int>(gridDim.x) < p.chunks) load_chunk<DT, EACH, VEC>(x, chunk + gridDim.x, p.vocab, next);
        // fmaxf passes over NaN, and so do the exponentials
        float top = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < EACH; ++k) top = fmaxf(top, fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])));
        top = wave_max(top);
        if (lane == 0) tops[wave] = top;
        lds_barrier();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        if (top > kLargest) {
            top = kLargest;
#pragma unroll
            for (int k = 0; k < EACH; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k][i] = logit(v[k][i]);
        }
        if (!(t > 0.0f)) {  // only the argmax asks which token it is
            int place = 0x7fffffff;
#pragma unroll
            for (int k = EACH - 1; k >= 0; --k)
#pragma unroll
                for (int i = 3; i >= 0; --i)
                    place = v[k][i] >= top ? (chunk * EACH + k) * kVerifyThreads * 4 + static_cast<int>(threadIdx.x) * 4 + i : place;
            place = wave_least(place);
            if (lane == 0) places[wave] = place;
        }
        double sum = 0.0;
        if (top > -__builtin_inff()) {
            // a logit of -infinity adds 2^-1000 to a sum of at least one: nothing
            const RowExp e(top, per_t);
#pragma unroll
            for (int k = 0; k < EACH; ++k)
                sum += (e.raw(v[k][0]) + e.raw(v[k][1])) + (e.raw(v[k][2]) + e.raw(v[k][3]));
        }
        sum = wave_sum(sum);
        if (lane == 0) sums[wave] = sum;
        lds_barrier();
        if (threadIdx.x == 0) {
            VerifyPart part;
            part.sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
            part.top = top;
            part.place = !(t > 0.0f) ? min(min(places[0], places[1]), min(places[2], places[3])) : 0;
            p.parts[(static_cast<size_t>(draft ? p.max_rows : 0) + row) * p.chunks + chunk] = part;
        }
    }
}

// -------------------------------------------------- (2) the deciding row
// The kernels of (2) and (3) run a few workgroups once: what they wait for is
// memory and, cold, their own code.  Loops over rows, over target and draft and
// over groups of tokens are kept rolled, which is faster here than unrolled
// (a finish of 21 KB of straight code took 14 us, of 6 KB 8 us).
__device__ __forceinline__ VerifyPart row_part(const VerifyParams &p, int row, bool draft, int c) {
    if (c >= p.chunks) return VerifyPart{0.0, -__builtin_inff(), 0x7fffffff};
    return p.parts[(static_cast<size_t>(draft ? p.max_rows : 0) + row) * p.chunks + c];
}

// first: row_part of chunk `lane`
__device__ __forceinline__ VerifyRow row_stats(const VerifyParams &p, int row, bool draft, const VerifyPart &first, double per_t) {
    const int lane = threadIdx.x & 63;
    VerifyRow r = {0.0, first.top, first.place};
#pragma unroll 1
    for (int c = lane + 64; c < p.chunks; c += 64) {
        const VerifyPart part = row_part(p, row, draft, c);
        take_larger(r.top, r.place, part.top, part.place);
    }
    wave_larger(r.top, r.place);
    const RowExp e(r.top, per_t);
    VerifyPart part = first;
#pragma unroll 1
    for (int c = lane; c < p.chunks; c += 64) {
        if (c > lane) part = row_part(p, row, draft, c);
        r.sum += part.sum * e(part.top);
    }
    r.sum = wave_sum(r.sum);
    return r;
}

template <Dtype DT>
__device__ __forceinline__ float logit_at(const void *logits, int64_t pitch, int row, int64_t token) {
    return logit(static_cast<float>(static_cast<const typename Element<DT>::type *>(logits)[static_cast<int64_t>(row) * pitch + token]));
}

// log(s) for s >= 1: s = 2^e m with m in [1/2, 1) doubled below sqrt(1/2), and
// log m = 2 atanh z, z = (m - 1) / (m + 1), |z| < 0.172: the series to z^17 is off by 1e-15.
__device__ __forceinline__ double log_above(double s) {
    int e = __builtin_amdgcn_frexp_exp(s);
    double m = __builtin_amdgcn_frexp_mant(s);
    if (m < 0.70710678118654752440) {
        m += m;
        --e;
    }
    const double z = (m - 1.0) / (m + 1.0), q = z * z;
    double y = 1.0 / 17.0;
    y = __builtin_fma(y, q, 1.0 / 15.0);
    y = __builtin_fma(y, q, 1.0 / 13.0);
    y = __builtin_fma(y, q, 1.0 / 11.0);
    y = __builtin_fma(y, q, 1.0 / 9.0);
    y = __builtin_fma(y, q, 1.0 / 7.0);
    y = __builtin_fma(y, q, 1.0 / 5.0);
    y = __builtin_fma(y, q, 1.0 / 3.0);
    y = __builtin_fma(y, q, 1.0);
    return __builtin_fma(static_cast<double>(e), 0.69314718055994530942, 2.0 * z * y);
}

__device__ __forceinline__ double inverse_sum(const VerifyRow &row) { return row.sum > 0.0 ? 1.0 / row.sum : 0.0; }

// Every thread of a workgroup of WAVES waves; a wave a row, WAVES rows at a time.
// write: the rows' statistics are kept for the finish.
template <Dtype DT, int WAVES>
__device__ __forceinline__ VerifyDecision decide(const VerifyParams &p, int seq, bool write) {
    __shared__ int stands[WAVES];
    __shared__ VerifyRow kept[WAVES][2];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int begin, end;
    sequence_rows(p, seq, &begin, &end);
    VerifyDecision d;
    d.begin = begin;
    d.end = end;
    d.row = -1;
    d.rejected = -1;
    d.against_draft = 0;
    d.uniform = end > begin ? static_cast<double>(p.uniforms[end - 1]) : 0.0;
    d.target = d.draft = VerifyRow{0.0, 0.0f, 0};
    const float t = temperature(p, seq);
    const double per_t = inverse_temperature(t) * kLog2e;
#pragma unroll 1
    for (int first = begin; first < end && d.row < 0; first += WAVES) {
        const int row = first + wave;
        if (row < end) {
            const bool has_draft = row + 1 < end, two = p.draft && has_draft;
            VerifyPart part = row_part(p, row, false, lane), draft_part = part;
            if (two) draft_part = row_part(p, row, true, lane);
            const int64_t x = has_draft ? p.tokens[row + 1] : -1;
            const bool judged = x >= 0 && x < p.vocab;
            const float u = p.uniforms[row];
            const float lp = judged ? logit_at<DT>(p.target, p.target_pitch, row, x) : 0.0f;
            const float lq = judged && p.draft ? logit_at<DT>(p.draft, p.draft_pitch, row, x) : 0.0f;
            double px = 0.0, qx = 1.0;
            bool best = false;
#pragma unroll 1
            for (int s = 0; s < (two ? 2 : 1); ++s) {
                const VerifyRow r = row_stats(p, row, s != 0, part, per_t);
                part = draft_part;
                if (lane == 0) kept[wave][s] = r;
                const double share = RowExp(r.top, per_t)(s ? lq : lp) * inverse_sum(r);
                if (s == 0) {
                    px = share;
                    best = r.sum > 0.0 && x == r.place;
                    if (write && lane == 0) p.row_stats[row] = r;
                } else {
                    qx = share;
                }
            }
            if (lane == 0) stands[wave] = judged && (t > 0.0f ? static_cast<double>(u) * qx < px : best);
        }
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < WAVES && first + w < end && d.row < 0; ++w)
            if (!stands[w]) {  // a sequence's last row never stands, so some row does not
                d.row = first + w;
                d.target = kept[w][0];
                if (p.draft && d.row + 1 < end) d.draft = kept[w][1];
            }
        __syncthreads();
    }
    if (d.row >= 0 && d.row + 1 < end) {
        const int64_t x = p.tokens[d.row + 1];
        d.against_draft = 1;
        d.rejected = x >= 0 && x < p.vocab ? static_cast<int>(x) : -1;
    }
    return d;
}

// What a token weighs in the draw: p, or what p has over q.
template <Dtype DT, bool VEC>
struct DrawWeights {
    typedef typename Element<DT>::type E;
    const E *target, *draft;
    RowExp te, qe;
    double per_target, per_draft;  // 1 / sum, 0 for a row without weight
    int certain;                   // the draft that counts as certain, or -1

    __device__ __forceinline__ DrawWeights(const VerifyParams &p, const VerifyDecision &d, bool left, double per_t)
        : target(static_cast<const E *>(p.target) + static_cast<int64_t>(d.row) * p.target_pitch),
          draft(left && p.draft ? static_cast<const E *>(p.draft) + static_cast<int64_t>(d.row) * p.draft_pitch : nullptr),
          te(d.target.top, per_t), qe(d.draft.top, per_t), per_target(inverse_sum(d.target)),
          per_draft(inverse_sum(d.draft)), certain(left && !p.draft ? d.rejected : -1) {}

    __device__ __forceinline__ f32x4_t logits(const E *row, int at, int until) const {
        if constexpr (VEC) {  // until is a multiple of four
            return at < until ? load4<DT, true>(row + at) : f32x4_t{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        } else {
            f32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = at + i < until ? static_cast<float>(row[at + i]) : -__builtin_inff();
            return x;
        }
    }
    // four tokens from `at` on, those before `until`
    __device__ __forceinline__ void get(int at, int until, double (&w)[4]) const {
        const f32x4_t x = logits(target, at, until);
        f32x4_t y = x;
        if (draft) y = logits(draft, at, until);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = te(logit(x[i])) * per_target;
        if (draft) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = fmax(w[i] - qe(logit(y[i])) * per_draft, 0.0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = at + i == certain ? 0.0 : w[i];
    }
};

template <Dtype DT, int THREADS, bool VEC>
__global__ __launch_bounds__(THREADS) void verify_weights_kernel(VerifyParams p) {
    constexpr int kW = THREADS / 64;
    __shared__ double sums[kW];
    const int seq = blockIdx.y;
    const float t = temperature(p, seq);
    // where the argmax is taken one workgroup decides, and nothing is weighed
    if (!(t > 0.0f) && blockIdx.x > 0) return;
    const VerifyDecision d = decide<DT, kW>(p, seq, blockIdx.x == 0);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.decisions[seq] = d;
        p.accepted[seq] = d.row < 0 ? 0 : d.row - d.begin;
    }
    if (!(t > 0.0f) || d.row < 0 || !d.against_draft) return;  // p's own chunk sums are known
    const DrawWeights<DT, VEC> weights(p, d, true, inverse_temperature(t) * kLog2e);
    const int until = min((static_cast<int>(blockIdx.x) + 1) * p.chunk, p.vocab);
    double sum = 0.0;
#pragma unroll 2
    for (int at = blockIdx.x * p.chunk + static_cast<int>(threadIdx.x) * 4; at < until; at += THREADS * 4) {
        double w[4];
        weights.get(at, until, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = sums[0];
#pragma unroll
        for (int k = 1; k < kW; ++k) sum += sums[k];
        p.weights[static_cast<size_t>(seq) * p.chunks + blockIdx.x] = sum;
    }
}

// sum over the lanes up to and including this one
__device__ __forceinline__ double wave_prefix(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int d = 1; d < 64; d <<= 1) {
        const double below = __shfl_up(v, d);
        v += lane >= d ? below : 0.0;
    }
    return v;
}

// ------------------------------------------------------- (3) the token
// THREADS x 4 tokens are a chunk of the vocabulary.
template <Dtype DT, int THREADS, bool VEC>
__global__ __launch_bounds__(THREADS) void verify_finish_kernel(VerifyParams p) {
    constexpr int kW = THREADS / 64;
    __shared__ double waves[kW];
    __shared__ int chosen[kW], last[kW], chunk_at;
    __shared__ double below_at, border_at;
    const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double *chunk_weights = p.weights + static_cast<size_t>(seq) * p.chunks;
    // the first chunks' weights are fetched before it is known whether they count
    const double early = lane < p.chunks ? chunk_weights[lane] : 0.0;
    const float t = temperature(p, seq);
    const VerifyDecision d = p.decisions[seq];
    if (d.row < 0) return;  // no rows
    // what the outputs need beside the token, in flight meanwhile
    const int out_row = d.begin + static_cast<int>(threadIdx.x);
    const int64_t stands = out_row < d.row ? p.tokens[out_row + 1] : -1;
    const VerifyRow out_stats = out_row <= d.row ? p.row_stats[out_row] : VerifyRow{1.0, 0.0f, 0};
    const double inverse_t = inverse_temperature(t), per_t = inverse_t * kLog2e;
    int token = -1;
    if (!(t > 0.0f)) {
        token = d.target.sum > 0.0 ? d.target.place : -1;
    } else {
        // p where nothing is left of it over q, which a draft of probability zero can leave
        bool left = d.against_draft != 0;
        if (wave == 0) {
            const VerifyPart *parts = p.parts + static_cast<size_t>(d.row) * p.chunks;
            const RowExp e(d.target.top, per_t);
            const double per_target = inverse_sum(d.target);
            double total = 0.0, below = 0.0, best_below = 0.0;
            int best = -1;
            // twice over the chunks: their total, then the first whose end lies over u total, else the
            // last that weighs anything; a third and fourth time for p alone
#pragma unroll 1
            for (int pass = 0; pass < 4; ++pass) {
                const bool adding = (pass & 1) == 0;
                if (pass == 2) left = false;
                below = 0.0;
                bool over = false;
#pragma unroll 1
                for (int c0 = 0; c0 < p.chunks && !over; c0 += 64) {
                    const int c = c0 + lane;
                    double w = 0.0;
                    if (c < p.chunks) w = left ? (c < 64 ? early : chunk_weights[c]) : parts[c].sum * e(parts[c].top) * per_target;
                    const double end = below + wave_prefix(w);
                    if (!adding) {
                        const uint64_t some = __ballot(w > 0.0), past = __ballot(w > 0.0 && end > d.uniform * total);
                        if (some) {
                            const int k = past ? __ffsll(static_cast<unsigned long long>(past)) - 1
                                               : 63 - __clzll(static_cast<long long>(some));
                            best = c0 + k;
                            best_below = __shfl(end - w, k);
                            over = past != 0;
                        }
                    }
                    below = __shfl(end, 63);
                }
                if (!adding) break;
                total = below;
                if (!(total > 0.0)) {
                    if (!left) break;
                    ++pass;
                }
            }
            if (lane == 0) {
                chunk_at = best < 0 ? -1 : left ? best : best + p.chunks;  // past the chunks: p alone
                below_at = best_below;
                border_at = d.uniform * total;
            }
        }
        __syncthreads();
        int at = chunk_at;
        if (at >= p.chunks) {
            at -= p.chunks;
            left = false;
        }
        if (at >= 0) {
            const DrawWeights<DT, VEC> draw(p, d, left, per_t);
            const int until = min((at + 1) * p.chunk, p.vocab), from = at * p.chunk + static_cast<int>(threadIdx.x) * 4;
            double w[4];
            draw.get(from, until, w);
            const double prefix = wave_prefix((w[0] + w[1]) + (w[2] + w[3]));
            if (lane == 63) waves[wave] = prefix;
            __syncthreads();
            double before = below_at;
#pragma unroll 1
            for (int v = 0; v < wave; ++v) before += waves[v];
            // Sums in another order may differ in their last places, also where a thread's tokens weigh
            // nothing: a thread offers only tokens that do, and every thread that ends past the border
            // offers one (its last where rounding hides the first), so that the lowest offered is the token.
            const double border = border_at, upto = before + prefix;
            double c = __shfl_up(upto, 1);
            if (lane == 0) c = before;
            int first = 0x7fffffff, end = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c += w[i];
                end = w[i] > 0.0 ? from + i : end;
                first = w[i] > 0.0 && c > border ? min(first, from + i) : first;
            }
            if (first > end) first = upto > border && end >= 0 ? end : 0x7fffffff;
            // the lowest token found, else the last that weighs anything
            first = wave_least(first);
            end = wave_most(end);
            if (lane == 0) {
                chosen[wave] = first;
                last[wave] = end;
            }
            __syncthreads();
#pragma unroll 1
            for (int v = 0; v < kW; ++v) {
                first = min(first, chosen[v]);
                end = max(end, last[v]);
            }
            token = first != 0x7fffffff ? first : end;
        }
    }
    // the standing drafts, the token, nothing behind them
#pragma unroll 1
    for (int row = out_row; row < d.end; row += THREADS) {
        int64_t out = row == out_row ? stands : row < d.row ? p.tokens[row + 1] : -1;
        if (row == d.row) out = token;
        p.emitted[row] = out;
        if (p.logprobs) {
            float y = row == d.row ? -__builtin_inff() : 0.0f;
            if (out >= 0) {
                const VerifyRow r = row == out_row ? out_stats : p.row_stats[row];
                y = static_cast<float>((static_cast<double>(logit_at<DT>(p.target, p.target_pitch, row, out)) -
                    static_cast<double>(r.top)) * inverse_t - log_above(r.sum));
            }
            p.logprobs[row] = y;
        }
    }
}

template <Dtype DT, int EACH, bool VEC>
hipError_t launch_variant(const VerifyParams &p, hipStream_t stream) {
    constexpr int kChunkThreads = EACH * kVerifyThreads;  // four tokens of a chunk a thread
    hipError_t e = hipSuccess;
    if (p.rows > 0) {
        // about 2048 workgroups, eight a CU, as long as there are chunks (1024: 39 us for the batch of eight, 2048: 37.5, all: 37.3)
        const int rows = p.rows * (p.draft ? 2 : 1), side = (2048 + rows - 1) / rows;
        const dim3 grid(p.chunks < side ? p.chunks : side, p.rows, p.draft ? 2 : 1);
        hipLaunchKernelGGL((verify_rows_kernel<DT, EACH, VEC>), grid, dim3(kVerifyThreads), 0, stream, p);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
    constexpr int kWeightThreads = EACH == 1 ? 256 : 512;
    hipLaunchKernelGGL((verify_weights_kernel<DT, kWeightThreads, VEC>), dim3(p.chunks, p.sequences), dim3(kWeightThreads), 0,
        stream, p);
    e = hipGetLastError();
    if (e == hipSuccess) {
        hipLaunchKernelGGL((verify_finish_kernel<DT, kChunkThreads, VEC>), dim3(p.sequences), dim3(kChunkThreads), 0,
            stream, p);
        e = hipGetLastError();
    }
    return e;
}

template <Dtype DT>
hipError_t launch_typed(const VerifyParams &p, bool vec, hipStream_t stream) {
    if (p.chunk == 1024) return vec ? launch_variant<DT, 1, true>(p, stream) : launch_variant<DT, 1, false>(p, stream);
    return vec ? launch_variant<DT, 4, true>(p, stream) : launch_variant<DT, 4, false>(p, stream);
}

}  // namespace

hipError_t launch_verify(const VerifyParams &p, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) return launch_typed<Dtype::F32>(p, vec, stream);
    if (dtype == Dtype::F16) return launch_typed<Dtype::F16>(p, vec, stream);
    return launch_typed<Dtype::BF16>(p, vec, stream);
}

}  // namespace fortai_hip
