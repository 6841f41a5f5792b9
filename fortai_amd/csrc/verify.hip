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
// the exponentials in 64 bits.
#include "fortai_hip_internal.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr float kLargest = 3.402823466e38f;

// exp(x) for x <= 0: x = n ln 2 + r, |r| <= ln 2 / 2, and the series of exp(r) to
// r^11 / 11! (off by 7e-15).
__device__ __forceinline__ double exp_below(double x) {
    if (!(x > -745.0)) return 0.0;
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(n, -0.693147180559945286227, x);
    r = __builtin_fma(n, -2.319046813846299558e-17, r);
    double y = 1.0 / 39916800.0;
    y = __builtin_fma(y, r, 1.0 / 3628800.0);
    y = __builtin_fma(y, r, 1.0 / 362880.0);
    y = __builtin_fma(y, r, 1.0 / 40320.0);
    y = __builtin_fma(y, r, 1.0 / 5040.0);
    y = __builtin_fma(y, r, 1.0 / 720.0);
    y = __builtin_fma(y, r, 1.0 / 120.0);
    y = __builtin_fma(y, r, 1.0 / 24.0);
    y = __builtin_fma(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    y = __builtin_fma(y, r, 1.0);
    return __builtin_ldexp(y, static_cast<int>(n));
}

// NaN counts as -infinity, +infinity as the largest number.
__device__ __forceinline__ float logit(float x) { return x != x ? -__builtin_inff() : fminf(x, kLargest); }

__device__ __forceinline__ double weight(float x, float top, double inverse_t) {
    return x == -__builtin_inff() ? 0.0 : exp_below((static_cast<double>(x) - static_cast<double>(top)) * inverse_t);
}

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
__device__ __forceinline__ double inverse_temperature(float t) { return t > 0.0f ? 1.0 / static_cast<double>(t) : 1.0; }

// the larger value, the lower index among equals
__device__ __forceinline__ void take_larger(float &v, int &i, float w, int j) {
    const bool other = w > v || (w == v && j < i);
    v = other ? w : v;
    i = other ? j : i;
}

__device__ __forceinline__ void wave_larger(float &v, int &i) {
    take_larger(v, i, xor_lane<32>(v), xor_lane<32>(i));
    take_larger(v, i, xor_lane<16>(v), xor_lane<16>(i));
    take_larger(v, i, xor_lane<8>(v), xor_lane<8>(i));
    take_larger(v, i, xor_lane<4>(v), xor_lane<4>(i));
    take_larger(v, i, xor_lane<2>(v), xor_lane<2>(i));
    take_larger(v, i, xor_lane<1>(v), xor_lane<1>(i));
}

// ---------------------------------------------------------------- (1) rows
// EACH: groups of four logits a thread holds (chunk = 1024 EACH)
template <Dtype DT, int EACH, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_rows_kernel(VerifyParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kChunk = kVerifyThreads * 4 * EACH;
    __shared__ int found;
    __shared__ float tops[kVerifyWaves];
    __shared__ int places[kVerifyWaves];
    __shared__ double sums[kVerifyWaves];
    const int row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool draft = blockIdx.z != 0;
    const E *x = static_cast<const E *>(draft ? p.draft : p.target) +
        static_cast<int64_t>(row) * (draft ? p.draft_pitch : p.target_pitch);
    float v[EACH][4];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int at = blockIdx.x * kChunk + (k * kVerifyThreads + static_cast<int>(threadIdx.x)) * 4;
        if (VEC && at + 3 < p.vocab) {
            const f32x4_t y = load4<DT, true>(x + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = logit(y[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = at + i < p.vocab ? logit(static_cast<float>(x[at + i])) : -__builtin_inff();
        }
    }
    // the row's sequence: its temperature, and whether it is a row with a draft
    if (threadIdx.x == 0) found = p.sequences;
    __syncthreads();
    for (int s = threadIdx.x; s < p.sequences; s += kVerifyThreads) {
        int begin, end;
        sequence_rows(p, s, &begin, &end);
        if (row >= begin && row < end - (draft ? 1 : 0)) atomicMin(&found, s);
    }
    float top = -__builtin_inff();
    int place = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < EACH; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            take_larger(top, place, v[k][i], blockIdx.x * kChunk + (k * kVerifyThreads + static_cast<int>(threadIdx.x)) * 4 + i);
    wave_larger(top, place);
    if (lane == 0) {
        tops[wave] = top;
        places[wave] = place;
    }
    __syncthreads();
    const int seq = found;
    if (seq >= p.sequences) return;
    top = tops[0];
    place = places[0];
#pragma unroll
    for (int w = 1; w < kVerifyWaves; ++w) take_larger(top, place, tops[w], places[w]);
    const double inverse_t = inverse_temperature(temperature(p, seq));
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += weight(v[k][i], top, inverse_t);
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        VerifyPart part;
        part.sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        part.top = top;
        part.place = place;
        p.parts[(static_cast<size_t>(draft ? p.max_rows : 0) + row) * p.chunks + blockIdx.x] = part;
    }
}

// ------------------------------------------------- which row decides
struct RowStats {
    double sum;  // of exp((x - top) / T)
    float top;
    int place;
};

__device__ __forceinline__ RowStats row_stats(const VerifyParams &p, int row, bool draft, double inverse_t) {
    const VerifyPart *parts = p.parts + (static_cast<size_t>(draft ? p.max_rows : 0) + row) * p.chunks;
    const int lane = threadIdx.x & 63;
    RowStats r = {0.0, -__builtin_inff(), 0x7fffffff};
    for (int c = lane; c < p.chunks; c += 64) take_larger(r.top, r.place, parts[c].top, parts[c].place);
    wave_larger(r.top, r.place);
    for (int c = lane; c < p.chunks; c += 64) r.sum += parts[c].sum * weight(parts[c].top, r.top, inverse_t);
    r.sum = wave_sum(r.sum);
    return r;
}

struct Decision {
    int accepted;       // drafts that stand
    int row;            // the row that decides, or -1: the sequence has none
    bool against_draft; // its draft was turned down: what is left of p over q is drawn from
    int rejected;       // that draft
    RowStats target, draft;
};

template <Dtype DT>
__device__ __forceinline__ float logit_at(const void *logits, int64_t pitch, int row, int64_t token) {
    return logit(static_cast<float>(static_cast<const typename Element<DT>::type *>(logits)[static_cast<int64_t>(row) * pitch + token]));
}

// Every thread of the workgroup; a wave a row, four rows at a time.  write: the
// standing drafts and their log probabilities are put out on the way.
template <Dtype DT>
__device__ __forceinline__ Decision decide(const VerifyParams &p, int seq, bool write) {
    __shared__ int stands[kVerifyWaves];
    __shared__ RowStats kept[kVerifyWaves][2];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int begin, end;
    sequence_rows(p, seq, &begin, &end);
    Decision d;
    d.accepted = 0;
    d.row = -1;
    d.against_draft = false;
    d.rejected = -1;
    d.target = d.draft = RowStats{0.0, 0.0f, 0};
    if (begin == end) return d;
    const float t = temperature(p, seq);
    const double inverse_t = inverse_temperature(t);
    for (int first = begin; first < end; first += kVerifyWaves) {
        const int row = first + wave;
        if (row < end) {
            const RowStats target = row_stats(p, row, false, inverse_t);
            RowStats draft = {0.0, 0.0f, 0};
            bool ok = false;
            if (row + 1 < end) {
                const int64_t x = p.tokens[row + 1];
                if (p.draft) draft = row_stats(p, row, true, inverse_t);
                if (x >= 0 && x < p.vocab) {
                    const float l = logit_at<DT>(p.target, p.target_pitch, row, x);
                    if (t > 0.0f) {
                        const double px = target.sum > 0.0 ? weight(l, target.top, inverse_t) / target.sum : 0.0;
                        double qx = 1.0;
                        if (p.draft)
                            qx = draft.sum > 0.0
                                ? weight(logit_at<DT>(p.draft, p.draft_pitch, row, x), draft.top, inverse_t) / draft.sum : 0.0;
                        ok = static_cast<double>(p.uniforms[row]) * qx < px;
                    } else {
                        ok = target.sum > 0.0 && x == target.place;
                    }
                    if (write && ok && lane == 0 && p.logprobs)
                        p.logprobs[row] = static_cast<float>(
                            (static_cast<double>(l) - static_cast<double>(target.top)) * inverse_t - log(target.sum));
                }
            }
            if (lane == 0) {
                stands[wave] = ok;
                kept[wave][0] = target;
                kept[wave][1] = draft;
            }
        }
        __syncthreads();
        for (int w = 0; w < kVerifyWaves && first + w < end && d.row < 0; ++w)
            if (!stands[w]) {
                d.row = first + w;
                d.accepted = d.row - begin;
                d.target = kept[w][0];
                d.draft = kept[w][1];
                d.against_draft = d.row + 1 < end;
                if (d.against_draft) {
                    const int64_t x = p.tokens[d.row + 1];
                    d.rejected = x >= 0 && x < p.vocab ? static_cast<int>(x) : -1;
                }
            }
        __syncthreads();
        if (d.row >= 0) break;  // the sequence's last row never stands, so some row does not
    }
    return d;
}

// what a token weighs in the draw: p, or what p has over q
template <Dtype DT>
__device__ __forceinline__ double draw_weight(const VerifyParams &p, const Decision &d, bool left, double inverse_t, int token) {
    const double pt = d.target.sum > 0.0
        ? weight(logit_at<DT>(p.target, p.target_pitch, d.row, token), d.target.top, inverse_t) / d.target.sum : 0.0;
    if (!left) return pt;
    double qt;
    if (!p.draft) qt = token == d.rejected ? 1.0 : 0.0;
    else if (d.draft.sum > 0.0)
        qt = weight(logit_at<DT>(p.draft, p.draft_pitch, d.row, token), d.draft.top, inverse_t) / d.draft.sum;
    else qt = 0.0;
    return fmax(pt - qt, 0.0);
}

// -------------------------------------------------- (2) the deciding row
template <Dtype DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_weights_kernel(VerifyParams p) {
    __shared__ double sums[kVerifyWaves];
    const int seq = blockIdx.y;
    const float t = temperature(p, seq);
    if (!(t > 0.0f)) return;  // the argmax is known
    const Decision d = decide<DT>(p, seq, false);
    if (d.row < 0 || !d.against_draft) return;  // p's own chunk sums are known
    const double inverse_t = inverse_temperature(t);
    const int from = blockIdx.x * p.chunk, until = min(from + p.chunk, p.vocab);
    double sum = 0.0;
    for (int k = from + threadIdx.x; k < until; k += kVerifyThreads) sum += draw_weight<DT>(p, d, true, inverse_t, k);
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) p.weights[static_cast<size_t>(seq) * p.chunks + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// sum over the lanes up to and including this one
__device__ __forceinline__ double wave_prefix(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double below = __shfl_up(v, d);
        if (lane >= d) v += below;
    }
    return v;
}

// ------------------------------------------------------- (3) the token
template <Dtype DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_finish_kernel(VerifyParams p) {
    __shared__ double waves[kVerifyWaves];
    __shared__ int chosen, last;
    __shared__ int chunk_at;
    __shared__ double below_at;
    const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float t = temperature(p, seq);
    const double inverse_t = inverse_temperature(t);
    const Decision d = decide<DT>(p, seq, true);
    int begin, end;
    sequence_rows(p, seq, &begin, &end);
    if (threadIdx.x == 0) {
        p.accepted[seq] = d.accepted;
        chosen = 0x7fffffff;
        last = -1;
        chunk_at = -1;
    }
    if (d.row < 0) return;
    __syncthreads();
    int token = -1;
    if (!(t > 0.0f)) {
        token = d.target.sum > 0.0 ? d.target.place : -1;
    } else {
        const VerifyPart *parts = p.parts + static_cast<size_t>(d.row) * p.chunks;
        const double *weights = p.weights + static_cast<size_t>(seq) * p.chunks;
        const double u = static_cast<double>(p.uniforms[end - 1]);
        // p where nothing is left of it over q, which a draft of probability zero can leave
        bool left = d.against_draft;
        double total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            total = 0.0;
            for (int c0 = 0; c0 < p.chunks; c0 += 64) {
                const int c = c0 + lane;
                double w = 0.0;
                if (c < p.chunks) w = left ? weights[c] : d.target.sum > 0.0 ? parts[c].sum * weight(parts[c].top, d.target.top, inverse_t) / d.target.sum : 0.0;
                total += __shfl(wave_prefix(w), 63);
            }
            if (total > 0.0 || !left) break;
            left = false;
        }
        if (wave == 0 && total > 0.0) {
            // the first chunk whose end lies over u total, else the last one that weighs anything
            double below = 0.0, best_below = 0.0;
            int best = -1;
            bool over = false;
            for (int c0 = 0; c0 < p.chunks && !over; c0 += 64) {
                const int c = c0 + lane;
                double w = 0.0;
                if (c < p.chunks) w = left ? weights[c] : parts[c].sum * weight(parts[c].top, d.target.top, inverse_t) / d.target.sum;
                const double upto = below + wave_prefix(w);
                const uint64_t past = __ballot(w > 0.0 && upto > u * total), some = __ballot(w > 0.0);
                if (past || some) {
                    const int k = past ? __ffsll(static_cast<unsigned long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(some));
                    best = c0 + k;
                    best_below = __shfl(upto - w, k);
                    over = past != 0;
                }
                below = __shfl(upto, 63);
            }
            if (lane == 0) {
                chunk_at = best;
                below_at = best_below;
            }
        }
        __syncthreads();
        if (chunk_at >= 0) {
            // consecutive tokens a thread
            const int each = (p.chunk + kVerifyThreads - 1) / kVerifyThreads;
            const int from = chunk_at * p.chunk + threadIdx.x * each, until = min(min(from + each, (chunk_at + 1) * p.chunk), p.vocab);
            double mine = 0.0;
            for (int k = from; k < until; ++k) mine += draw_weight<DT>(p, d, left, inverse_t, k);
            const double prefix = wave_prefix(mine);
            if (lane == 63) waves[wave] = prefix;
            __syncthreads();
            double c = below_at + prefix - mine;
            for (int w = 0; w < wave; ++w) c += waves[w];
            const double border = u * total;
            for (int k = from; k < until; ++k) {
                const double w = draw_weight<DT>(p, d, left, inverse_t, k);
                c += w;
                if (w > 0.0) {
                    atomicMax(&last, k);
                    if (c > border) {
                        atomicMin(&chosen, k);
                        break;
                    }
                }
            }
            __syncthreads();
            token = chosen != 0x7fffffff ? chosen : last;
        }
    }
    for (int row = begin + threadIdx.x; row < end; row += kVerifyThreads) {
        p.emitted[row] = row < d.row ? p.tokens[row + 1] : row == d.row ? token : -1;
        if (p.logprobs && row >= d.row) {
            float y = 0.0f;
            if (row == d.row)
                y = token < 0 ? -__builtin_inff()
                    : static_cast<float>((static_cast<double>(logit_at<DT>(p.target, p.target_pitch, row, token)) -
                          static_cast<double>(d.target.top)) * inverse_t - log(d.target.sum));
            p.logprobs[row] = y;
        }
    }
}

template <Dtype DT, int EACH>
void launch_rows(const VerifyParams &p, bool vec, hipStream_t stream) {
    const dim3 grid(p.chunks, p.rows, p.draft ? 2 : 1);
    if (vec) hipLaunchKernelGGL((verify_rows_kernel<DT, EACH, true>), grid, dim3(kVerifyThreads), 0, stream, p);
    else hipLaunchKernelGGL((verify_rows_kernel<DT, EACH, false>), grid, dim3(kVerifyThreads), 0, stream, p);
}

template <Dtype DT>
hipError_t launch_typed(const VerifyParams &p, bool vec, hipStream_t stream) {
    if (p.rows == 0) {
        // sequences without rows: the finish writes that no draft stands
    } else if (p.chunk == 1024) launch_rows<DT, 1>(p, vec, stream);
    else launch_rows<DT, 4>(p, vec, stream);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) {
        hipLaunchKernelGGL((verify_weights_kernel<DT>), dim3(p.chunks, p.sequences), dim3(kVerifyThreads), 0, stream, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        hipLaunchKernelGGL((verify_finish_kernel<DT>), dim3(p.sequences), dim3(kVerifyThreads), 0, stream, p);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

hipError_t launch_verify(const VerifyParams &p, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) return launch_typed<Dtype::F32>(p, vec, stream);
    if (dtype == Dtype::F16) return launch_typed<Dtype::F16>(p, vec, stream);
    return launch_typed<Dtype::BF16>(p, vec, stream);
}

}  // namespace fortai_hip
