// The gated delta rule over a batch's rows, for sequences of many rows (prompts): 64
// rows at a time.
//
// With c_i the sum of the chunk's logarithmic decays up to row i, S the state before the
// chunk and d_i the updates (gdn_rows.hip has the recurrence):
//   A_ij = b_i exp(c_i - c_j) k_i.k_j  (j < i),  T = (I + A)^-1
//   W = T diag(b exp(c)) K,  U = T diag(b) V
//   D = U - W S^T,  O = diag(exp(c)) Q S^T + tril(exp(c_i - c_j) q_i.k_j) D
//   S <- exp(c_n) S + sum_j exp(c_n - c_j) d_j k_j^T
// Only the last two lines go from chunk to chunk.  Three launches: convolution, norms and
// gates of all rows; W, U and the weights of every chunk and head at once; then the
// states through their chunks, a workgroup 16 or 32 value dims of a head, whose part of S
// stays in registers.
//
// Products run in fp16 matrix instructions with fp32 sums: an operand is two numbers,
// x scale = h + l, and h h + h l + l h keeps 22 bits of either (three instructions of a
// sixteenth of the fp32 one's time each), down to l's smallest step.  q, k, W, T and the weights are
// at most 1 (decays are at most 1, and a row's update answers any value at most its own
// size: the rule is a contraction) and scaled by 2^15, weights by 2^18 (a query's length is at most an eighth).
// Values (times b), S and D have any size: a column (one value
// dim) is scaled by a power of two, b V by its largest in the chunk, S and D by bounds: with
// s the largest of S before the chunk and u that of U,
//   |D| <= u + sqrt(head) s,  |S after it| <= exp(c_n) s + sum_j exp(c_n - c_j) max |D|,
// which no wave has to wait for another's numbers for.  S itself, the
// updates and all sums are fp32.
//
// So a chunk's numbers are off by 2^-38 or so of R, the largest of s and |b v| in their column (64 errors of 2^-39
// of it that all point one way: 2^-31).  That is rounding for a row in whose text something of R's size is left: it has
// at least 2^-20 R among b v and s up to it, with the decays since.  Where a row has less (tokens before a far louder
// one, or behind one that is forgotten), it and the chunk's rows before it go one by one, in fp32, as few rows do, for
// the 16 or 32 columns of a workgroup at once.  The chunk kernel looks for such rows, since it has the values, makes
// their U in fp32 products, and says in a word a column which s is enough for them; the kernel that has s compares.
// (Where, of ordinary values, one first row in 10^5 is that small: 4 us.)  2000 rows of 16 heads 113 us, of which
// this is 3; with every row one by one, 0.75 us each, 1.6 ms.  Outputs of the 56 rows before one that is 1 to 2^30 times
// as loud are off by 2^-22 of their size throughout.
//
// The sums c are taken in 64 bits: far into a decay they are large, and their differences
// are not.  A row's logarithm is -256 at least (gdn_log_decay), so that 64 of them stay below
// 2^15 and keep 2^-38 of what lies between any two rows.
#include "gdn_device.h"

#include <type_traits>

namespace fortai_hip {

namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int kRun = kGdnRun;       // rows that a wave of the first launch takes
constexpr float kOne = 32768.0f;    // 2^15
constexpr float kWeight = 262144.0f;  // 2^18
constexpr float kWithin = 0x1p-20f, kWithinLog = -20.0f;  // what a row has of its column's largest, or it goes by itself
constexpr int kLoadsMayCross = 0x2 | 0x4 | 0x10;  // for sched_barrier: vector, scalar and memory, not matrix and LDS instructions
constexpr float kProduct = 1.0f / (kOne * kOne);

template <typename V>
struct Pair {
    V h, l;
};
typedef Pair<f16x4_t> Pair4;
typedef Pair<f16x8_t> Pair8;

// scaled: x times what brings it to 2^15 at most.  It is rounded to fp32 before anything is
// done with it: the compiler folds a multiplication into a conversion to fp16 (one
// rounding), but not into every use of it, and a lower half that is left over from
// another upper half is off by a whole step.
__device__ __forceinline__ void split(float scaled, _Float16 &h, _Float16 &l) {
    asm("" : "+v"(scaled));
    h = static_cast<_Float16>(scaled);
    l = static_cast<_Float16>(scaled - static_cast<float>(h));
}

__device__ __forceinline__ Pair4 split4(f32x4_t scaled) {
    Pair4 p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 h, l;
        split(scaled[e], h, l);
        p.h[e] = h;
        p.l[e] = l;
    }
    return p;
}

__device__ __forceinline__ f32x4_t product(const Pair4 &a, const Pair4 &b, f32x4_t c) {
    c = __builtin_amdgcn_mfma_f32_16x16x16f16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x16f16(a.h, b.l, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a.h, b.h, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t product(const Pair8 &a, const Pair8 &b, f32x4_t c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.l, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}

// the four elements are the four k indexes of lane group g, the same ones on both sides
__device__ __forceinline__ f32x4_t product32(f32x4_t a, f32x4_t b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// The power of two that brings numbers up to `top` below 2^15, and back from a product with
// a number times 2^15 (1 for nothing).
struct Scale {
    float to, from, least;  // least: what keeps 22 bits (2^-3, scaled), unless it is near the end of fp32
    __device__ __forceinline__ explicit Scale(float top) {
        const int e = top > 0.0f ? min(max(__builtin_amdgcn_frexp_expf(top), -100), 128) : 0;
        to = __builtin_ldexpf(32768.0f, -e);
        from = __builtin_ldexpf(1.0f / (32768.0f * kOne), e);
        least = __builtin_ldexpf(e > -100 ? 0x1p-18f : 0.0f, e);
    }
};

__device__ __forceinline__ float largest(f32x4_t x) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); }
// over the four lane groups that share a column
__device__ __forceinline__ float largest_of_column(float x) {
    x = fmaxf(x, xor_lane<16>(x));
    return fmaxf(x, xor_lane<32>(x));
}

__device__ __forceinline__ bool gdn_is_many(const GdnRowsParams &p, const GdnSequence &s) { return s.count > p.few && s.slot >= 0; }

// Operands are kept as the matrix instructions take them, a run (16 rows) of a head at a
// time, lane after lane, so that a wave's load is one piece of memory: a lane has row or
// dim m = lane & 15 and, of the index that is summed over, four or eight numbers from lane
// group g = lane >> 4.  Sequences of more than 16 rows begin at least 17 apart, so that no two
// runs have the same place.  (One sequence by itself may have fewer.)
__device__ __forceinline__ int64_t run_place(const GdnSequence &s, int64_t row) { return row / kRun + s.begin / (kRun + 1); }

template <int D>
struct Runs {
    // numbers of a row that a lane has at once, of D key dims in four steps
    static constexpr int kAsk = D / 16;
    typedef std::conditional_t<D == 128, f16x8_t, f16x4_t> Ask;
    static constexpr int kHead = kRun * D * 2;  // halves of a run of a head
    // queries, keys (rows m) and W: [step][upper, lower][lane][kAsk]
    static __device__ __forceinline__ Pair<Ask> row_step(const _Float16 *run, int step, int lane) {
        const _Float16 *at = run + (step * 2 * 64 + lane) * kAsk;
        return Pair<Ask>{*reinterpret_cast<const Ask *>(at), *reinterpret_cast<const Ask *>(at + 64 * kAsk)};
    }
};
// keys (dims m of a tile) and the weights (rows m, of 16 updates): [lane][upper four, lower four]
__device__ __forceinline__ Pair4 four_step(const _Float16 *tile, int lane) {
    const f16x8_t v = *reinterpret_cast<const f16x8_t *>(tile + lane * 8);
    return Pair4{f16x4_t{v[0], v[1], v[2], v[3]}, f16x4_t{v[4], v[5], v[6], v[7]}};
}
__device__ __forceinline__ void store_four_step(_Float16 *tile, int lane, const Pair4 &x) {
    *reinterpret_cast<f16x8_t *>(tile + lane * 8) = f16x8_t{x.h[0], x.h[1], x.h[2], x.h[3], x.l[0], x.l[1], x.l[2], x.l[3]};
}

// Convolution, norms and gates: a wave has 128 channels (two a lane) of a run, or every
// gate.  TAPS: of the convolution, 0: as many as there are.  PAIRS: two elements at once.
// Bound by memory: 2456 rows of 8192 channels in fp32, 180 MB in and out, 43 us.
template <Dtype DT, int D, int TAPS, bool PAIRS>
__global__ __launch_bounds__(256) void gdn_inputs_kernel(const GdnRowsParams p) {
    typedef typename Element<DT>::type E;
    typedef E E2 __attribute__((ext_vector_type(2)));
    constexpr int kTaps = TAPS ? TAPS : kGdnMaxTaps;
    // a wave's results as they lie in memory, 16 bytes a unit: written from here a piece at a time
    __shared__ u32x4_t images[4][512];
    const int lane = threadIdx.x & 63, part = blockIdx.x * 4 + (threadIdx.x >> 6), seq = blockIdx.z;
    const GdnView &c = p.cache;
    GdnSequence s = gdn_sequence(p, seq);
    if (!gdn_is_many(p, s)) return;
    const int i0 = blockIdx.y * kRun, rows = min(s.count - i0, kRun), channels = c.channels(), parts = (channels + 127) / 128;
    if (rows <= 0 || part > parts) return;
    if (part == parts) {
        const int all = rows * c.value_heads;
        for (int at0 = lane; at0 < all; at0 += 256) {
            float alpha[4], beta[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = min(at0 + 64 * k, all - 1), h = at % c.value_heads;
                const int64_t row = s.begin + i0 + at / c.value_heads;
                alpha[k] = static_cast<float>(static_cast<const E *>(p.alpha)[row * p.alpha_row + h]);
                beta[k] = static_cast<float>(static_cast<const E *>(p.beta)[row * p.beta_row + h]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = min(at0 + 64 * k, all - 1), h = at % c.value_heads;
                const int64_t to = (s.begin + i0) * static_cast<int64_t>(c.value_heads) + at;
                p.decay[to] = gdn_log_decay(p.ssm_a[h], alpha[k], p.ssm_dt[h]);
                p.rate[to] = gdn_sigmoid(beta[k]);
            }
        }
        return;
    }
    const int taps = TAPS ? TAPS : c.taps, before = taps - 1, first = kTaps - taps;
    if (i0 == 0) s.stands = gdn_stands(p, s);
    // heads of 64: the last wave may have one head only (its other lanes repeat it and store nothing)
    const bool mine = part * 128 + 2 * lane < channels;
    const int channel = mine ? part * 128 + 2 * lane : channels - D + (2 * lane) % D;
    f32x2_t x[kTaps - 1 + 4], ahead[4], w[kTaps];
    const E *rows_at = static_cast<const E *>(p.qkv) + channel;
    const auto input = [&](int row) {
        const E *at = rows_at + (s.begin + min(row, s.count - 1)) * p.qkv_row;
        if constexpr (PAIRS) {
            const E2 v = *reinterpret_cast<const E2 *>(at);
            return f32x2_t{static_cast<float>(v[0]), static_cast<float>(v[1])};
        }
        else return f32x2_t{static_cast<float>(at[0]), static_cast<float>(at[1])};
    };
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) {
        const int row = i0 + j - (kTaps - 1);
        x[j] = f32x2_t{0.0f, 0.0f};
        if (row >= 0) {
            x[j] = input(row);
        } else if (row >= -before && !s.begins) {
            const float *at = c.inputs + (static_cast<int64_t>(s.slot) * (before + c.pending) + s.stands + before + row) * channels + channel;
            x[j] = f32x2_t{at[0], at[1]};
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) ahead[k] = input(i0 + k);
#pragma unroll
    for (int j = 0; j < kTaps; ++j) {
        const float *at = p.conv + static_cast<int64_t>(channel) * taps + j - first;
        w[j] = j >= first ? f32x2_t{at[0], at[taps]} : f32x2_t{0.0f, 0.0f};
    }
    const int head = channel / D, dim = channel % D;
    const bool is_value = head >= 2 * c.key_heads, is_key = !is_value && head >= c.key_heads;
    const int64_t run = run_place(s, s.begin + i0);
    // 2^15 over the length, but no more than over epsilon; queries also over sqrt(head)
    const float one = is_key ? kOne : kOne / sqrtf(static_cast<float>(D)), most = fminf(one / p.eps, 3e38f);
    // the head's part of the image, D * 4 units (heads of 64: two heads a wave, half its lanes each)
    constexpr int kAsk = Runs<D>::kAsk, kUnits = D * 4, kHeadLanes = D / 2;
    u32x4_t *image = images[threadIdx.x >> 6] + (lane / kHeadLanes) * kUnits;
    // lanes that write together have the same row, or four rows, of different steps or tiles: their units are turned so
    // that they meet different banks
    const int turn_shift = is_value ? 6 : 4, turn_low = is_value ? 1 : 3, turn_high = is_value ? 0 : 12;
    const auto turned = [&](int unit) { return unit ^ (unit >> turn_shift & turn_low) ^ (unit >> 5 & turn_high); };
    const int tile_at = (dim >> 4) * 64 + (dim & 15);  // the first of its tile's lanes that have this dim
    const int ask_at = (dim / (4 * kAsk) * 2 * 64 + dim / kAsk % 4 * 16) * kAsk + dim % kAsk;  // in halves, of row 0
    _Float16 *by_dim = p.keys_by_dim + (run * c.key_heads + (is_key ? head - c.key_heads : 0)) * Runs<D>::kHead + tile_at * 8;
    // rows past the last are those of the last inputs again: finite, and their updates are zero
#pragma unroll 1
    for (int four = 0; four < kRun / 4; ++four) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[kTaps - 1 + k] = ahead[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) ahead[k] = input(i0 + min(4 * four + 4, kRun - 4) + k);
        f32x4_t y[2], inverse;  // this lane's dims, four rows
        float most_sum = 0.0f, least_sum = 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u0 = 0.0f, u1 = 0.0f;
#pragma unroll
            for (int j = 0; j < kTaps; ++j)
                if (j >= first) {
                    u0 = __builtin_fmaf(w[j][0], x[i + j][0], u0);
                    u1 = __builtin_fmaf(w[j][1], x[i + j][1], u1);
                }
            u0 = gdn_silu(u0);
            u1 = gdn_silu(u1);
            y[0][i] = u0;
            y[1][i] = u1;
            const float sum = group_sum_up(u0 * u0 + u1 * u1, kHeadLanes);
            inverse[i] = fminf(__builtin_amdgcn_rsqf(sum) * one, most);
            most_sum = fmaxf(most_sum, sum);
            least_sum = fminf(least_sum, sum);
        }
        if (__any((gdn_length_is_lost(most_sum, p.eps) | gdn_length_is_lost(least_sum, p.eps)) & !is_value)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = fmaxf(fabsf(y[0][i]), fabsf(y[1][i]));
                top = fmaxf(top, xor_lane<1>(top));
                top = fmaxf(top, xor_lane<2>(top));
                top = fmaxf(top, xor_lane<4>(top));
                top = fmaxf(top, xor_lane<8>(top));
                top = fmaxf(top, xor_lane<16>(top));
                if constexpr (kHeadLanes == 64) top = fmaxf(top, xor_lane<32>(top));
                const int e = is_value ? 0 : __builtin_amdgcn_frexp_expf(top);
                y[0][i] = __builtin_ldexpf(y[0][i], -e);
                y[1][i] = __builtin_ldexpf(y[1][i], -e);
                const float near_one = group_sum_up(y[0][i] * y[0][i] + y[1][i] * y[1][i], kHeadLanes);
                inverse[i] = fminf(__builtin_amdgcn_rsqf(near_one) * one, one / __builtin_ldexpf(p.eps, -e));
            }
        }
        if (!is_value) {
            y[0] *= inverse;
            y[1] *= inverse;
        }
#pragma unroll
        for (int j = 0; j + 1 < kTaps; ++j) x[j] = x[j + 4];
        if (is_value) {
            reinterpret_cast<f32x4_t *>(image)[turned(tile_at + 16 * four)] = y[0];
            reinterpret_cast<f32x4_t *>(image)[turned(tile_at + 16 * four + 1)] = y[1];
            continue;
        }
        const Pair4 a = split4(y[0]), b = split4(y[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = ask_at + (4 * four + i) * kAsk;
            reinterpret_cast<f16x2_t *>(image + turned(at / 8))[at % 8 / 2] = f16x2_t{a.h[i], b.h[i]};
            reinterpret_cast<f16x2_t *>(image + turned((at + 64 * kAsk) / 8))[at % 8 / 2] = f16x2_t{a.l[i], b.l[i]};
        }
        if (is_key && mine) {
            store_four_step(by_dim + 16 * four * 8, 0, a);
            store_four_step(by_dim + 16 * four * 8, 1, b);
        }
    }
    wave_lds_fence();
    u32x4_t *to = is_value ? reinterpret_cast<u32x4_t *>(p.values + (run * c.value_heads + head - 2 * c.key_heads) * (kRun * D))
                           : reinterpret_cast<u32x4_t *>(p.asks + (run * 2 * c.key_heads + head) * Runs<D>::kHead);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int unit = k * kHeadLanes + lane % kHeadLanes;
        const u32x4_t v = image[turned(unit)];
        if (mine) to[unit] = v;
    }
    if (i0 != 0) return;
    // its own channels' reads of the slot's inputs are done
    if (mine) {
        gdn_keep_inputs<E>(p, s, false, channel);
        gdn_keep_inputs<E>(p, s, false, channel + 1);
    }
    if (channel == 0 && lane == 0) p.stands[seq] = s.begins ? -1 : s.stands;
}

// What a column's numbers ask of the state before them.  A row is faint if it has less than kWithin of the column's
// largest number, most, in its text (b v so far, with the decays since).  A lane has rows 16 b + 4 g + e.  In binary
// logarithms: the largest of log |v_j| - c_j up to row i, and c_i.
struct Faint {
    int last;     // faint row, -1: none
    float least;  // in the text of rows at which the state is gone
};

__device__ __forceinline__ Faint faint_rows(const f32x4_t (&v)[4], float most, const float *logs, int n, int lane) {
    Faint f = {-1, __builtin_inff()};
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        f32x4_t x = v[b];
        if (n < kGdnChunk) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (16 * b + 4 * (lane >> 4) + e >= n) x[e] = f.least;
        }
        f.least = fminf(f.least, fminf(fminf(fabsf(x[0]), fabsf(x[1])), fminf(fabsf(x[2]), fabsf(x[3]))));
    }
    // whatever the decays, and with room for states of up to four times the largest (of ordinary values one tile in 50
    // does not get by)
    if (__all(f.least >= most * (8.0f * kWithin))) {
        f.least = fminf(f.least, xor_lane<16>(f.least));
        f.least = fminf(f.least, xor_lane<32>(f.least));
        return f;
    }
    const int g = lane >> 4;
    const float none = -__builtin_inff(), low = __builtin_amdgcn_logf(most * kWithin);
    float before = none, least = __builtin_inff();  // before: the largest of the runs before
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const f32x4_t c = *reinterpret_cast<const f32x4_t *>(logs + 16 * b + 4 * g);
        float up_to[4], x = none;
#pragma unroll
        for (int e = 0; e < 4; ++e) up_to[e] = x = fmaxf(x, __builtin_amdgcn_logf(fabsf(v[b][e])) - c[e]);
        // of the lanes of the rows before these, and of all of the run
        const float one = __shfl(x, lane - 16), two = __shfl(x, lane - 32), three = __shfl(x, lane - 48);
        float earlier = before;
        if (g > 0) earlier = fmaxf(earlier, one);
        if (g > 1) earlier = fmaxf(earlier, two);
        if (g > 2) earlier = fmaxf(earlier, three);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * b + 4 * g + e;
            const float text = fmaxf(up_to[e], earlier) + c[e];
            if (row < n && text < low) f.last = row;
            if (row < n && c[e] < kWithinLog) least = fminf(least, text);
        }
        before = fmaxf(before, largest_of_column(x));
    }
    f.last = max(f.last, xor_lane<16>(f.last));
    f.last = max(f.last, xor_lane<32>(f.last));
    least = fminf(least, xor_lane<16>(least));
    f.least = __builtin_amdgcn_exp2f(fminf(least, xor_lane<32>(least)));
    return f;
}

// A column of U and what its rows ask of the largest of S in it, s, as the exponents of four powers of two in a word, the
// first in the lowest bits: need is enough of s for the faint rows (they have kWithin of the chunk's largest from it); limit
// leaves the rows at which S is gone kWithin of it in their text, and bounds within fp32; top and left are no less than
// the largest of U and the sum of the decays to the chunk's end.  The others' bits stand behind an exponent and
// make its number up to twice as large (need has none).
struct Column {
    float need, limit, top, left;
    __device__ __forceinline__ explicit Column(uint32_t word)
        : need(fabsf(__builtin_bit_cast(float, word << 23))), limit(fabsf(__builtin_bit_cast(float, word << 15))),
          top(fabsf(__builtin_bit_cast(float, word << 7))), left(__builtin_bit_cast(float, word >> 1)) {}
    __device__ __forceinline__ bool exceeded(float s) const { return !(s <= limit); }
    __device__ __forceinline__ bool wanting(float s) const { return s < need; }
    static __device__ __forceinline__ uint32_t word(float top, float left, const Faint &f, float most, const float *logs) {
        const float gone = f.last >= 0 ? logs[f.last] : 0.0f, infinite = __builtin_inff();
        float need = f.last < 0 ? 0.0f : gone < kWithinLog ? infinite : most * kWithin * __builtin_amdgcn_exp2f(-gone);
        float limit = fminf(logs[kGdnChunk - 1] < kWithinLog ? f.least * (0.5f / kWithin) : infinite, 0x1p100f);
        if (!(top < 0x1p100f)) {  // no s will do
            need = infinite;
            limit = 0.0f;
        }
        const auto up = [](float x) { return (__builtin_bit_cast(uint32_t, x) + 0x7fffffu) >> 23; };
        return up(left) << 24 | up(top) << 16 | __builtin_bit_cast(uint32_t, limit) >> 23 << 8 | up(need);
    }
};

// One tile of U = T b V, over V, in fp32 products; its largest number.
template <typename Rows>
__device__ __forceinline__ float exact_updates(float *values, int64_t run_values, int last_run, const float *rates, int g, const Rows &rows_of_t) {
    f32x4_t v[4];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < 4; ++b)
        v[b] = *reinterpret_cast<const f32x4_t *>(values + min(b, last_run) * run_values) * *reinterpret_cast<const f32x4_t *>(rates + 16 * b + 4 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i > last_run) break;
        f32x4_t u = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b <= i; ++b) u = product32(rows_of_t(i, b), v[b], u);
        top = fmaxf(top, largest(u));
        *reinterpret_cast<f32x4_t *>(values + i * run_values) = u;
    }
    return top;
}

// W, U and the weights of one chunk and value head.
// Three workgroups a CU: each goes through a chain of small steps with barriers between
// them, and waits most of the time.  Everything that comes from memory is asked for before
// the first of them, without conditions, so that no wait is for more than it needs.  43
// chunks of 32 heads: 49 us, which is 4.1 TB/s of operands read and written; 32 chunks of 16
// heads 23.7 us, two chains one after the other.  Of these the search for faint rows takes 3 and 1.9 us.
template <int D>
__global__ __launch_bounds__(256, 3) void gdn_chunk_kernel(const GdnRowsParams p) {
    typedef typename Runs<D>::Ask Ask;
    constexpr int kPitch = kGdnChunk + 4, kPitchT = kGdnChunk + 4, kTiles = D / 64, kHead = Runs<D>::kHead, kAsk = Runs<D>::kAsk;
    // first the keys by rows; then A, and T beside it; then T with b exp(c) (where A was) and with b, in halves
    __shared__ __align__(16) float as[2 * kGdnChunk * kPitch], ts[kGdnChunk * kPitch];
    static_assert(sizeof(as) >= 4 * kHead * sizeof(_Float16), "the keys of four runs");
    _Float16(*halves)[2][kGdnChunk * kPitchT] = reinterpret_cast<_Float16(*)[2][kGdnChunk * kPitchT]>(as);
    __shared__ double sums[kGdnChunk];  // binary logarithms
    __shared__ __align__(16) float rates[kGdnChunk], asked_rates[kGdnChunk], logs[kGdnChunk];  // b, with exp(c); c, in 32 bits
    __shared__ float left_sum;  // of the decays to the chunk's end
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GdnView &c = p.cache;
    const GdnSequence s = gdn_sequence(p, blockIdx.z);
    if (!gdn_is_many(p, s)) return;
    const int n = min(s.count - static_cast<int>(blockIdx.y) * kGdnChunk, kGdnChunk), h = blockIdx.x;
    if (n <= 0) return;
    const int64_t row0 = s.begin + static_cast<int64_t>(blockIdx.y) * kGdnChunk, run0 = run_place(s, row0);
    const int kh = h / (c.value_heads / c.key_heads), last_run = (n - 1) / kRun;

    // gates (of lane's row), a run of keys a wave, and the rows whose products with keys this wave has: of keys
    // (waves 0 and 1) or queries (2 and 3), runs 0 and 3, or 1 and 2
    const int64_t gate_at = (row0 + min(lane, n - 1)) * c.value_heads + h;
    const float my_decay = p.decay[gate_at], my_rate = p.rate[gate_at];
    const auto run_of = [&](int run, int head) { return p.asks + ((run0 + min(run, last_run)) * 2 * c.key_heads + head) * kHead; };
    const bool of_queries = wave >= 2;
    const int odd = wave & 1;
    Pair<Ask> own[4], a0[4], a1[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) own[k] = Runs<D>::row_step(run_of(wave, c.key_heads + kh), k, lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        a0[k] = Runs<D>::row_step(run_of(odd, of_queries ? kh : c.key_heads + kh), k, lane);
        a1[k] = Runs<D>::row_step(run_of(3 - odd, of_queries ? kh : c.key_heads + kh), k, lane);
    }
    {
        double sum = lane < n ? static_cast<double>(my_decay) * 1.4426950408889634 : 0.0;
        const float rate = lane < n ? my_rate : 0.0f;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const double other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        const double all = __shfl(sum, 63);
        if (wave == 0) {
            const float decay = __builtin_amdgcn_exp2f(static_cast<float>(sum)), left = __builtin_amdgcn_exp2f(static_cast<float>(all - sum));
            sums[lane] = sum;
            logs[lane] = static_cast<float>(sum);
            rates[lane] = rate;
            asked_rates[lane] = rate * decay;
            if (lane / kRun <= last_run) {  // for the launch that follows
                float *to = p.chunk_gates + ((run0 + lane / kRun) * c.value_heads + h) * (2 * kRun) + lane % kRun;
                to[0] = decay;
                to[kRun] = left;
            }
            const float lefts = wave_sum(lane < n ? left : 0.0f);
            if (lane == 0) left_sum = lefts;
        }
    }
    _Float16 *keys = reinterpret_cast<_Float16 *>(as);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        _Float16 *to = keys + wave * kHead + (k * 2 * 64 + lane) * kAsk;
        *reinterpret_cast<Ask *>(to) = own[k].h;
        *reinterpret_cast<Ask *>(to + 64 * kAsk) = own[k].l;
    }
    lds_barrier();  // keys, sums and rates
    // five products of 16 keys j and 16 rows i: run `odd` with runs 0 (and 1), run 3 - odd with the others up to its own
    f32x4_t dots[5];
    int row_run[5], key_run[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        const bool first = k <= odd;
        row_run[k] = first ? odd : 3 - odd;
        key_run[k] = first ? k : k - 1 - odd;
        dots[k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < 4; ++step) {
            const Pair<Ask> b = Runs<D>::row_step(keys + key_run[k] * kHead, step, lane);
            // only the second product may be of either
            Pair<Ask> a = k == 0 ? a0[step] : a1[step];
            if (k == 1) a = odd ? a0[step] : a1[step];
            dots[k] = product(b, a, dots[k]);
        }
        __builtin_amdgcn_sched_barrier(0);  // five products' operands at once are more registers than there are
    }
    lds_barrier();  // the keys' place is A's now
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        const int i = 16 * row_run[k] + m, j0 = 16 * key_run[k] + 4 * g;
        const double at_i = sums[i];
        const float factor = of_queries ? kProduct * kWeight : rates[i] * kProduct;
        const int past = of_queries ? i : i - 1;  // the last j that counts
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float weight = __builtin_amdgcn_exp2f(static_cast<float>(at_i - sums[j0 + e]));
            x[e] = j0 + e <= past ? weight * dots[k][e] * factor : 0.0f;
        }
        if (!of_queries) *reinterpret_cast<f32x4_t *>(as + i * kPitch + j0) = x;
        else if (row_run[k] <= last_run)
            store_four_step(p.inner + (((run0 + row_run[k]) * c.value_heads + h) * 4 + key_run[k]) * (kRun * 32), lane, split4(x));
    }
    lds_barrier();  // A

    // the inverse of a wave's block on the diagonal, a column a lane
    {
        const float *block = as + 16 * wave * kPitch + 16 * wave;
        float x[16];
        f32x4_t four[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == m ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < 15; ++j) {
            if (j % 4 == 0) {  // four columns of A
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 1; i < 16; ++i)
                    if (i > j) four[i] = *reinterpret_cast<const f32x4_t *>(block + i * kPitch + j);
            }
#pragma unroll
            for (int i = 1; i < 16; ++i)
                if (i > j) x[i] = __builtin_fmaf(-four[i][j % 4], x[j], x[i]);
        }
        float *to = ts + 16 * wave * kPitch + 16 * wave + m;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i / 4 == g) to[i * kPitch] = x[i];
    }
    // this wave's columns of V, on their way
    float *values = p.values + (run0 * c.value_heads + h) * (kRun * D) + (kTiles * wave * 64 + lane) * 4;
    const int64_t run_values = static_cast<int64_t>(c.value_heads) * (kRun * D);
    f32x4_t v[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b) v[t][b] = *reinterpret_cast<const f32x4_t *>(values + min(b, last_run) * run_values + t * 256);
    // and its key dims
    Pair4 ks[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            ks[t][b] = four_step(p.keys_by_dim + ((run0 + min(b, last_run)) * c.key_heads + kh) * kHead + (kTiles * wave + t) * (kRun * 32), lane);
    // below it: T_ij = -T_ii sum_k A_ik T_kj, a distance from the diagonal at a time
    const auto column_of = [&](int block_row, int block_column) {  // [k = 4 g + e][m]
        const float *at = ts + (16 * block_row + 4 * g) * kPitch + 16 * block_column + m;
        return f32x4_t{at[0], at[kPitch], at[2 * kPitch], at[3 * kPitch]};
    };
    const auto row_of = [&](const float *matrix, int block_row, int block_column) {  // [m][k = 4 g + e]
        return *reinterpret_cast<const f32x4_t *>(matrix + (16 * block_row + m) * kPitch + 16 * block_column + 4 * g);
    };
#pragma unroll 1
    for (int distance = 1; distance < 4; ++distance) {
        lds_barrier();
        if (wave + distance < 4) {
            const int i = wave + distance, j = wave;
            f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int k = 0; k < distance; ++k) sum = product32(row_of(as, i, j + k), column_of(j + k, j), sum);
            const f32x4_t block = product32(row_of(ts, i, i), sum, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int e = 0; e < 4; ++e) ts[(16 * i + 4 * g + e) * kPitch + 16 * j + m] = -block[e];
        }
    }
    lds_barrier();  // T
    // the columns' factors go into T
    for (int at = 4 * tid; at < kGdnChunk * kGdnChunk; at += 1024) {
        const int i = at / kGdnChunk, j = at % kGdnChunk;
        if (j / 16 > i / 16) continue;
        const f32x4_t t = *reinterpret_cast<const f32x4_t *>(ts + i * kPitch + j) * kOne;
        const Pair4 w = split4(t * *reinterpret_cast<const f32x4_t *>(asked_rates + j)), u = split4(t);
        *reinterpret_cast<f16x4_t *>(&halves[0][0][i * kPitchT + j]) = w.h;
        *reinterpret_cast<f16x4_t *>(&halves[0][1][i * kPitchT + j]) = w.l;
        *reinterpret_cast<f16x4_t *>(&halves[1][0][i * kPitchT + j]) = u.h;
        *reinterpret_cast<f16x4_t *>(&halves[1][1][i * kPitchT + j]) = u.l;
    }
    // this wave's columns of b V as operands (b is 0 behind the last row)
    float from[kTiles], largest_v[kTiles];
    Faint faint[kTiles];
    Pair4 vs[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
        for (int b = 0; b < 4; ++b) v[t][b] *= *reinterpret_cast<const f32x4_t *>(rates + 16 * b + 4 * g);
        const float most = largest_of_column(fmaxf(fmaxf(largest(v[t][0]), largest(v[t][1])), fmaxf(largest(v[t][2]), largest(v[t][3]))));
        const Scale scale(most);
        from[t] = scale.from;
#pragma unroll
        for (int b = 0; b < 4; ++b) vs[t][b] = split4(v[t][b] * scale.to);
        largest_v[t] = most;
        faint[t] = faint_rows(v[t], most, logs, n, lane);
    }
    lds_barrier();
    const auto half_at = [&](int which, int i, int b) {
        const int at = (16 * i + m) * kPitchT + 16 * b + 4 * g;
        return Pair4{*reinterpret_cast<const f16x4_t *>(&halves[which][0][at]), *reinterpret_cast<const f16x4_t *>(&halves[which][1][at])};
    };
    // of W a lane has four key dims of row m, of U four rows of value dim m
    const int lane_dim = 16 * kTiles * wave + 4 * g;
    float top[kTiles];  // of U's columns
    // where rows are faint U is made of fp32 products, which keep every row's bits
    bool exact[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        top[t] = 0.0f;
        exact[t] = __any(faint[t].last >= 0);
        if (exact[t]) top[t] = exact_updates(values + t * 256, run_values, last_run, rates, g, [&](int i, int b) { return row_of(ts, i, b); });
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i > last_run) break;
        f32x4_t w[kTiles], u[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) w[t] = u[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b <= i; ++b) {
            const Pair4 of_w = half_at(0, i, b), of_u = half_at(1, i, b);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                w[t] = product(ks[t][b], of_w, w[t]);
                u[t] = product(of_u, vs[t][b], u[t]);
            }
        }
        _Float16 *through = p.through + ((run0 + i) * c.value_heads + h) * kHead;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (!exact[t]) {
                u[t] *= from[t];
                top[t] = fmaxf(top[t], largest(u[t]));
                *reinterpret_cast<f32x4_t *>(values + i * run_values + t * 256) = u[t];
            }
            const Pair4 x = split4(w[t] * (kProduct * kOne));
            const int dim = lane_dim + 16 * t;
            _Float16 *to = through + (dim / (4 * kAsk) * 2 * 64 + dim / kAsk % 4 * 16 + m) * kAsk + dim % kAsk;
            *reinterpret_cast<f16x4_t *>(to) = x.h;
            *reinterpret_cast<f16x4_t *>(to + 64 * kAsk) = x.l;
        }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        top[t] = largest_of_column(top[t]);
        if (g == 0) {
            const int64_t at = (run0 * c.value_heads + h) * D + 16 * (kTiles * wave + t) + m;
            p.columns[at] = Column::word(top[t], left_sum, faint[t], largest_v[t], logs);
            p.faint[at] = faint[t].last;
        }
    }
}

// The state of 16 NT value dims of a head through a sequence's chunks.  In the matrix
// instructions' results a lane has value dim m and four key dims (of S) or rows (of D and
// O).  A wave has 16 rows of the chunk and a quarter of the key dims.  A chunk is a chain of
// two products with a barrier before each: 4400 cycles for one workgroup a CU (64 us for 32
// chunks), of which its 112 KB through the L1 are 1900; 68 us for eight sequences of up to
// 8 chunks and 32 heads, two workgroups a CU.
template <Dtype DT, int D, int NT>
__global__ __launch_bounds__(256, NT) void gdn_states_kernel(const GdnRowsParams p) {
    typedef typename Element<DT>::type E;
    typedef typename Runs<D>::Ask Ask;
    constexpr int kSlices = D / (16 * NT), kTiles = D / 64, kPitch = D + 8, kPitchD = kGdnChunk + 8, kAsk = Runs<D>::kAsk;
    constexpr int kHead = Runs<D>::kHead;
    // two workgroups a CU: loads stand between the products and the arithmetic, not among the products, where a CU
    // takes 64 bytes a cycle (eight prompts in all 151 -> 149 us; one workgroup by itself would lose 2 of a document's 62)
    constexpr bool kSpread = NT == 2;
    __shared__ __align__(16) _Float16 sh[2][16 * NT * kPitch], dh[2][16 * NT * kPitchD], rh[2][16 * NT * kPitchD];
    __shared__ float tops[4][16 * NT], outputs[kGdnChunk][16 * NT];  // outputs: of rows that go by themselves
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GdnView &c = p.cache;
    const GdnSequence s = gdn_sequence(p, blockIdx.y);
    if (!gdn_is_many(p, s)) return;
    // a head's slices on one die, whose L2 then serves them all
    const int blocks = gridDim.x, block = blocks % 8 == 0 ? (blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8 : blockIdx.x;
    const int h = block / kSlices, r0 = (block % kSlices) * 16 * NT;
    const int kh = h / (c.value_heads / c.key_heads);
    const int stands = p.stands[blockIdx.y];

    f32x4_t S[NT][kTiles];
    float *state = c.states + ((static_cast<int64_t>(s.slot) * c.value_heads + h) * D + r0 + m) * D + 16 * kTiles * wave + 4 * g;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            S[u][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (stands >= 0) S[u][t] = *reinterpret_cast<const f32x4_t *>(state + 16 * u * D + 16 * t);
        }
#pragma unroll 1
    for (int i = 0; i < stands; i += 2) {  // the pending rows that stand, two on their way at once
        float a[2], d[2][NT];
        f32x4_t k[2][kTiles];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t row = static_cast<int64_t>(s.slot) * c.pending + min(i + j, stands - 1);
            a[j] = c.decays[row * c.value_heads + h];
#pragma unroll
            for (int t = 0; t < NT; ++t) d[j][t] = c.updates[(row * c.value_heads + h) * D + r0 + m + 16 * t];
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                k[j][t] = *reinterpret_cast<const f32x4_t *>(c.keys + (row * c.key_heads + kh) * D + 16 * kTiles * wave + 4 * g + 16 * t);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (i + j >= stands) break;
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int t = 0; t < kTiles; ++t) S[u][t] = S[u][t] * a[j] + d[j][u] * k[j][t];
        }
    }
    if (h == 0 && r0 == 0 && tid == 0) c.counts[s.slot] = 0;

    // A chunk's operands are asked for as soon as the one before has used its own, without
    // conditions (the last chunk asks for its own again), so that no wait is for more than it
    // needs.  A wave whose rows are none asks for whatever lies behind (there is room, and nothing comes of it).
    const int64_t run_first = run_place(s, s.begin);
    const int chunks = (s.count + kGdnChunk - 1) / kGdnChunk, last_run = (s.count - 1) / kRun;
    const _Float16 *w_at = p.through + ((run_first + wave) * c.value_heads + h) * kHead;
    const _Float16 *q_at = p.asks + ((run_first + wave) * 2 * c.key_heads + kh) * kHead;
    const _Float16 *inner_at = p.inner + ((run_first + wave) * c.value_heads + h) * (4 * kRun * 32);
    const float *u_at = p.values + ((run_first + wave) * c.value_heads + h) * (kRun * D) + (r0 / 16 * 64 + lane) * 4;
    const float *gates_at = p.chunk_gates + ((run_first + wave) * c.value_heads + h) * (2 * kRun) + 4 * g;
    const uint32_t *columns_at = p.columns + (run_first * c.value_heads + h) * D + r0 + m;
    const _Float16 *keys_at = p.keys_by_dim + (run_first * c.key_heads + kh) * kHead + kTiles * wave * (kRun * 32);
    const float *whole_at = p.chunk_gates + (run_first * c.value_heads + h) * (2 * kRun);
    const int64_t w_step = static_cast<int64_t>(4) * c.value_heads * kHead, q_step = static_cast<int64_t>(8) * c.key_heads * kHead;
    const int64_t inner_step = static_cast<int64_t>(4) * c.value_heads * (4 * kRun * 32), u_step = static_cast<int64_t>(4) * c.value_heads * (kRun * D);
    const int64_t gates_step = static_cast<int64_t>(4) * c.value_heads * (2 * kRun), columns_step = static_cast<int64_t>(4) * c.value_heads * D;
    Pair<Ask> w[4], q[4];
    f32x4_t u[NT], through, left;
    float whole;
    uint32_t column[NT];
    Pair4 inner[4], keys[kTiles][4];
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto load_ask = [&](int chunk, int k) {
        w[k] = Runs<D>::row_step(w_at + chunk * w_step, k, lane);
        q[k] = Runs<D>::row_step(q_at + chunk * q_step, k, lane);
    };
    const auto load_updates = [&](int chunk) {
        through = *reinterpret_cast<const f32x4_t *>(gates_at + chunk * gates_step);
        left = *reinterpret_cast<const f32x4_t *>(gates_at + chunk * gates_step + kRun);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            u[t] = *reinterpret_cast<const f32x4_t *>(u_at + chunk * u_step + t * 256);
            column[t] = columns_at[chunk * columns_step + 16 * t];
        }
    };
    const auto load_run = [&](int chunk, int b) {
        inner[b] = four_step(inner_at + chunk * inner_step + min(b, wave) * (kRun * 32), lane);
        const int64_t run = min(4 * chunk + b, last_run);  // past it keys may be anything, and count
#pragma unroll
        for (int t = 0; t < kTiles; ++t) keys[t][b] = four_step(keys_at + run * c.key_heads * kHead + t * (kRun * 32), lane);
    };
    const auto load_whole = [&](int chunk) {
        const int row = min(s.count - 1, chunk * kGdnChunk + kGdnChunk - 1);
        whole = whole_at[static_cast<int64_t>(row / kRun) * c.value_heads * (2 * kRun) + row % kRun];
    };
    E *out = static_cast<E *>(p.out) + (s.begin + static_cast<int64_t>(16 * wave + 4 * g)) * p.out_row + h * D + r0 + m;
    // a column's largest number of this wave's part of S
    const auto top_of = [&](int t) {
        float top = largest(S[t][0]);
        if constexpr (kTiles > 1) top = fmaxf(top, largest(S[t][1]));
        return largest_of_column(top);
    };
    const auto column_top = [&](int t) {
        return fmaxf(fmaxf(tops[0][16 * t + m], tops[1][16 * t + m]), fmaxf(tops[2][16 * t + m], tops[3][16 * t + m]));
    };
    float s_to[NT], s_from[NT], s_least[NT];  // s_least: below it halves at this scale are cut short
    // the first `rows` rows of a chunk one by one, in fp32, as few rows go; the whole chunk's also leave S.  A row's asking
    // and the row before's output are one exchange between the waves, in the updates' place.
    const auto go_by_rows = [&](int chunk, int rows, bool all) {
        // places are worked out here, and nothing of them is held through the chunks
        int m = tid & 15, g = lane >> 4, h = block / kSlices, first = r0;
        asm volatile("" : "+v"(m), "+v"(g), "+s"(h), "+s"(first));
        const int kh = h / (c.value_heads / c.key_heads);
        float(*parts)[4][2][16 * NT] = reinterpret_cast<float(*)[4][2][16 * NT]>(dh);
        static_assert(sizeof(dh) >= 2 * sizeof(*parts), "two rows' exchanges");
        // U holds what the rows change of a state of nothing: `before` is what the state before them has become
        f32x4_t before[NT][kTiles], state[NT][kTiles], k[kTiles], q[kTiles], q_before[kTiles];
        Pair4 next_k[kTiles], next_q[kTiles];  // a row ahead
        float next_d[NT], next_log, next_rate;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < kTiles; ++u) before[t][u] = state[t][u] = S[t][u];
        const int64_t row0 = s.begin + static_cast<int64_t>(chunk) * kGdnChunk;
        const auto load_row = [&](int row) {
            const int64_t run = run_first + 4 * static_cast<int64_t>(chunk) + row / kRun;
            const int r = row % kRun;
            next_log = p.decay[(row0 + row) * c.value_heads + h];
            next_rate = p.rate[(row0 + row) * c.value_heads + h];
#pragma unroll
            for (int t = 0; t < NT; ++t) next_d[t] = p.values[(run * c.value_heads + h) * (kRun * D) + ((first / 16 + t) * 64 + r / 4 * 16 + m) * 4 + r % 4];
#pragma unroll
            for (int u = 0; u < kTiles; ++u) {
                const int dim = 16 * (kTiles * wave + u) + 4 * g;
                const _Float16 *at = p.asks + (run * 2 * c.key_heads + kh) * kHead + (dim / (4 * kAsk) * 2 * 64 + dim / kAsk % 4 * 16 + r) * kAsk + dim % kAsk;
                next_q[u] = {*reinterpret_cast<const f16x4_t *>(at), *reinterpret_cast<const f16x4_t *>(at + 64 * kAsk)};
                at += c.key_heads * kHead;
                next_k[u] = {*reinterpret_cast<const f16x4_t *>(at), *reinterpret_cast<const f16x4_t *>(at + 64 * kAsk)};
            }
        };
        const auto joined = [](const Pair4 &x) {
            f32x4_t y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (static_cast<float>(x.h[e]) + static_cast<float>(x.l[e])) * (1.0f / kOne);
            return y;
        };
#pragma unroll
        for (int u = 0; u < kTiles; ++u) q[u] = zero;
        load_row(0);
#pragma unroll 1
        for (int row = 0; row <= rows; ++row) {
            const float a = expf(next_log), rate = next_rate;
            float d[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) d[t] = next_d[t];
#pragma unroll
            for (int u = 0; u < kTiles; ++u) {
                q_before[u] = q[u];
                q[u] = joined(next_q[u]);
                k[u] = joined(next_k[u]);
            }
            load_row(min(row + 1, rows - 1));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x = 0.0f, y = 0.0f;
#pragma unroll
                for (int u = 0; u < kTiles; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x = __builtin_fmaf(before[t][u][e], k[u][e], x);
                        y = __builtin_fmaf(state[t][u][e], q_before[u][e], y);
                    }
                x += xor_lane<16>(x);
                y += xor_lane<16>(y);
                x += xor_lane<32>(x);
                y += xor_lane<32>(y);
                if (g == 0) {
                    parts[row & 1][wave][0][16 * t + m] = x;
                    parts[row & 1][wave][1][16 * t + m] = y;
                }
            }
            lds_barrier();
            const auto sum = [&](int which, int t) {
                const float(*part)[2][16 * NT] = parts[row & 1];
                const int at = 16 * t + m;
                return (part[0][which][at] + part[1][which][at]) + (part[2][which][at] + part[3][which][at]);
            };
            if (row > 0 && wave == 0 && g == 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) outputs[row - 1][16 * t + m] = sum(1, t);
            }
            if (row == rows) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float of_before = -rate * (a * sum(0, t)), both = d[t] + of_before;
#pragma unroll
                for (int u = 0; u < kTiles; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        before[t][u][e] = __builtin_fmaf(of_before, k[u][e], before[t][u][e] * a);
                        state[t][u][e] = __builtin_fmaf(both, k[u][e], state[t][u][e] * a);
                    }
            }
        }
        lds_barrier();  // every wave has read the last sums
        if (!all) return;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < kTiles; ++u) S[t][u] = state[t][u];
    };
    const auto store_outputs = [&](int chunk, int rows) {
        __syncthreads();  // the waves' own outputs of these rows are stored
        E *to = static_cast<E *>(p.out) + (s.begin + static_cast<int64_t>(chunk) * kGdnChunk) * p.out_row + h * D + r0;
        for (int at = tid; at < rows * 16 * NT; at += 256) to[at / (16 * NT) * p.out_row + at % (16 * NT)] = static_cast<E>(outputs[at / (16 * NT)][at % (16 * NT)]);
    };
    int chunk = 0, alone = 0;  // alone: rows of this chunk that have gone by themselves
    bool looked_at = false;    // this chunk's rows
#pragma unroll 1
    while (chunk < chunks) {
#pragma unroll
        for (int k = 0; k < 4; ++k) load_ask(chunk, k);
        load_updates(chunk);
#pragma unroll
        for (int b = 0; b < 4; ++b) load_run(chunk, b);
        load_whole(chunk);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float top = top_of(t);
            if (g == 0) tops[wave][16 * t + m] = top;
        }
        lds_barrier();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const Scale scale(column_top(t));
            s_to[t] = scale.to;
            s_from[t] = scale.from;
            s_least[t] = 0.0f;
        }
        lds_barrier();
        bool stopped = false;
        const int end = looked_at ? chunk + 1 : chunks;
#pragma unroll 1
        do {
            int mine = s.count - chunk * kGdnChunk - 16 * wave - 4 * g;  // this lane's rows that are there
            const int next = min(chunk + 1, chunks - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float top = top_of(t);
                if (g == 0) tops[wave][16 * t + m] = top;
#pragma unroll
                for (int k = 0; k < kTiles; ++k) {
                    const Pair4 x = split4(S[t][k] * s_to[t]);
                    const int at = (16 * t + m) * kPitch + 16 * (kTiles * wave + k) + 4 * g;
                    *reinterpret_cast<f16x4_t *>(&sh[0][at]) = x.h;
                    *reinterpret_cast<f16x4_t *>(&sh[1][at]) = x.l;
                }
            }
            lds_barrier();  // every wave's part of S is there

            f32x4_t asked[NT], o[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) asked[t] = o[t] = zero;
            // a step's numbers of S are read from LDS while the step before multiplies
            Pair<Ask> of_s[2][NT];
            const auto read_s = [&](int k) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int at = (16 * t + m) * kPitch + 4 * kAsk * k + kAsk * g;
                    of_s[k & 1][t] = {*reinterpret_cast<const Ask *>(&sh[0][at]), *reinterpret_cast<const Ask *>(&sh[1][at])};
                }
            };
            read_s(0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < 3) read_s(k + 1);
                __builtin_amdgcn_sched_barrier(kLoadsMayCross);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    asked[t] = product(w[k], of_s[k & 1][t], asked[t]);
                    o[t] = product(q[k], of_s[k & 1][t], o[t]);
                }
                if (!kSpread) load_ask(next, k);
            }
            if (kSpread) {
                load_ask(next, 0);
                load_ask(next, 1);
            }
            // All waves see the same numbers here and go the same way.
            bool rare = false;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const Column col(column[t]);
                const float top = column_top(t);
                rare |= col.exceeded(top) | col.wanting(top) | (top < s_least[t]);  // without branches
            }
            // Such a chunk goes through to its end without rows and changes nothing: the only way out of the loop is at its
            // end, so that no wait has to allow for another (a branch here took 7 us of 62 and 12 of 68).
            stopped = !looked_at & (__any(rare) != 0);
            mine = stopped ? 0 : mine;
            whole = stopped ? 1.0f : whole;
            float d_from[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const Column col(column[t]);
                const float top = column_top(t), most = __builtin_fmaf(top, D == 128 ? 11.32f : 8.01f, col.top) * 1.001f;
                const Scale scale(most), after(__builtin_fmaf(top, whole, col.left * most));
                f32x4_t d, d_left;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    d[e] = e < mine ? __builtin_fmaf(asked[t][e], -s_from[t], u[t][e]) : 0.0f;
                    d_left[e] = e < mine ? d[e] * left[e] : 0.0f;
                    o[t][e] *= through[e] * s_from[t];
                }
                d_from[t] = scale.from;
                s_to[t] = after.to;
                s_from[t] = after.from;
                s_least[t] = after.least;
                const Pair4 x = split4(d * scale.to), y = split4(d_left * scale.to);
                const int at = (16 * t + m) * kPitchD + 16 * wave + 4 * g;
                *reinterpret_cast<f16x4_t *>(&dh[0][at]) = x.h;
                *reinterpret_cast<f16x4_t *>(&dh[1][at]) = x.l;
                *reinterpret_cast<f16x4_t *>(&rh[0][at]) = y.h;
                *reinterpret_cast<f16x4_t *>(&rh[1][at]) = y.l;
            }
            load_updates(next);
            lds_barrier();  // every wave's updates are there, and its reads of S done
            f32x4_t added[NT][kTiles], among[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                among[t] = zero;
#pragma unroll
                for (int k = 0; k < kTiles; ++k) added[t][k] = zero;
            }
            Pair4 of_r[2][NT], of_d[2][NT];
            const auto read_d = [&](int b) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int at = (16 * t + m) * kPitchD + 16 * b + 4 * g;
                    of_r[b & 1][t] = {*reinterpret_cast<const f16x4_t *>(&rh[0][at]), *reinterpret_cast<const f16x4_t *>(&rh[1][at])};
                    of_d[b & 1][t] = {*reinterpret_cast<const f16x4_t *>(&dh[0][at]), *reinterpret_cast<const f16x4_t *>(&dh[1][at])};
                }
            };
            read_d(0);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b < 3) read_d(b + 1);
                __builtin_amdgcn_sched_barrier(kLoadsMayCross);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int k = 0; k < kTiles; ++k) added[t][k] = product(keys[k][b], of_r[b & 1][t], added[t][k]);
                    if (b <= wave) among[t] = product(inner[b], of_d[b & 1][t], among[t]);
                }
                if (!kSpread) load_run(next, b);
                else if (b >= 2) load_ask(next, b);
            }
            if (kSpread) {
                load_run(next, 0);
                load_run(next, 1);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int k = 0; k < kTiles; ++k) S[t][k][e] = __builtin_fmaf(added[t][k][e], d_from[t], S[t][k][e] * whole);
                    o[t][e] = __builtin_fmaf(among[t][e], d_from[t] * (kOne / kWeight), o[t][e]);
                }
            load_whole(next);
            if (kSpread) {
                load_run(next, 2);
                load_run(next, 3);
            }
            E *to = out + static_cast<int64_t>(chunk) * kGdnChunk * p.out_row;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= mine) continue;
#pragma unroll
                for (int t = 0; t < NT; ++t) to[e * p.out_row + 16 * t] = static_cast<E>(o[t][e]);
            }
            chunk += stopped ? 0 : 1;
        } while (!stopped & (chunk < end));
        if (!stopped) {
            if (alone > 0) store_outputs(chunk - 1, alone);
            alone = 0;
            looked_at = false;
            continue;
        }
        // a chunk with rows that go by themselves, or a bound that was too far off: from its beginning again
        const int rows = min(s.count - chunk * kGdnChunk, kGdnChunk);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int64_t at = chunk * columns_step + 16 * t;
            const Column col(columns_at[at]);
            const float top = column_top(t);
            if (col.exceeded(top)) alone = rows;
            else if (col.wanting(top)) alone = max(alone, p.faint[columns_at - p.columns + at] + 1);
        }
        alone = max(alone, xor_lane<1>(alone));
        alone = max(alone, xor_lane<2>(alone));
        alone = max(alone, xor_lane<4>(alone));
        alone = __builtin_amdgcn_readfirstlane(max(alone, xor_lane<8>(alone)));
        lds_barrier();  // every wave has read S and its largest
        if (alone > 0) go_by_rows(chunk, alone, alone >= rows);
        looked_at = alone < rows;
        if (!looked_at) {
            store_outputs(chunk, rows);
            alone = 0;
            ++chunk;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < kTiles; ++k) *reinterpret_cast<f32x4_t *>(state + 16 * t * D + 16 * k) = S[t][k];
}

template <Dtype DT, int D>
hipError_t many_typed(const GdnRowsParams &p, hipStream_t stream) {
    const GdnView &c = p.cache;
    const int parts = (c.channels() + 127) / 128 + 1;  // one more for the gates
    const dim3 runs((parts + 3) / 4, (p.batch.max_rows + kRun - 1) / kRun, p.batch.sequences);
    if (c.taps == 4 && p.pairs) hipLaunchKernelGGL((gdn_inputs_kernel<DT, D, 4, true>), runs, dim3(256), 0, stream, p);
    else if (p.pairs) hipLaunchKernelGGL((gdn_inputs_kernel<DT, D, 0, true>), runs, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_inputs_kernel<DT, D, 0, false>), runs, dim3(256), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // heads first: they go round the dies, of which each then has as many chunks
    hipLaunchKernelGGL((gdn_chunk_kernel<D>), dim3(c.value_heads, (p.batch.max_rows + kGdnChunk - 1) / kGdnChunk, p.batch.sequences),
        dim3(256), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    // 32 value dims a workgroup where that leaves two workgroups a CU: they read a chunk's operands half as often (four
    // prompts of 32 heads 79 us against 84, eight 147 against 166; two 63 against 57, a document of 16 heads 135 against 104)
    if (static_cast<int64_t>(p.batch.sequences) * c.value_heads * (D / 32) >= 512)
        hipLaunchKernelGGL((gdn_states_kernel<DT, D, 2>), dim3(c.value_heads * (D / 32), p.batch.sequences), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((gdn_states_kernel<DT, D, 1>), dim3(c.value_heads * (D / 16), p.batch.sequences), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <Dtype DT>
hipError_t many_head(const GdnRowsParams &p, hipStream_t stream) {
    return p.cache.head == 64 ? many_typed<DT, 64>(p, stream) : many_typed<DT, 128>(p, stream);
}

}  // namespace

hipError_t launch_gdn_many(const GdnRowsParams &p, Dtype dtype, hipStream_t stream) {
    if (dtype == Dtype::F32) return many_head<Dtype::F32>(p, stream);
    if (dtype == Dtype::F16) return many_head<Dtype::F16>(p, stream);
    return many_head<Dtype::BF16>(p, stream);
}

}  // namespace fortai_hip
