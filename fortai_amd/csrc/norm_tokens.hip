// Residual sum, norm and gate of rows, into the 8-bit tokens that the token
// products take.
//
//   h = x + r, rounded to the arrays' type
//   y = h w / sqrt(mean_group(h^2) + eps) * z / (1 + exp(-z))
//   a block of 32 values, m = max |y|: scale fp16(m / 127), codes the integers
//   nearest to 127 y / m
//
// A code has to be the nearest integer, and in 32 bits one in some 10^4 values falls on the
// other side of a half, so y is computed in 64 bits; the quotient is rounded to 32 bits
// before it is rounded to an integer, so that quotients that are halves but for the
// rounding of y (where gates are equal) go to the even code whatever the order of the
// arithmetic.  That hides behind the memory but for the gate's exponential, which took 46 us
// of 64 bits for 2000 rows of 4096 in bf16: gated values are computed in 32 bits first, and
// again in 64 where a quotient of the wave's 256 may lie on either side of a half for all
// that 32 bits say, or a scale on either side of a border of fp16 (one wave in eight): 22 us.
//
// Bound by memory: rows of up to 4096 stay in registers from the sum to the codes (4096 rows
// of 2560 in fp32 with a sum, 138 MB: 31 us, 4.4 TB/s; read twice 39 us; a wave a row, which
// needs no barrier but has a long piece of code to go through, 33 to 34 us).
#include "fortai_hip_internal.h"
#include "step_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kNormThreads = 256;

__device__ __forceinline__ double block_top(double top) {
    top = fmax(top, xor_lane<1>(top));
    top = fmax(top, xor_lane<2>(top));
    return fmax(top, xor_lane<4>(top));
}
__device__ __forceinline__ float block_top(float top) {
    top = fmaxf(top, xor_lane<1>(top));
    top = fmaxf(top, xor_lane<2>(top));
    return fmaxf(top, xor_lane<4>(top));
}

// z / (1 + exp(-z)) to 7 2^-24 of itself for z above -80: the exponent's product with log2 e
// in two parts, the power and the reciprocal each to the last place
__device__ __forceinline__ float silu_close(float z) {
    const float t = fminf(z * -1.44269504f, 126.0f), rest = __builtin_fmaf(z, -1.44269504f, -t) + z * -1.92596303e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, rest * 0.693147181f, e));
}

struct Codes {
    uint32_t codes;
    float scale;
};

// ROW_WAVES waves a row: sums stay within a wave, or go through LDS.  HELD: 256-value
// pieces that a wave has at most, which then stay in registers; 0: any.  Where the norm is
// of parts of a row or there is none, blockIdx.y has the row's next HELD pieces.
// With a gate the loop over pieces is not unrolled, the held ones move down instead: a row
// of 4096 by one wave in 16 copies of that code (64 KB) took 37 us.
template <Dtype DT, bool VEC, int ROW_WAVES, int HELD, bool GATE>
__global__ __launch_bounds__(kNormThreads) void norm_tokens_kernel(NormTokensParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kRowThreads = ROW_WAVES * 64, kRows = kNormThreads / kRowThreads;
    __shared__ double sums[ROW_WAVES];
    const int thread = threadIdx.x % kRowThreads, lane = threadIdx.x & 63;
    const int row = blockIdx.x * kRows + threadIdx.x / kRowThreads;
    if (row >= p.rows) return;  // whole waves; with ROW_WAVES > 1 a workgroup has one row
    const E *x = static_cast<const E *>(p.x) + static_cast<int64_t>(row) * p.x_row;
    const E *residual = static_cast<const E *>(p.residual) + (p.residual ? static_cast<int64_t>(row) * p.residual_row : 0);
    const E *gate = static_cast<const E *>(p.gate) + (GATE ? static_cast<int64_t>(row) * p.gate_row : 0);
    E *sum = static_cast<E *>(p.sum) + (p.sum ? static_cast<int64_t>(row) * p.sum_row : 0);
    E *out = static_cast<E *>(p.out) + (p.out ? static_cast<int64_t>(row) * p.out_row : 0);
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};

    const auto load_h = [&](int i) {
        f32x4_t h = load4<DT, VEC>(x + i);
        if (p.residual) {
            h += load4<DT, VEC>(residual + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = static_cast<float>(static_cast<E>(h[k]));
        }
        return h;
    };
    const auto squares = [](f32x4_t h) {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) s += static_cast<double>(h[k]) * static_cast<double>(h[k]);
        return s;
    };
    // a wave's pieces: thread's values from 4 thread + piece * 4 kRowThreads on
    const int start = HELD > 0 ? static_cast<int>(blockIdx.y) * HELD * 4 * kRowThreads : 0;
    const auto place = [&](int piece) { return start + 4 * thread + piece * 4 * kRowThreads; };
    f32x4_t held[HELD > 0 ? HELD : 1];
    const bool whole = p.norm && p.group == p.width;
    double inverse = 1.0;
    if (HELD > 0) {
#pragma unroll
        for (int piece = 0; piece < HELD; ++piece) held[piece] = place(piece) < p.width ? load_h(place(piece)) : zero;
    }
    if (whole || p.sum) {
        double total = 0.0;
        if (HELD > 0) {
#pragma unroll
            for (int piece = 0; piece < HELD; ++piece) {
                total += squares(held[piece]);
                if (p.sum && place(piece) < p.width) store4<DT, VEC>(sum + place(piece), held[piece]);
            }
        } else {
            for (int i = 4 * thread; i < p.width; i += 4 * kRowThreads) {
                const f32x4_t h = load_h(i);
                total += squares(h);
                if (p.sum) store4<DT, VEC>(sum + i, h);
            }
        }
        if (whole) {
            total = wave_sum(total);
            if constexpr (ROW_WAVES > 1) {
                if (lane == 0) sums[threadIdx.x >> 6] = total;
                __syncthreads();
                total = sums[0];
#pragma unroll
                for (int w = 1; w < ROW_WAVES; ++w) total += sums[w];
            }
            inverse = 1.0 / sqrt(total / p.width + static_cast<double>(p.eps));
        }
    }

    const int padded = p.codes ? p.blocks_pad * 32 : p.width;
    const auto load_w = [&](int i) {
        const float *at = p.norm + (i < p.width ? (whole ? i : i & (p.group - 1)) : 0);
        return f32x4_t{at[0], at[1], at[2], at[3]};
    };
    const auto load_z = [&](int i) { return i < p.width ? load4<DT, VEC>(gate + i) : zero; };
    const auto piece_of = [&](int i, f32x4_t h, f32x4_t w, f32x4_t z) {
        const bool mine = i < p.width;
        if (p.norm && !whole) inverse = 1.0 / sqrt(group_sum_up(squares(h), p.group / 4) / p.group + static_cast<double>(p.eps));
        f32x4_t y32;
        Codes c = {0, 0.0f};
        bool close = !GATE;  // to a border, for all that 32 bits say
        if constexpr (GATE) {
            // y is off by at most 11 2^-24 of itself (the inverse, silu's seven, three products), the quotient by
            // 24 2^-24 127 = 1.8e-4, the scale by 15 2^-24.  Numbers near the ends of 32 bits are left to 64: within
            // these limits an intermediate result that 32 bits flush belongs to a quotient below 0.2.
            const float inverse32 = static_cast<float>(inverse);
            close = !(inverse32 > 1e-30f && inverse32 < 1e30f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                y32[k] = (h[k] * inverse32) * w[k] * silu_close(z[k]);
                close = close || !(fabsf(w[k]) < 1e5f && z[k] > -80.0f && z[k] < 1e5f);
            }
            const float top = block_top(fmaxf(fmaxf(fabsf(y32[0]), fabsf(y32[1])), fmaxf(fabsf(y32[2]), fabsf(y32[3]))));
            const float to_code = 127.0f / top, scale = top * (1.0f / 127.0f);
            close = close || !(top > 1e-25f && top < 1e25f);
            const _Float16 over = static_cast<_Float16>(scale * (1.0f + 0x1p-19f)), under = static_cast<_Float16>(scale * (1.0f - 0x1p-19f));
            close = close || over != under;
            c.scale = static_cast<float>(over);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float q = y32[k] * to_code, code = __builtin_rintf(q);
                close = close || !(fabsf(q - code) < 0.5f - 2.5e-4f);
                c.codes |= (static_cast<uint32_t>(static_cast<int>(code)) & 0xffu) << (8 * k);
            }
            close = __any(close || p.out);  // the output is rounded from 64 bits too
        }
        if (close) {
            double y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                y[k] = static_cast<double>(h[k]) * static_cast<double>(w[k]);
                if (p.norm) y[k] *= inverse;
                if constexpr (GATE) y[k] *= static_cast<double>(z[k]) / (1.0 + exp(-static_cast<double>(z[k])));
                if (!mine) y[k] = 0.0;
            }
            if (p.out && mine)
                store4<DT, VEC>(out + i, f32x4_t{static_cast<float>(y[0]), static_cast<float>(y[1]), static_cast<float>(y[2]), static_cast<float>(y[3])});
            const double top = block_top(fmax(fmax(fabs(y[0]), fabs(y[1])), fmax(fabs(y[2]), fabs(y[3]))));
            // fmax drops a NaN: a block that has one keeps it in its scale
            float poison = static_cast<float>((y[0] + y[1] + y[2] + y[3]) * 0.0);
            poison += xor_lane<1>(poison);
            poison += xor_lane<2>(poison);
            poison += xor_lane<4>(poison);
            const double to_code = top > 0.0 ? 127.0 / top : 0.0;
            c.codes = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float q = __builtin_rintf(static_cast<float>(y[k] * to_code));
                c.codes |= (static_cast<uint32_t>(q == q ? static_cast<int>(q) : 0) & 0xffu) << (8 * k);
            }
            c.scale = static_cast<float>(static_cast<_Float16>(static_cast<float>(top / 127.0))) + poison;
        }
        const int block = i >> 5;
        if (!p.codes || block >= p.blocks_pad) return;
        const size_t at = static_cast<size_t>(block) * p.ld + row;
        reinterpret_cast<uint32_t *>(p.codes)[at * 8 + (lane & 7)] = c.codes;
        if ((lane & 7) == 0) p.scales[at] = c.scale;
    };
    // the trip count is the wave's, so that every lane takes part in its block's maximum
    f32x4_t w = {1.0f, 1.0f, 1.0f, 1.0f}, z = zero;
    if (HELD > 0) {
        if (p.norm) w = load_w(place(0));
        if (GATE) z = load_z(place(0));
#pragma unroll(GATE ? 1 : HELD)
        for (int piece = 0; piece < HELD && place(piece) - 4 * lane < padded; ++piece) {
            const f32x4_t h = held[0], w_now = w, z_now = z;
            if (p.norm) w = load_w(place(piece + 1));
            if (GATE) z = load_z(place(piece + 1));
#pragma unroll
            for (int k = 0; k + 1 < HELD; ++k) held[k] = held[k + 1];
            piece_of(place(piece), h, w_now, z_now);
        }
    } else {
        for (int base = 4 * (thread - lane); base < padded; base += 4 * kRowThreads) {
            const int i = base + 4 * lane;
            if (p.norm) w = load_w(i);
            if (GATE) z = load_z(i);
            // with a sum, what this thread stored above
            piece_of(i, i < p.width ? (p.sum ? load4<DT, VEC>(sum + i) : load_h(i)) : zero, w, z);
        }
    }
}

// Four rows a workgroup: their codes of a block are 128 bytes in a row.  A wave has two
// blocks at a time, four codes a lane.
template <Dtype DT, bool VEC>
__global__ __launch_bounds__(256) void tokens_read_kernel(const int8_t *codes, const float *scales, int ld, int rows, int width,
    void *out, int64_t out_row) {
    typedef typename Element<DT>::type E;
    constexpr int kAtOnce = 4;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (lane >> 3 & 3), blocks = width / 32;
    const int first = (threadIdx.x >> 6) * 2 + (lane >> 5);
    E *to = static_cast<E *>(out) + static_cast<int64_t>(min(row, rows - 1)) * out_row + 4 * (lane & 7);
    for (int block0 = first; block0 < blocks; block0 += 8 * kAtOnce) {
        uint32_t c[kAtOnce];
        float scale[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const size_t at = static_cast<size_t>(min(block0 + 8 * k, blocks - 1)) * ld + row;  // rows up to ld are there
            c[k] = reinterpret_cast<const uint32_t *>(codes)[at * 8 + (lane & 7)];
            scale[k] = scales[at];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (block0 + 8 * k >= blocks || row >= rows) continue;
            f32x4_t y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(static_cast<int8_t>(c[k] >> (8 * e))) * scale[k];
            store4<DT, VEC>(to + (block0 + 8 * k) * 32, y);
        }
    }
}

template <Dtype DT, bool VEC, int ROW_WAVES, int HELD>
void norm_rows(const NormTokensParams &p, int columns, hipStream_t stream) {
    const dim3 grid((p.rows + 4 / ROW_WAVES - 1) / (4 / ROW_WAVES), columns), block(kNormThreads);
    if (p.gate) hipLaunchKernelGGL((norm_tokens_kernel<DT, VEC, ROW_WAVES, HELD, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((norm_tokens_kernel<DT, VEC, ROW_WAVES, HELD, false>), grid, block, 0, stream, p);
}

template <Dtype DT>
hipError_t norm_typed(const NormTokensParams &p, bool vec, hipStream_t stream) {
    // parts of rows are nobody else's: a wave has 256 values of a row (2000 rows of 4096, gated: 22 us, with 512 25,
    // with 1024 27: the fewer registers, the more waves a SIMD has to choose from); a whole row's norm takes
    // a workgroup, which reads rows again that are longer than it holds, or not aligned
    const int padded = p.codes ? p.blocks_pad * 32 : p.width;
    if (!vec) norm_rows<DT, false, 4, 0>(p, 1, stream);
    else if (!p.norm || p.group < p.width) norm_rows<DT, true, 1, 1>(p, (padded + 255) / 256, stream);
    else if (p.width <= 4096) norm_rows<DT, true, 4, 4>(p, 1, stream);
    else norm_rows<DT, true, 4, 0>(p, 1, stream);
    return hipGetLastError();
}

template <Dtype DT>
hipError_t read_typed(const int8_t *codes, const float *scales, int ld, int rows, int width, void *out, int64_t out_row,
    bool vec, hipStream_t stream) {
    const dim3 grid((rows + 3) / 4);
    if (vec) hipLaunchKernelGGL((tokens_read_kernel<DT, true>), grid, dim3(256), 0, stream, codes, scales, ld, rows, width, out, out_row);
    else hipLaunchKernelGGL((tokens_read_kernel<DT, false>), grid, dim3(256), 0, stream, codes, scales, ld, rows, width, out, out_row);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_norm_tokens(const NormTokensParams &p, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) return norm_typed<Dtype::F32>(p, vec, stream);
    if (dtype == Dtype::F16) return norm_typed<Dtype::F16>(p, vec, stream);
    return norm_typed<Dtype::BF16>(p, vec, stream);
}

hipError_t launch_tokens_read(const int8_t *codes, const float *scales, int ld, int rows, int width, void *out,
    int64_t out_row, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) return read_typed<Dtype::F32>(codes, scales, ld, rows, width, out, out_row, vec, stream);
    if (dtype == Dtype::F16) return read_typed<Dtype::F16>(codes, scales, ld, rows, width, out, out_row, vec, stream);
    return read_typed<Dtype::BF16>(codes, scales, ld, rows, width, out, out_row, vec, stream);
}

}  // namespace fortai_hip
