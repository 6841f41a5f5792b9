// Residual sum, norm and gate of rows, into the 8-bit tokens that the token
// products take.
//
//   h = x + r, rounded to the arrays' type
//   y = h w / sqrt(mean_group(h^2) + eps) * z / (1 + exp(-z))
//   a block of 32 values, m = max |y|: scale fp16(m / 127), codes the integers
//   nearest to 127 y / m
//
// All in 64 bits: a code is a border between integers away from the next one, and
// in 32 bits one in some 10^5 values falls on the other side.  The quotient is
// rounded to 32 bits before it is rounded to an integer, so that quotients that are
// halves but for the rounding of y (where gates are equal) go to the even code
// whatever the order of the arithmetic.  The chip has half the rate of fp32 for it
// and this is bound by memory.
#include "fortai_hip_internal.h"
#include "step_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kNormThreads = 256;

// ROW_WAVES waves a row: sums stay within a wave, or go through LDS.
template <Dtype DT, bool VEC, int ROW_WAVES>
__global__ __launch_bounds__(kNormThreads) void norm_tokens_kernel(NormTokensParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kRowThreads = ROW_WAVES * 64, kRows = kNormThreads / kRowThreads;
    __shared__ double sums[ROW_WAVES];
    const int thread = threadIdx.x % kRowThreads, lane = threadIdx.x & 63;
    const int row = blockIdx.x * kRows + threadIdx.x / kRowThreads;
    if (row >= p.rows) return;  // whole waves; with ROW_WAVES > 1 a workgroup has one row
    const E *x = static_cast<const E *>(p.x) + static_cast<int64_t>(row) * p.x_row;
    const E *residual = static_cast<const E *>(p.residual) + (p.residual ? static_cast<int64_t>(row) * p.residual_row : 0);
    const E *gate = static_cast<const E *>(p.gate) + (p.gate ? static_cast<int64_t>(row) * p.gate_row : 0);
    E *sum = static_cast<E *>(p.sum) + (p.sum ? static_cast<int64_t>(row) * p.sum_row : 0);
    E *out = static_cast<E *>(p.out) + (p.out ? static_cast<int64_t>(row) * p.out_row : 0);

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
    const bool whole = p.norm && p.group == p.width;
    double inverse = 1.0;
    if (whole || p.sum) {
        double total = 0.0;
        for (int i = 4 * thread; i < p.width; i += 4 * kRowThreads) {
            const f32x4_t h = load_h(i);
            total += squares(h);
            if (p.sum) store4<DT, VEC>(sum + i, h);
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
    // the trip count is the wave's, so that every lane takes part in its block's maximum
    const int padded = p.codes ? p.blocks_pad * 32 : p.width;
    for (int base = 4 * (thread - lane); base < padded; base += 4 * kRowThreads) {
        const int i = base + 4 * lane;
        const bool mine = i < p.width;
        f32x4_t h = {0.0f, 0.0f, 0.0f, 0.0f};
        // what this thread stored above
        if (mine) h = p.sum ? load4<DT, VEC>(sum + i) : load_h(i);
        double y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = static_cast<double>(h[k]);
        if (p.norm) {
            if (!whole) inverse = 1.0 / sqrt(group_sum_up(squares(h), p.group / 4) / p.group + static_cast<double>(p.eps));
            const int at = whole ? i : i & (p.group - 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] *= static_cast<double>(mine ? p.norm[at + k] : 0.0f) * inverse;
        }
        if (p.gate && mine) {
            const f32x4_t z = load4<DT, VEC>(gate + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] *= static_cast<double>(z[k]) / (1.0 + exp(-static_cast<double>(z[k])));
        }
        if (p.out && mine)
            store4<DT, VEC>(out + i, f32x4_t{static_cast<float>(y[0]), static_cast<float>(y[1]), static_cast<float>(y[2]), static_cast<float>(y[3])});
        if (!p.codes) continue;
        double top = fmax(fmax(fabs(y[0]), fabs(y[1])), fmax(fabs(y[2]), fabs(y[3])));
        // fmax drops a NaN: a block that has one keeps it in its scale
        double poison = (y[0] + y[1] + y[2] + y[3]) * 0.0;
        top = fmax(top, xor_lane<1>(top));
        top = fmax(top, xor_lane<2>(top));
        top = fmax(top, xor_lane<4>(top));
        poison += xor_lane<1>(poison);
        poison += xor_lane<2>(poison);
        poison += xor_lane<4>(poison);
        const double to_code = top > 0.0 ? 127.0 / top : 0.0;
        uint32_t codes = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float q = __builtin_rintf(static_cast<float>(y[k] * to_code));
            codes |= (static_cast<uint32_t>(q == q ? static_cast<int>(q) : 0) & 0xffu) << (8 * k);
        }
        const int block = i >> 5;
        if (block >= p.blocks_pad) continue;
        const size_t at = static_cast<size_t>(block) * p.ld + row;
        reinterpret_cast<uint32_t *>(p.codes)[at * 8 + (lane & 7)] = codes;
        if ((lane & 7) == 0)
            p.scales[at] = static_cast<float>(static_cast<_Float16>(static_cast<float>(top / 127.0))) + static_cast<float>(poison);
    }
}

// One workgroup a row, four values a thread at a time.
template <Dtype DT, bool VEC>
__global__ __launch_bounds__(256) void tokens_read_kernel(const int8_t *codes, const float *scales, int ld, int width,
    void *out, int64_t out_row) {
    typedef typename Element<DT>::type E;
    const int row = blockIdx.x;
    for (int i = 4 * threadIdx.x; i < width; i += 1024) {
        const size_t at = static_cast<size_t>(i >> 5) * ld + row;
        const uint32_t c = reinterpret_cast<const uint32_t *>(codes)[at * 8 + ((i >> 2) & 7)];
        const float scale = scales[at];
        f32x4_t y;
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = static_cast<float>(static_cast<int8_t>(c >> (8 * k))) * scale;
        store4<DT, VEC>(static_cast<E *>(out) + row * out_row + i, y);
    }
}

template <Dtype DT>
hipError_t norm_typed(const NormTokensParams &p, bool vec, hipStream_t stream) {
    const dim3 block(kNormThreads);
    if (p.rows >= 1024) {
        const dim3 grid((p.rows + 3) / 4);
        if (vec) hipLaunchKernelGGL((norm_tokens_kernel<DT, true, 1>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((norm_tokens_kernel<DT, false, 1>), grid, block, 0, stream, p);
    } else {
        if (vec) hipLaunchKernelGGL((norm_tokens_kernel<DT, true, 4>), dim3(p.rows), block, 0, stream, p);
        else hipLaunchKernelGGL((norm_tokens_kernel<DT, false, 4>), dim3(p.rows), block, 0, stream, p);
    }
    return hipGetLastError();
}

template <Dtype DT>
hipError_t read_typed(const int8_t *codes, const float *scales, int ld, int rows, int width, void *out, int64_t out_row,
    bool vec, hipStream_t stream) {
    if (vec) hipLaunchKernelGGL((tokens_read_kernel<DT, true>), dim3(rows), dim3(256), 0, stream, codes, scales, ld, width, out, out_row);
    else hipLaunchKernelGGL((tokens_read_kernel<DT, false>), dim3(rows), dim3(256), 0, stream, codes, scales, ld, width, out, out_row);
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
