// Rotary positions of query and key heads, with the RMSNorm that the model has
// in front of them.
//
//   y = x / sqrt(mean(x^2) + eps) * w           (per head; only with w)
//   (a, b) -> (a c - b s, a s + b c)            c = f cos(p theta_i), s = f sin(p theta_i)
//
// for the pairs i of the first `rotary` dims: (i, i + rotary / 2) in the half
// layout, (2 i, 2 i + 1) interleaved.  The angle is taken in turns in 64 bits,
// p * (theta_i / 2 pi), and only its fraction is rounded to fp32: at position
// 10^6 an fp32 angle would be off by 0.03 rad.
//
// Bound by memory: every value is read and written once for a handful of
// operations.  A group of LPH lanes holds one head's vector, four values a
// lane, so the norm's sum is a lane butterfly and nothing goes through LDS; the
// partner dims of the half layout are read a second time (the same wave has
// just fetched their lines).  A workgroup works out its row's sines and cosines once
// and keeps them for all the heads that it walks, kHeadsAtOnce of them in flight.
// 4096 rows of 20 heads of 128 (bf16, 42 MB): 11.4 us, 3.7 TB/s; 16.0 when every lane
// worked out the angles of its own dims.  Eight rows: 4.5 us.
#include "element_types.h"
#include "fortai_hip_internal.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kRopeWaves = 4;
constexpr int kHeadsAtOnce = 4;

template <Dtype DT, int LPH, bool INTERLEAVED, bool VEC>
__global__ __launch_bounds__(kRopeWaves * 64) void rope_kernel(RopeParams p) {
    typedef typename Element<DT>::type E;
    constexpr int HPW = 64 / LPH;  // heads a wave holds at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, d = (lane % LPH) * 4, r = p.rotary, half = r / 2;
    const bool mine = d < p.head;  // heads of fewer than 4 LPH dims leave lanes idle
    const E *x = static_cast<const E *>(p.x) + static_cast<int64_t>(row) * p.x_row;
    E *out = static_cast<E *>(p.out) + static_cast<int64_t>(row) * p.out_row;

    // this lane's four dims: the partner's dim, the sine with its sign, the norm's weights
    float c[4], s[4], w[4], wp[4];
    int partner[4], pairs[4];
    float signs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = d + i;
        const bool turned = mine && e < r;
        bool second;
        int pair;
        if constexpr (INTERLEAVED) {
            second = i & 1;
            pair = e >> 1;
            partner[i] = e ^ 1;
        } else {
            second = e >= half;
            pair = second ? e - half : e;
            partner[i] = second ? e - half : e + half;
        }
        pairs[i] = turned ? pair : -1;
        signs[i] = second ? 1.0f : -1.0f;
        if (!turned) partner[i] = mine ? e : 0;
        w[i] = p.norm && mine ? p.norm[e] : 1.0f;
        wp[i] = p.norm ? p.norm[partner[i]] : 1.0f;
    }
    const bool rotates = mine && d < r;

    const int stride = gridDim.y * kRopeWaves * HPW;
    const int first = (blockIdx.y * kRopeWaves + wave) * HPW + lane / LPH;
    // the trip count is the wave's, so that every lane takes part in the norm's sum
    int base = first - lane / LPH;
    f32x4_t v[kHeadsAtOnce], b[kHeadsAtOnce];
    const auto load_heads = [&]() {
#pragma unroll
        for (int k = 0; k < kHeadsAtOnce; ++k) {
            const int h = base + lane / LPH + k * stride;
            v[k] = b[k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (mine && h < p.heads) {
                const E *at = x + static_cast<int64_t>(h) * p.x_head;
                v[k] = load4<DT, VEC>(at + d);
                if constexpr (INTERLEAVED) {
                    b[k] = f32x4_t{v[k][1], v[k][0], v[k][3], v[k][2]};
                } else if (rotates) {
                    if (VEC && p.half4) {  // rotary / 2 a multiple of 4: the partners are four in a row
                        b[k] = load4<DT, VEC>(at + partner[0]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) b[k][i] = static_cast<float>(at[partner[i]]);
                    }
                }
            }
        }
    };
    load_heads();
    __shared__ float2 angles[128];
    // the row's angles, a pair a thread
    if (static_cast<int>(threadIdx.x) < half) {
        const double turns = static_cast<double>(p.positions[row]) * p.turns[threadIdx.x];
        float sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - __builtin_rint(turns)), &sine, &cosine);
        angles[threadIdx.x] = make_float2(cosine * p.attention, sine * p.attention);
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 angle = angles[max(pairs[i], 0)];
        c[i] = pairs[i] < 0 ? 1.0f : angle.x;
        s[i] = pairs[i] < 0 ? 0.0f : angle.y * signs[i];
    }
#pragma unroll 1
    while (base < p.heads) {
#pragma unroll
        for (int k = 0; k < kHeadsAtOnce; ++k) {
            const int h = base + lane / LPH + k * stride;
            if (p.norm) {
                float sum = (v[k][0] * v[k][0] + v[k][1] * v[k][1]) + (v[k][2] * v[k][2] + v[k][3] * v[k][3]);
                sum = group_sum_up(sum, LPH);
                const float inverse = 1.0f / sqrtf(sum / static_cast<float>(p.head) + p.eps);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[k][i] = v[k][i] * inverse * w[i];
                    b[k][i] = b[k][i] * inverse * wp[i];
                }
            }
            f32x4_t y = v[k];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d + i < r) y[i] = v[k][i] * c[i] + b[k][i] * s[i];
            if (mine && h < p.heads) store4<DT, VEC>(out + static_cast<int64_t>(h) * p.out_head + d, y);
        }
        base += stride * kHeadsAtOnce;
        load_heads();
    }
}

template <Dtype DT, int LPH>
void rope_variant(const RopeParams &p, bool vec, dim3 grid, hipStream_t stream) {
    const dim3 block(kRopeWaves * 64);
    if (p.interleaved) {
        if (vec) hipLaunchKernelGGL((rope_kernel<DT, LPH, true, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((rope_kernel<DT, LPH, true, false>), grid, block, 0, stream, p);
    } else {
        if (vec) hipLaunchKernelGGL((rope_kernel<DT, LPH, false, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((rope_kernel<DT, LPH, false, false>), grid, block, 0, stream, p);
    }
}

template <Dtype DT>
void rope_typed(const RopeParams &p, bool vec, hipStream_t stream) {
    const int lph = p.head <= 64 ? 16 : p.head <= 128 ? 32 : 64;
    // heads side by side until the chip is full, then walked by the waves of one row
    const int groups = (p.heads + kRopeWaves * (64 / lph) - 1) / (kRopeWaves * (64 / lph));
    const int wanted = (2048 + p.rows - 1) / p.rows;
    const dim3 grid(p.rows, groups < wanted ? groups : wanted);
    if (lph == 16) rope_variant<DT, 16>(p, vec, grid, stream);
    else if (lph == 32) rope_variant<DT, 32>(p, vec, grid, stream);
    else rope_variant<DT, 64>(p, vec, grid, stream);
}

}  // namespace

hipError_t launch_rope(const RopeParams &p, Dtype dtype, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) rope_typed<Dtype::F32>(p, vec, stream);
    else if (dtype == Dtype::F16) rope_typed<Dtype::F16>(p, vec, stream);
    else rope_typed<Dtype::BF16>(p, vec, stream);
    return hipGetLastError();
}

}  // namespace fortai_hip
