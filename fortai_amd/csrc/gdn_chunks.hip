// The gated delta rule over a batch's rows, for sequences of many rows (prompts): 64
// rows at a time.
//
// With c_i the sum of the chunk's logarithmic decays up to row i, S the state before the
// chunk and d_i the updates (gdn_rows.hip has the recurrence):
//   A_ij = b_i exp(c_i - c_j) k_i.k_j  (j < i)
//   (I + A) W = diag(b exp(c)) K,  (I + A) U = diag(b) V
//   D = U - W S^T,  O = diag(exp(c)) Q S^T + tril(exp(c_i - c_j) q_i.k_j) D
//   S <- exp(c_n) S + sum_j exp(c_n - c_j) d_j k_j^T
// Only the last two lines go from chunk to chunk.  Three launches: convolution, norms and
// gates of all rows; W, U and the weights of every chunk and head at once; then the
// states through their chunks, a workgroup 16 value dims of a head, whose part of S stays
// in registers.
//
// The sums c are taken in 64 bits: far into a decay they are large, and their differences
// are not.  Products are in fp32 matrix instructions.
#include "gdn_device.h"

namespace fortai_hip {

namespace {

constexpr int kRun = 16;  // rows that a wave of the first launch takes

__device__ __forceinline__ f32x4_t mfma4(f32x4_t a, f32x4_t b, f32x4_t c) {
    // the four elements are the four k indexes of lane group g, the same ones on both sides
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ bool gdn_is_many(const GdnSequence &s) { return s.count > kGdnFewRows && s.slot >= 0; }

// Convolution, norms and gates: a wave has one head of q, k or v, or every gate, of a run.
template <Dtype DT, int D>
__global__ __launch_bounds__(256) void gdn_inputs_kernel(const GdnRowsParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kMine = D / 64;
    const int lane = threadIdx.x & 63, head = blockIdx.x * 4 + (threadIdx.x >> 6), seq = blockIdx.z;
    const GdnView &c = p.cache;
    GdnSequence s = gdn_sequence(p, seq);
    if (!gdn_is_many(s)) return;
    const int i0 = blockIdx.y * kRun, rows = min(s.count - i0, kRun), heads = 2 * c.key_heads + c.value_heads;
    if (rows <= 0 || head > heads) return;
    if (head == heads) {
        for (int at = lane; at < rows * c.value_heads; at += 64) {
            const int64_t row = s.begin + i0 + at / c.value_heads;
            const int h = at % c.value_heads;
            const float alpha = static_cast<float>(static_cast<const E *>(p.alpha)[row * p.alpha_row + h]);
            const float beta = static_cast<float>(static_cast<const E *>(p.beta)[row * p.beta_row + h]);
            p.decay[row * c.value_heads + h] = gdn_log_decay(p.ssm_a[h], alpha, p.ssm_dt[h]);
            p.rate[row * c.value_heads + h] = gdn_sigmoid(beta);
        }
        return;
    }
    const int channels = c.channels(), before = c.taps - 1, first = kGdnMaxTaps - c.taps;
    if (i0 == 0) s.stands = gdn_stands(p, s);
    float x[kGdnMaxTaps - 1 + kRun][kMine], w[kGdnMaxTaps][kMine];
#pragma unroll
    for (int j = 0; j < kGdnMaxTaps - 1 + kRun; ++j) {
        const int row = i0 + j - (kGdnMaxTaps - 1);
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int channel = head * D + 64 * k + lane;
            x[j][k] = 0.0f;
            if (row >= 0) {
                x[j][k] = static_cast<float>(static_cast<const E *>(p.qkv)[(s.begin + min(row, s.count - 1)) * p.qkv_row + channel]);
            } else if (row >= -before && !s.begins) {
                x[j][k] = c.inputs[(static_cast<int64_t>(s.slot) * (before + c.pending) + s.stands + before + row) * channels + channel];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kGdnMaxTaps; ++j)
#pragma unroll
        for (int k = 0; k < kMine; ++k)
            w[j][k] = j >= first ? p.conv[static_cast<int64_t>(head * D + 64 * k + lane) * c.taps + j - first] : 0.0f;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        if (i >= rows) break;
        float y[kMine], sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            float u = 0.0f;
#pragma unroll
            for (int j = 0; j < kGdnMaxTaps; ++j)
                if (j >= first) u = __builtin_fmaf(w[j][k], x[i + j][k], u);
            y[k] = gdn_silu(u);
            sum += y[k] * y[k];
        }
        if (head < 2 * c.key_heads) {
            float inverse = 1.0f / fmaxf(sqrtf(wave_sum(sum)), p.eps);
            if (head < c.key_heads) inverse *= 1.0f / sqrtf(static_cast<float>(D));
#pragma unroll
            for (int k = 0; k < kMine; ++k) y[k] *= inverse;
        }
#pragma unroll
        for (int k = 0; k < kMine; ++k) p.rows[static_cast<int64_t>(s.begin + i0 + i) * channels + head * D + 64 * k + lane] = y[k];
    }
    if (i0 != 0) return;
    // its own channels' reads of the slot's inputs are done
#pragma unroll
    for (int k = 0; k < kMine; ++k) gdn_keep_inputs<E>(p, s, false, head * D + 64 * k + lane);
    if (head == 0 && lane == 0) p.stands[seq] = s.begins ? -1 : s.stands;
}

// W, U and the weights of one chunk and value head.
template <int D>
__global__ __launch_bounds__(256) void gdn_chunk_kernel(const GdnRowsParams p) {
    constexpr int kPitch = D + 4, kPitchA = kGdnChunk + 4;
    __shared__ __align__(16) float ks[kGdnChunk * kPitch], qs[kGdnChunk * kPitch], as[kGdnChunk * kPitchA];
    __shared__ double sums[kGdnChunk];
    __shared__ float rates[kGdnChunk];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
    const GdnView &c = p.cache;
    const GdnSequence s = gdn_sequence(p, blockIdx.z);
    if (!gdn_is_many(s)) return;
    const int n = min(s.count - static_cast<int>(blockIdx.x) * kGdnChunk, kGdnChunk), h = blockIdx.y;
    if (n <= 0) return;
    const int64_t row0 = s.begin + static_cast<int64_t>(blockIdx.x) * kGdnChunk;
    const int kh = h / (c.value_heads / c.key_heads), channels = c.channels();
    const float *base = p.rows + row0 * channels;

    // the solution's columns: one a thread, W's, then U's
    const int column = tid % (2 * D);
    const bool of_u = column >= D;
    float x[kGdnChunk];
    if (tid < 2 * D && of_u) {
        const float *v = base + (2 * c.key_heads + h) * D + column - D;
#pragma unroll
        for (int i = 0; i < kGdnChunk; ++i) x[i] = v[static_cast<int64_t>(min(i, n - 1)) * channels];
    }
    for (int at = 4 * tid; at < kGdnChunk * D; at += 1024) {
        const int i = at / D, d = at % D;
        f32x4_t q = {0.0f, 0.0f, 0.0f, 0.0f}, k = q;
        if (i < n) {
            q = *reinterpret_cast<const f32x4_t *>(base + static_cast<int64_t>(i) * channels + kh * D + d);
            k = *reinterpret_cast<const f32x4_t *>(base + static_cast<int64_t>(i) * channels + (c.key_heads + kh) * D + d);
        }
        *reinterpret_cast<f32x4_t *>(qs + i * kPitch + d) = q;
        *reinterpret_cast<f32x4_t *>(ks + i * kPitch + d) = k;
    }
    if (wave == 0) {
        const int64_t at = (row0 + min(lane, n - 1)) * c.value_heads + h;
        double sum = lane < n ? static_cast<double>(p.decay[at]) : 0.0;
        const float rate = lane < n ? p.rate[at] : 0.0f;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const double other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        sums[lane] = sum;
        rates[lane] = rate;
        const double all = __shfl(sum, 63);
        if (lane < n) {  // for the launch that follows
            p.decay[at] = expf(static_cast<float>(sum));
            p.rate[at] = expf(static_cast<float>(all - sum));
        }
    }
    __syncthreads();

    // k_i.k_j and q_i.k_j of 16 rows i a wave, 16 columns j at a time
    const int i_of = 16 * wave + 4 * g;
#pragma unroll 1
    for (int tile = 0; tile <= wave; ++tile) {
        f32x4_t kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = kk;
#pragma unroll
        for (int d = 0; d < D; d += 16) {
            const f32x4_t b = *reinterpret_cast<const f32x4_t *>(ks + (16 * tile + m) * kPitch + d + 4 * g);
            kk = mfma4(*reinterpret_cast<const f32x4_t *>(ks + (16 * wave + m) * kPitch + d + 4 * g), b, kk);
            qk = mfma4(*reinterpret_cast<const f32x4_t *>(qs + (16 * wave + m) * kPitch + d + 4 * g), b, qk);
        }
        const int j = 16 * tile + m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = i_of + e;
            const float weight = j <= i ? expf(static_cast<float>(sums[i] - sums[j])) : 0.0f;
            as[i * kPitchA + j] = j < i ? rates[i] * weight * kk[e] : 0.0f;
            if (i < n) p.inner[((row0 + i) * c.value_heads + h) * kGdnChunk + j] = weight * qk[e];
        }
    }
    __syncthreads();

    if (tid >= 2 * D) return;
#pragma unroll
    for (int i = 0; i < kGdnChunk; ++i) {
        if (!of_u) x[i] = ks[i * kPitch + column] * expf(static_cast<float>(sums[i]));
        x[i] *= rates[i];
    }
#pragma unroll
    for (int i = 1; i < kGdnChunk; ++i) {
#pragma unroll
        for (int j = 0; j < i; j += 4) {
            const f32x4_t a = *reinterpret_cast<const f32x4_t *>(as + i * kPitchA + j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < i) x[i] = __builtin_fmaf(-a[e], x[j + e], x[i]);
        }
    }
    if (of_u) {
        float *v = p.rows + row0 * channels + (2 * c.key_heads + h) * D + column - D;
#pragma unroll
        for (int i = 0; i < kGdnChunk; ++i)
            if (i < n) v[static_cast<int64_t>(i) * channels] = x[i];
    } else {
        float *w = p.through + (row0 * c.value_heads + h) * D + column;
#pragma unroll
        for (int i = 0; i < kGdnChunk; ++i)
            if (i < n) w[static_cast<int64_t>(i) * c.value_heads * D] = x[i];
    }
}

// The state of 16 value dims of a head through a sequence's chunks.  In the matrix
// instructions' results a lane has value dim m and four key dims (of S) or rows (of D and O).
template <Dtype DT, int D>
__global__ __launch_bounds__(256) void gdn_states_kernel(const GdnRowsParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kSlices = D / 16, kTiles = D / 64, kPitch = D + 4, kPitchD = kGdnChunk + 4;
    __shared__ __align__(16) float ss[16 * kPitch], ds[16 * kPitchD], rest[16 * kPitchD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
    const GdnView &c = p.cache;
    const GdnSequence s = gdn_sequence(p, blockIdx.y);
    if (!gdn_is_many(s)) return;
    const int blocks = gridDim.x, block = blocks % 8 == 0 ? (blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8 : blockIdx.x;
    const int h = block / kSlices, r0 = (block % kSlices) * 16;
    const int kh = h / (c.value_heads / c.key_heads), channels = c.channels();
    const int stands = p.stands[blockIdx.y];

    f32x4_t S[kTiles];
    float *state = c.states + ((static_cast<int64_t>(s.slot) * c.value_heads + h) * D + r0 + m) * D + 16 * kTiles * wave + 4 * g;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        S[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (stands >= 0) S[t] = *reinterpret_cast<const f32x4_t *>(state + 16 * t);
    }
#pragma unroll 1
    for (int i = 0; i < stands; ++i) {  // the pending rows that stand
        const int64_t row = static_cast<int64_t>(s.slot) * c.pending + i;
        const float a = c.decays[row * c.value_heads + h], d = c.updates[(row * c.value_heads + h) * D + r0 + m];
        const float *k = c.keys + (row * c.key_heads + kh) * D + 16 * kTiles * wave + 4 * g;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) S[t] = S[t] * a + d * *reinterpret_cast<const f32x4_t *>(k + 16 * t);
    }
    if (h == 0 && r0 == 0 && tid == 0) c.counts[s.slot] = 0;

    f32x4_t w[D / 16], q[D / 16];
    const auto load_asked = [&](int64_t row0, int n) {
        const int64_t row = row0 + min(16 * wave + m, n - 1);
        const float *w_at = p.through + (row * c.value_heads + h) * D + 4 * g;
        const float *q_at = p.rows + row * channels + kh * D + 4 * g;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            w[d] = *reinterpret_cast<const f32x4_t *>(w_at + 16 * d);
            q[d] = *reinterpret_cast<const f32x4_t *>(q_at + 16 * d);
        }
    };
    load_asked(s.begin, min(s.count, kGdnChunk));
#pragma unroll 1
    for (int i0 = 0; i0 < s.count; i0 += kGdnChunk) {
        const int n = min(s.count - i0, kGdnChunk);
        const int64_t row0 = s.begin + i0;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) *reinterpret_cast<f32x4_t *>(ss + m * kPitch + 16 * (kTiles * wave + t) + 4 * g) = S[t];
        // what the chunk needs later on
        float u[4], through[4], left[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t row = row0 + min(16 * wave + 4 * g + e, n - 1);
            u[e] = p.rows[row * channels + (2 * c.key_heads + h) * D + r0 + m];
            through[e] = p.decay[row * c.value_heads + h];
            left[e] = p.rate[row * c.value_heads + h];
        }
        const float whole = p.decay[(row0 + n - 1) * c.value_heads + h];
        f32x4_t inner[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
            inner[t] = *reinterpret_cast<const f32x4_t *>(p.inner + ((row0 + min(16 * wave + m, n - 1)) * c.value_heads + h) * kGdnChunk +
                16 * min(t, wave) + 4 * g);
        f32x4_t k[kTiles][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    k[t][b][e] = p.rows[(row0 + min(16 * b + 4 * g + e, n - 1)) * channels + (c.key_heads + kh) * D +
                        16 * (kTiles * wave + t) + m];
        __syncthreads();  // every wave's part of S is there

        f32x4_t asked = {0.0f, 0.0f, 0.0f, 0.0f}, o = asked;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const f32x4_t b = *reinterpret_cast<const f32x4_t *>(ss + m * kPitch + 16 * d + 4 * g);
            asked = mfma4(w[d], b, asked);
            o = mfma4(q[d], b, o);
        }
        if (i0 + kGdnChunk < s.count) load_asked(row0 + kGdnChunk, min(s.count - i0 - kGdnChunk, kGdnChunk));
        f32x4_t d, d_left;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            d[e] = 16 * wave + 4 * g + e < n ? u[e] - asked[e] : 0.0f;
            d_left[e] = d[e] * left[e];
            o[e] *= through[e];
        }
        *reinterpret_cast<f32x4_t *>(ds + m * kPitchD + 16 * wave + 4 * g) = d;
        *reinterpret_cast<f32x4_t *>(rest + m * kPitchD + 16 * wave + 4 * g) = d_left;
        __syncthreads();  // every wave's updates are there, and its reads of S done
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (t <= wave) o = mfma4(inner[t], *reinterpret_cast<const f32x4_t *>(ds + m * kPitchD + 16 * t + 4 * g), o);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) S[t] *= whole;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f32x4_t updates = *reinterpret_cast<const f32x4_t *>(rest + m * kPitchD + 16 * b + 4 * g);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) S[t] = mfma4(k[t][b], updates, S[t]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 16 * wave + 4 * g + e;
            if (i < n) static_cast<E *>(p.out)[(row0 + i) * p.out_row + h * D + r0 + m] = static_cast<E>(o[e]);
        }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) *reinterpret_cast<f32x4_t *>(state + 16 * t) = S[t];
}

template <Dtype DT, int D>
hipError_t many_typed(const GdnRowsParams &p, hipStream_t stream) {
    const GdnView &c = p.cache;
    const int heads = 2 * c.key_heads + c.value_heads + 1;  // one more for the gates
    hipLaunchKernelGGL((gdn_inputs_kernel<DT, D>), dim3((heads + 3) / 4, (p.batch.max_rows + kRun - 1) / kRun, p.batch.sequences),
        dim3(256), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((gdn_chunk_kernel<D>), dim3((p.batch.max_rows + kGdnChunk - 1) / kGdnChunk, c.value_heads, p.batch.sequences),
        dim3(256), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((gdn_states_kernel<DT, D>), dim3(c.value_heads * (D / 16), p.batch.sequences), dim3(256), 0, stream, p);
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
