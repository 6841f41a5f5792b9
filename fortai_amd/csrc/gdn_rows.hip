// The gated delta rule over a batch's rows, for sequences of few rows (decode steps
// and drafts), and the slots' copies.
//
//   u = sum_i w_i x_{t - taps + 1 + i}, y = u / (1 + exp(-u))        per channel: q, k, v
//   q = y_q / max(|y_q|, eps) / sqrt(head), k = y_k / max(|y_k|, eps)
//   a = exp(ssm_a softplus(alpha + ssm_dt)), b = 1 / (1 + exp(-beta))
//   d = b (v - a S k),  S = a S + d k^T,  o = S q
//
// Rows that wait: S is stored as it stands before them, their k, d and a beside it.
// The next call applies those that stand while S is in registers: one read and one
// write of S a step, whether drafts stand or not.
//
// Bound by memory: a step reads and writes S, 128 KiB a head of 128, for 7 operations a
// value.  A workgroup has ROWS rows of one head's S, eight lanes a row, a lane four
// columns of every 32: the products with k and q are sums over a lane's columns and three
// exchanges between neighbours, and nothing of S goes through LDS.  The convolution of
// the head's q and k, 2 head channels, is done by every workgroup of the head again
// instead of a launch of its own.  What bounds it in fact is the chain of dependent loads (row starts, slot,
// count, pending rows) in front of the arithmetic: all loads of a stage are asked for before the first
// is waited for.  Eight sequences of one row, 16 heads of 128: 8.3 us for 17 MB; of up to five rows and five
// pending ones, 32 heads, bf16: 14.9 us for 34 MB; 64 of one row, 32 heads, 50 us for 268 MB.
//
// Who may overwrite what others read: the inputs and keys of a key head are read by all
// its workgroups.  Each counts itself in once its reads are done, and the last one
// writes; the slot's count likewise for the whole sequence.  Nothing that one workgroup
// writes is read by another, so a plain count is enough.
#include "gdn_device.h"

namespace fortai_hip {

namespace {

// TAPS: 4 or, 0, as many as the cache says.
template <Dtype DT, int D, int ROWS, int TAPS>
__global__ __launch_bounds__(ROWS * 8) void gdn_few_kernel(const GdnRowsParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kThreads = ROWS * 8, kWaves = kThreads / 64, kFours = D / 32, kBlocks = D / ROWS;
    constexpr int kChannels = 2 * D + ROWS, kTurns = (kChannels + kThreads - 1) / kThreads;
    constexpr int kAtOnce = 4;  // a thread's rows of a channel on their way at once
    __shared__ __align__(16) float qs[kGdnFewRows][D], ks[kGdnFewRows][D], log_k[kGdnMaxPending][D];
    __shared__ float vs[kGdnFewRows][ROWS], log_d[kGdnMaxPending][ROWS], os[kGdnFewRows][ROWS], ds[kGdnFewRows][ROWS];
    __shared__ float rates[kGdnFewRows], decays[kGdnFewRows], log_a[kGdnMaxPending];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const GdnView &c = p.cache;
    GdnSequence s = gdn_sequence(p, blockIdx.y);
    if (s.count == 0 || s.count > kGdnFewRows || s.slot < 0) return;
    const int r = s.count, h = blockIdx.x / kBlocks, block = blockIdx.x % kBlocks, r0 = block * ROWS;
    const int group = c.value_heads / c.key_heads, kh = h / group, channels = c.channels(), before = c.taps - 1;
    const bool waits = r <= c.pending;

    // Everything is asked for before anything is waited for: the rows' inputs and weights of this workgroup's
    // channels, a thread's row of S, then what needs the number of pending rows that stand.
    const auto channel_of = [&](int at) {
        return at < D ? kh * D + at : at < 2 * D ? (c.key_heads + kh) * D + at - D : (2 * c.key_heads + h) * D + r0 + at - 2 * D;
    };
    constexpr int kTaps = TAPS > 0 ? TAPS : kGdnMaxTaps;
    const int first = TAPS > 0 ? 0 : kGdnMaxTaps - c.taps;  // aligned to the newest: seen[kTaps - 1] is the row's own
    const E *x[kTurns];
    float seen[kTurns][kTaps], w[kTurns][kTaps], next[kTurns][kAtOnce];
    const auto load_rows = [&](int row) {
#pragma unroll
        for (int turn = 0; turn < kTurns; ++turn)
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) next[turn][k] = static_cast<float>(x[turn][min(row + k, r - 1) * p.qkv_row]);
    };
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn) {
        const int channel = channel_of(min(turn * kThreads + tid, kChannels - 1));
        x[turn] = static_cast<const E *>(p.qkv) + static_cast<int64_t>(s.begin) * p.qkv_row + channel;
#pragma unroll
        for (int j = 0; j < kTaps; ++j) w[turn][j] = p.conv[static_cast<int64_t>(channel) * c.taps + max(j - first, 0)];
    }
    load_rows(0);
    const int gate_row = s.begin + min(tid, r - 1);
    const E alpha = static_cast<const E *>(p.alpha)[static_cast<int64_t>(gate_row) * p.alpha_row + h];
    const E beta = static_cast<const E *>(p.beta)[static_cast<int64_t>(gate_row) * p.beta_row + h];
    const int local = tid >> 3, l = tid & 7;
    f32x4_t S[kFours];
    float *state = c.states + ((static_cast<int64_t>(s.slot) * c.value_heads + h) * D + r0 + local) * D + 4 * l;
#pragma unroll
    for (int f = 0; f < kFours; ++f) S[f] = *reinterpret_cast<const f32x4_t *>(state + 32 * f);
    s.stands = gdn_stands(p, s);
    const int stands = s.begins ? 0 : s.stands;
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn) {
        const int channel = channel_of(min(turn * kThreads + tid, kChannels - 1));
        const float *window = c.inputs + static_cast<int64_t>(s.slot) * (before + c.pending) * channels + channel;
#pragma unroll
        for (int j = 0; j + 1 < kTaps; ++j) seen[turn][j] = window[static_cast<int64_t>(stands + max(j - first, 0)) * channels];
    }
    // the pending rows that stand
    if (stands > 0) {
        const int64_t row0 = static_cast<int64_t>(s.slot) * c.pending;
        const float *keys = c.keys + (row0 * c.key_heads + kh) * D, *updates = c.updates + (row0 * c.value_heads + h) * D + r0;
        const int64_t key_row = static_cast<int64_t>(c.key_heads) * D, update_row = static_cast<int64_t>(c.value_heads) * D;
        const int all = stands * D, few = stands * ROWS;
        const int at_d = min(tid, few - 1);
        const float d = updates[at_d / ROWS * update_row + at_d % ROWS];
        const float a = c.decays[(row0 + min(tid, stands - 1)) * c.value_heads + h];
#pragma unroll 1
        for (int base = tid; base < all; base += 4 * kThreads) {
            float k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = min(base + i * kThreads, all - 1);
                k[i] = keys[at / D * key_row + at % D];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (base + i * kThreads < all) log_k[0][base + i * kThreads] = k[i];
        }
        if (tid < few) log_d[0][tid] = d;
        for (int at = tid + kThreads; at < few; at += kThreads) log_d[0][at] = updates[at / ROWS * update_row + at % ROWS];
        if (tid < stands) log_a[tid] = a;
    }
    // the rows' gates
    if (tid < r) {
        rates[tid] = gdn_sigmoid(static_cast<float>(beta));
        decays[tid] = expf(gdn_log_decay(p.ssm_a[h], static_cast<float>(alpha), p.ssm_dt[h]));
    }
    // the convolution
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn)
#pragma unroll
        for (int j = 0; j + 1 < kTaps; ++j) {
            if (s.begins || j < first) seen[turn][j] = 0.0f;
            if (j < first) w[turn][j] = 0.0f;
        }
#pragma unroll 1
    for (int i = 0; i < r; i += kAtOnce) {
        float now[kTurns][kAtOnce];
#pragma unroll
        for (int turn = 0; turn < kTurns; ++turn)
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) now[turn][k] = next[turn][k];
        if (i + kAtOnce < r) load_rows(i + kAtOnce);
#pragma unroll
        for (int turn = 0; turn < kTurns; ++turn) {
            const int at = turn * kThreads + tid;
            if (at >= kChannels) break;
            float *to = at < D ? &qs[0][at] : at < 2 * D ? &ks[0][at - D] : &vs[0][at - 2 * D];
            const int pitch = at < 2 * D ? D : ROWS;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (i + k >= r) break;
                seen[turn][kTaps - 1] = now[turn][k];
                float u = 0.0f;
#pragma unroll
                for (int j = 0; j < kTaps; ++j) u = __builtin_fmaf(w[turn][j], seen[turn][j], u);
                to[(i + k) * pitch] = gdn_silu(u);
#pragma unroll
                for (int j = 0; j + 1 < kTaps; ++j) seen[turn][j] = seen[turn][j + 1];
            }
        }
    }
    __syncthreads();
    // every read of what others may overwrite has its data
    int arrived = 0;
    int *arrivals = p.arrivals + static_cast<int64_t>(blockIdx.y) * (c.key_heads + 1);
    if (tid == 0) arrived = __hip_atomic_fetch_add(arrivals + kh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // norms, a row's q or k a wave at a time
    for (int i = wave; i < 2 * r; i += kWaves) {
        float *v = i < r ? qs[i] : ks[i - r];
        float x[D / 64], sum = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            x[k] = v[64 * k + lane];
            sum += x[k] * x[k];
        }
        sum = wave_sum(sum);
        float eps = p.eps;
        if (gdn_length_is_lost(sum, eps)) {
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 64; ++k) top = fmaxf(top, fabsf(x[k]));
            const int e = __builtin_amdgcn_frexp_expf(wave_max(top));
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                x[k] = __builtin_ldexpf(x[k], -e);
                sum += x[k] * x[k];
            }
            sum = wave_sum(sum);
            eps = __builtin_ldexpf(eps, -e);
        }
        float inverse = 1.0f / fmaxf(sqrtf(sum), eps);
        if (i < r) inverse *= 1.0f / sqrtf(static_cast<float>(D));
#pragma unroll
        for (int k = 0; k < D / 64; ++k) v[64 * k + lane] = x[k] * inverse;
    }
    __syncthreads();

    if (s.begins) {
#pragma unroll
        for (int f = 0; f < kFours; ++f) S[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll 1
    for (int i = 0; i < stands; ++i) {
        const float a = log_a[i], d = log_d[i][local];
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const f32x4_t k = *reinterpret_cast<const f32x4_t *>(&log_k[i][32 * f + 4 * l]);
#pragma unroll
            for (int e = 0; e < 4; ++e) S[f][e] = __builtin_fmaf(d, k[e], S[f][e] * a);
        }
    }
    if (waits && (stands > 0 || s.begins)) {
#pragma unroll
        for (int f = 0; f < kFours; ++f) *reinterpret_cast<f32x4_t *>(state + 32 * f) = S[f];
    }
#pragma unroll 1
    for (int i = 0; i < r; ++i) {
        const float a = decays[i];
        f32x4_t k[kFours];
        float asked = 0.0f;
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            k[f] = *reinterpret_cast<const f32x4_t *>(&ks[i][32 * f + 4 * l]);
            S[f] *= a;
#pragma unroll
            for (int e = 0; e < 4; ++e) asked = __builtin_fmaf(S[f][e], k[f][e], asked);
        }
        asked = group_sum_up(asked, 8);
        const float d = rates[i] * (vs[i][local] - asked);
        float o = 0.0f;
#pragma unroll
        for (int f = 0; f < kFours; ++f) {
            const f32x4_t q = *reinterpret_cast<const f32x4_t *>(&qs[i][32 * f + 4 * l]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[f][e] = __builtin_fmaf(d, k[f][e], S[f][e]);
                o = __builtin_fmaf(S[f][e], q[e], o);
            }
        }
        o = group_sum_up(o, 8);
        if (l == 0) {
            os[i][local] = o;
            ds[i][local] = d;
        }
    }
    if (!waits) {
#pragma unroll
        for (int f = 0; f < kFours; ++f) *reinterpret_cast<f32x4_t *>(state + 32 * f) = S[f];
    }
    if (tid == 0) {
        last = arrived == group * kBlocks - 1;
        if (last) __hip_atomic_store(arrivals + kh, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    for (int at = tid; at < r * ROWS; at += kThreads) {
        const int i = at / ROWS, local_row = at % ROWS;
        static_cast<E *>(p.out)[(s.begin + i) * p.out_row + h * D + r0 + local_row] = static_cast<E>(os[i][local_row]);
        if (waits)
            c.updates[((static_cast<int64_t>(s.slot) * c.pending + i) * c.value_heads + h) * D + r0 + local_row] = ds[i][local_row];
    }
    // this workgroup's own channels, and as the last of its key head the ones it shares
    if (tid < ROWS) gdn_keep_inputs<E>(p, s, waits, channel_of(2 * D + tid));
    if (!last) return;
    for (int at = tid; at < 2 * D; at += kThreads) gdn_keep_inputs<E>(p, s, waits, channel_of(at));
    if (waits) {
        for (int at = tid; at < r * D; at += kThreads)
            c.keys[((static_cast<int64_t>(s.slot) * c.pending + at / D) * c.key_heads + kh) * D + at % D] = ks[at / D][at % D];
        for (int at = tid; at < r * group; at += kThreads) {
            const int i = at / group, head = kh * group + at % group;
            const float alpha = static_cast<float>(static_cast<const E *>(p.alpha)[(s.begin + i) * p.alpha_row + head]);
            c.decays[(static_cast<int64_t>(s.slot) * c.pending + i) * c.value_heads + head] =
                expf(gdn_log_decay(p.ssm_a[head], alpha, p.ssm_dt[head]));
        }
    }
    if (tid == 0) {
        int *heads = arrivals + c.key_heads;
        if (__hip_atomic_fetch_add(heads, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == c.key_heads - 1) {
            __hip_atomic_store(heads, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            c.counts[s.slot] = waits ? r : 0;
        }
    }
}

struct SlotPairs {
    int32_t from[kKv8PairsPerLaunch], to[kKv8PairsPerLaunch];
};

// planes of `count` floats a slot, one behind the other, [layers][slots][count] each
__global__ __launch_bounds__(256) void gdn_copy_slots_kernel(float *plane, int64_t count, int slots, SlotPairs pairs) {
    const int64_t layer = static_cast<int64_t>(blockIdx.z) * slots;
    const float *from = plane + (layer + pairs.from[blockIdx.y]) * count;
    float *to = plane + (layer + pairs.to[blockIdx.y]) * count;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += step) to[i] = from[i];
}

template <Dtype DT, int D, int TAPS>
hipError_t few_typed(const GdnRowsParams &p, hipStream_t stream) {
    const GdnView &c = p.cache;
    // Fewer rows of S a workgroup do the convolution more often, and win nothing where there are few workgroups: one
    // sequence of 16 heads 8.4 us with 16 rows, 7.5 with 32, 7.6 with 64, 7.3 with 128; eight of up to five rows and 32
    // heads 28, 17.0, 14.9 and 14.7; 64 of one row and 32 heads with 32 rows 56, 50 and 52.
    constexpr int kRows = 64;
    hipLaunchKernelGGL((gdn_few_kernel<DT, D, kRows, TAPS>), dim3(c.value_heads * (D / kRows), p.batch.sequences), dim3(kRows * 8), 0, stream, p);
    return hipGetLastError();
}

template <Dtype DT>
hipError_t few_head(const GdnRowsParams &p, hipStream_t stream) {
    if (p.cache.taps == 4) return p.cache.head == 64 ? few_typed<DT, 64, 4>(p, stream) : few_typed<DT, 128, 4>(p, stream);
    return p.cache.head == 64 ? few_typed<DT, 64, 0>(p, stream) : few_typed<DT, 128, 0>(p, stream);
}

}  // namespace

hipError_t launch_gdn_few(const GdnRowsParams &p, Dtype dtype, hipStream_t stream) {
    if (dtype == Dtype::F32) return few_head<Dtype::F32>(p, stream);
    if (dtype == Dtype::F16) return few_head<Dtype::F16>(p, stream);
    return few_head<Dtype::BF16>(p, stream);
}

hipError_t launch_gdn_copy_slots(const GdnView &c, int layers, const int32_t *from, const int32_t *to, int count, hipStream_t stream) {
    const int64_t d = c.head;
    struct Plane {
        float *at;
        int64_t count;
    } planes[6] = {{c.states, c.value_heads * d * d}, {c.inputs, static_cast<int64_t>(c.taps - 1 + c.pending) * c.channels()},
        {c.keys, c.pending * c.key_heads * d}, {c.updates, c.pending * c.value_heads * d},
        {c.decays, static_cast<int64_t>(c.pending) * c.value_heads}, {reinterpret_cast<float *>(c.counts), 1}};
    for (int at = 0; at < count; at += kKv8PairsPerLaunch) {
        const int n = count - at < kKv8PairsPerLaunch ? count - at : kKv8PairsPerLaunch;
        SlotPairs pairs = {};
        for (int i = 0; i < n; ++i) {
            pairs.from[i] = from[at + i];
            pairs.to[i] = to[at + i];
        }
        for (const Plane &plane : planes) {
            if (plane.count == 0) continue;
            const int64_t wanted = (plane.count + 1023) / 1024;
            const dim3 grid(static_cast<unsigned>(wanted < 1024 ? wanted : 1024), n, layers);
            hipLaunchKernelGGL(gdn_copy_slots_kernel, grid, dim3(256), 0, stream, plane.at, plane.count, c.slots, pairs);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace fortai_hip
