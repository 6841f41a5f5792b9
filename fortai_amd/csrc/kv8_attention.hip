// Attention over the 8-bit paged cache.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j [* sigmoid(gate)],  p_j = exp(scale q.k_j - max)
//
// over the tokens j <= lengths[s] + t of row t's sequence, k_j = codes * (A_k / 127)
// and v_j = codes * (A_v / 127) with one A per page and head.
//
// One pass over the cache with a running maximum.  The rows of a kv head (tokens
// x heads of its group) are the columns of 16-wide matrix instructions, its
// cached tokens the rows:
//   S^T [token][row] = K Q^T,   O^T [dim][row] += V^T P^T
// in v_mfma_f32_16x16x32_f16, the codes turned into fp16 (exact) in registers.
// A tile is 64 tokens.  Lane (r = lane & 15, g = lane >> 4) of tile part u (0..3)
// feeds key token 16 (r >> 2) + 4 u + (r & 3), so that S leaves the instruction
// with lane group g holding the 16 consecutive tokens 16 g .. 16 g + 15 of row r:
// those are exactly the value codes that lane reads as one 16-byte word per dim
// (pages are [dim][token]), in the order in which the next instruction takes its
// k index.  Neither P nor a code ever goes through LDS.
//
// Numerics.  A row of q is scaled by a power of two to a magnitude below 1 and
// rounded to fp16.  With SPLIT the 16 columns are 8 rows and, in the other 8, what
// that rounding left over (times 2^11), and p is split the same way, so that
// products keep 22 bits: used for fp32 queries, and where no more than 8 rows are
// there to fill the columns.  Without it p is one fp16 number (2^-11 of itself).
// A_v enters the running maximum by its exponent: the numerator's terms are
// p_j A_v / 127, and what is rounded to fp16 is that product over the largest such
// product (times 2^14, away from fp16's subnormals), so that pages of very
// different magnitude lose nothing against each other.  All sums are fp32.
//
// Bound by the cache's bytes for few rows: 32 KiB of codes a tile and head of 256.
// The four waves of a workgroup take tiles in turn; `splits` workgroups share a
// sequence's head, joined by a second launch.
#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int kTileTokens = 64;
constexpr int kWaves = 4;
constexpr float kLoScale = 2048.0f;          // 2^11: the left-over halves of a split
constexpr float kPScale = 16384.0f;          // 2^14

// 8 codes as fp16: with the sign bit turned a code is code + 128, which under the
// exponent byte 0x64 reads 1024 + code + 128.
__device__ __forceinline__ f16x8_t codes_to_half(uint32_t a, uint32_t b) {
    const f16x2_t bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const f16x2_t p0 = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + bias;
    const f16x2_t p1 = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + bias;
    const f16x2_t p2 = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + bias;
    const f16x2_t p3 = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + bias;
    return f16x8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// exponent that A_v adds to the running maximum, and what is left of A_v
__device__ __forceinline__ int value_exponent(float top) { return min(max(__builtin_amdgcn_frexp_expf(top), -100), 100); }

template <Dtype DT>
__device__ __forceinline__ float gated(float y, const typename Element<DT>::type *gate) {
    const float g = static_cast<float>(*gate);
    return y / (1.0f + expf(-g));
}

// The rows of one sequence: the first in the batch's arrays, how many of a kv head; how many tokens the last row
// that a workgroup holds sees, and tiles of them.
struct RowTile {
    int begin, total, length, seen, tiles;
};

__device__ __forceinline__ RowTile row_tile(const Kv8AttentionParams &p, int seq, int first_row, int rows) {
    RowTile t;
    int count;
    p.batch.range(seq, &t.begin, &count);
    t.total = count * p.group;
    t.length = p.batch.length(seq);
    const int last = min(first_row + rows, t.total) - 1;
    t.seen = last < first_row ? 0 : min(t.length + last / p.group + 1, p.batch.pitch * p.cache.page_tokens);
    t.tiles = t.seen <= 0 ? 0 : (t.seen + kTileTokens - 1) / kTileTokens;
    return t;
}

template <int D, Dtype DT, bool SPLIT, int RT>
__global__ __launch_bounds__(kWaves * 64, RT == 1 ? 2 : 1) void kv8_attention_kernel(Kv8AttentionParams p) {
    typedef typename Element<DT>::type E;
    constexpr int kCols = SPLIT ? 8 : 16;           // rows in an instruction's 16 columns
    constexpr int kRows = kCols * RT;
    constexpr int kChunks = D / 64, kDims = D / 16;
    __shared__ f32x4_t join[kWaves][RT][kDims][4 * kCols];
    __shared__ float join_m[kWaves][kRows], join_l[kWaves][kRows];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int seq = blockIdx.z, kvh = blockIdx.y % p.cache.kv_heads, row0 = (blockIdx.y / p.cache.kv_heads) * kRows;
    const int split = blockIdx.x;
    const RowTile tile = row_tile(p, seq, row0, kRows);
    if (row0 >= tile.total) return;
    if (split > 0 && split * kWaves >= tile.tiles) return;  // the join does not look at it

    // ---- queries: column r's row, as fp16 halves
    const int col = SPLIT ? r & 7 : r;
    const bool low = SPLIT && r >= 8;
    f16x8_t q[RT][kChunks][2];
    float factor[RT];  // of S: softmax scale, log2 e, the query's power of two, 1 / 127
    int position[RT];  // the last token that the row sees
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = row0 + t * kCols + col;
        const bool there = row < tile.total;
        const int token = there ? row / p.group : 0, head = kvh * p.group + (there ? row % p.group : 0);
        const E *at = static_cast<const E *>(p.q) + static_cast<int64_t>(tile.begin + token) * p.q_row +
            static_cast<int64_t>(head) * p.q_head + 16 * g;
        position[t] = there ? tile.length + token : -1;
        f32x4_t v[kChunks][4];
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[c][k] = p.vec ? load4<DT, true>(at + 64 * c + 4 * k) : load4<DT, false>(at + 64 * c + 4 * k);
                top = fmaxf(top, fmaxf(fmaxf(fabsf(v[c][k][0]), fabsf(v[c][k][1])), fmaxf(fabsf(v[c][k][2]), fabsf(v[c][k][3]))));
            }
        top = fmaxf(top, xor_lane<16>(top));
        top = fmaxf(top, xor_lane<32>(top));
        const int e = __builtin_amdgcn_frexp_expf(top);
        factor[t] = __builtin_ldexpf(p.scale_log2, e);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_ldexpf(v[c][k][i], -e);
                    const _Float16 hi = static_cast<_Float16>(x);
                    const _Float16 lo = static_cast<_Float16>((x - static_cast<float>(hi)) * kLoScale);
                    q[t][c][k >> 1][(k & 1) * 4 + i] = low ? lo : hi;
                }
    }

    const int P = p.cache.page_tokens;
    const size_t page_stride = static_cast<size_t>(p.cache.kv_heads) * P * D;
    const int8_t *keys = p.cache.keys + static_cast<size_t>(kvh) * P * D + 16 * g;
    const int8_t *values = p.cache.values + static_cast<size_t>(kvh) * P * D + static_cast<size_t>(r) * P;
    const float *key_max = p.cache.key_max + kvh, *value_max = p.cache.value_max + kvh;
    const float share = SPLIT ? (low ? 1.0f / kLoScale : 1.0f) : 1.0f;

    f32x4_t o[RT][kDims];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[t][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int step = p.splits * kWaves;
    const int first = split * kWaves + wave;
    // pages of this lane's key tokens (16 (r >> 2) ..) and of its value tokens (16 g ..)
    int key_page = p.batch.page(seq, (first * kTileTokens + 16 * (r >> 2)) / P, p.cache.pages);
    int value_page = p.batch.page(seq, (first * kTileTokens + 16 * g) / P, p.cache.pages);
    u32x4_t k[4][kChunks];
    if (first < tile.tiles) {
        const int8_t *at = keys + static_cast<size_t>(max(key_page, 0)) * page_stride;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
                k[u][c] = *reinterpret_cast<const u32x4_t *>(
                    at + ((first * kTileTokens + 16 * (r >> 2) + 4 * u + (r & 3)) % P) * D + 64 * c);
    }
    for (int n = first; n < tile.tiles; n += step) {
        const int token = n * kTileTokens + 16 * g;  // the first of this lane's 16
        const int page = max(value_page, 0);
        u32x4_t v[kDims];
        const int8_t *at = values + static_cast<size_t>(page) * page_stride + token % P;
#pragma unroll
        for (int d = 0; d < kDims; ++d) v[d] = *reinterpret_cast<const u32x4_t *>(at + static_cast<size_t>(16 * d) * P);
        // a page that holds no token yet may hold anything: its magnitudes are not used, and its codes are
        // finite whatever they are
        const bool there = value_page >= 0 && token < tile.seen;
        float key_top = key_max[static_cast<size_t>(page) * p.cache.kv_heads];
        float value_top = value_max[static_cast<size_t>(page) * p.cache.kv_heads];
        key_top = there ? key_top : 0.0f;
        value_top = there ? value_top : 0.0f;
        // the next tile's pages
        const int next = n + step;
        key_page = p.batch.page(seq, (next * kTileTokens + 16 * (r >> 2)) / P, p.cache.pages);
        value_page = p.batch.page(seq, (next * kTileTokens + 16 * g) / P, p.cache.pages);

        f32x4_t s[RT][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int t = 0; t < RT; ++t) s[t][u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const f16x8_t a0 = codes_to_half(k[u][c][0], k[u][c][1]), a1 = codes_to_half(k[u][c][2], k[u][c][3]);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, q[t][c][0], s[t][u], 0, 0, 0);
                    s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, q[t][c][1], s[t][u], 0, 0, 0);
                }
            }
        }
        if (next < tile.tiles) {
            const int8_t *from = keys + static_cast<size_t>(max(key_page, 0)) * page_stride;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    k[u][c] = *reinterpret_cast<const u32x4_t *>(
                        from + ((next * kTileTokens + 16 * (r >> 2) + 4 * u + (r & 3)) % P) * D + 64 * c);
        }

        const int exponent = value_exponent(value_top);
        const float shift = static_cast<float>(exponent);
        const float inverse = __builtin_ldexpf(1.0f, -exponent), rest = __builtin_ldexpf(value_top, -exponent) * kPScale;
        f16x8_t b[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float f = factor[t] * key_top;
            const int seen = there ? position[t] + 1 - token : 0;  // of this lane's 16 tokens
            float x[16];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float y = s[t][u][i];
                    if constexpr (SPLIT) {
                        y = y * share;
                        y = y + xor_lane<8>(y);
                    }
                    x[4 * u + i] = __builtin_fmaf(y, f, shift);
                }
            if (__any(seen < 16)) {
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = j < seen ? x[j] : -__builtin_inff();
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]);
            top = fmaxf(top, xor_lane<16>(top));
            top = fmaxf(top, xor_lane<32>(top));
            const float now = fmaxf(m[t], top);
            const float base = now == -__builtin_inff() ? 0.0f : now;  // nothing seen yet: p = 0, not exp(nan)
            const float alpha = exp2_fast(m[t] - base);
            m[t] = now;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = exp2_fast(x[j] - base);
                sum += e;
                const float y = e * rest;
                _Float16 h = static_cast<_Float16>(y);
                if constexpr (SPLIT) {
                    const _Float16 left = static_cast<_Float16>((y - static_cast<float>(h)) * kLoScale);
                    h = low ? left : h;
                }
                b[t][j >> 3][j & 7] = h;
            }
            l[t] = l[t] * alpha + sum * inverse;
            if (__any(alpha != 1.0f)) {
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[t][d][i] *= alpha;
            }
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            const f16x8_t a0 = codes_to_half(v[d][0], v[d][1]), a1 = codes_to_half(v[d][2], v[d][3]);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b[t][0], o[t][d], 0, 0, 0);
                o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b[t][1], o[t][d], 0, 0, 0);
            }
        }
    }

    // ---- join the waves
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] += xor_lane<16>(l[t]);
        l[t] += xor_lane<32>(l[t]);
        if (g == 0 && !low) {
            join_m[wave][t * kCols + col] = m[t];
            join_l[wave][t * kCols + col] = l[t];
        }
    }
    __syncthreads();
    float total[RT], top[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = t * kCols + col;
        top[t] = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top[t] = fmaxf(top[t], join_m[w][row]);
        const float base = top[t] == -__builtin_inff() ? 0.0f : top[t];
        total[t] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total[t] += join_l[w][row] * exp2_fast(join_m[w][row] - base);
        const float mine = exp2_fast(m[t] - base) * share;
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            f32x4_t y = o[t][d] * mine;
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = y[i] + xor_lane<8>(y[i]);
            }
            if (!low) join[wave][t][d][g * kCols + col] = y;
        }
    }
    __syncthreads();
    const size_t item = ((static_cast<size_t>(seq) * gridDim.y + blockIdx.y) * p.splits) + split;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = row0 + t * kCols + col;
        if (low || row >= tile.total) continue;
        const int head = kvh * p.group + row % p.group;
        const int64_t at = tile.begin + row / p.group;
#pragma unroll
        for (int k0 = 0; k0 < kChunks; ++k0) {
            const int d = wave * kChunks + k0;
            f32x4_t y = join[0][t][d][g * kCols + col];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) y += join[w][t][d][g * kCols + col];
            const int dim = 16 * d + 4 * g;
            if (p.splits > 1) {
                *reinterpret_cast<f32x4_t *>(p.partial + (item * kRows + t * kCols + col) * D + dim) = y;
            } else {
                const float norm = total[t] > 0.0f || total[t] != total[t] ? 1.0f / (total[t] * (kPScale * 127.0f)) : 0.0f;
                y = y * norm;
                if (p.gate) {
                    const E *gate = static_cast<const E *>(p.gate) + at * p.q_row + static_cast<int64_t>(head) * p.q_head + dim;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = norm != 0.0f ? gated<DT>(y[i], gate + i) : 0.0f;
                }
                E *to = static_cast<E *>(p.out) + at * p.out_row + static_cast<int64_t>(head) * D + dim;
                if (p.vec) store4<DT, true>(to, y);
                else store4<DT, false>(to, y);
            }
        }
        if (p.splits > 1 && wave == 0 && g == 0) {
            float *ml = p.partial_ml + (item * kRows + t * kCols + col) * 2;
            ml[0] = top[t];
            ml[1] = total[t];
        }
    }
}

// The splits of one row and head: a workgroup of eight waves, each over every
// eighth split, four dims a lane.
constexpr int kJoinWaves = 8;
template <int D, Dtype DT>
__global__ __launch_bounds__(kJoinWaves * 64) void kv8_attention_join_kernel(Kv8AttentionParams p, int tile_rows) {
    typedef typename Element<DT>::type E;
    constexpr int kLanes = D / 4;                    // of one vector
    constexpr int kGroups = kJoinWaves * 64 / kLanes;  // splits side by side
    __shared__ float weight[kKv8MaxSplits];
    __shared__ f32x4_t sums[kGroups][kLanes];
    const int seq = blockIdx.z, kvh = blockIdx.y, row = blockIdx.x;
    const int row0 = row / tile_rows * tile_rows;
    const RowTile tile = row_tile(p, seq, row0, tile_rows);
    if (row >= tile.total) return;
    const int active = min(p.splits, max((tile.tiles + kWaves - 1) / kWaves, 1));
    const size_t y_index = static_cast<size_t>(row / tile_rows) * p.cache.kv_heads + kvh;
    const size_t tiles_y = static_cast<size_t>(p.row_tiles) * p.cache.kv_heads;
    const size_t item = (static_cast<size_t>(seq) * tiles_y + y_index) * p.splits;
    const float *ml = p.partial_ml + (item * tile_rows + row % tile_rows) * 2;
    const size_t ml_step = static_cast<size_t>(tile_rows) * 2;

    const int lane = threadIdx.x & 63;
    float top = -__builtin_inff();
    for (int i = lane; i < active; i += 64) top = fmaxf(top, ml[i * ml_step]);
    top = wave_max(top);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float total = 0.0f;
    for (int i = lane; i < active; i += 64) {
        const float w = exp2_fast(ml[i * ml_step] - base);
        total += ml[i * ml_step + 1] * w;
        if (threadIdx.x < 64) weight[i] = w;
    }
    total = wave_sum(total);
    __syncthreads();
    const int group = threadIdx.x / kLanes, at = threadIdx.x % kLanes;
    const float *from = p.partial + (item * tile_rows + row % tile_rows) * D + 4 * at;
    const size_t step = static_cast<size_t>(tile_rows) * D;
    f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = group; i < active; i += kGroups) y += *reinterpret_cast<const f32x4_t *>(from + i * step) * weight[i];
    sums[group][at] = y;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) y += sums[k][at];
    const float norm = total > 0.0f || total != total ? 1.0f / (total * (kPScale * 127.0f)) : 0.0f;
    y = y * norm;
    const int head = kvh * p.group + row % p.group;
    const int64_t index = tile.begin + row / p.group;
    if (p.gate) {
        const E *gate = static_cast<const E *>(p.gate) + index * p.q_row + static_cast<int64_t>(head) * p.q_head + 4 * at;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = norm != 0.0f ? gated<DT>(y[i], gate + i) : 0.0f;
    }
    E *to = static_cast<E *>(p.out) + index * p.out_row + static_cast<int64_t>(head) * D + 4 * at;
    if (p.vec) store4<DT, true>(to, y);
    else store4<DT, false>(to, y);
}

template <int D, Dtype DT, bool SPLIT, int RT>
hipError_t launch_rows(Kv8AttentionParams p, const Kv8Plan &plan, hipStream_t stream) {
    const dim3 grid(plan.splits, plan.row_tiles * p.cache.kv_heads, p.batch.sequences);
    p.splits = plan.splits;
    p.row_tiles = plan.row_tiles;
    hipLaunchKernelGGL((kv8_attention_kernel<D, DT, SPLIT, RT>), grid, dim3(kWaves * 64), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && plan.splits > 1) {
        const dim3 rows(p.batch.max_rows * p.group, p.cache.kv_heads, p.batch.sequences);
        hipLaunchKernelGGL((kv8_attention_join_kernel<D, DT>), rows, dim3(kJoinWaves * 64), 0, stream, p, plan.rows);
        e = hipGetLastError();
    }
    return e;
}

template <int D, Dtype DT>
hipError_t launch_typed(const Kv8AttentionParams &p, const Kv8Plan &plan, hipStream_t stream) {
    if constexpr (DT == Dtype::F32) {
        return plan.rows == 8 ? launch_rows<D, DT, true, 1>(p, plan, stream) : launch_rows<D, DT, true, 2>(p, plan, stream);
    } else {
        if (plan.split_halves) return launch_rows<D, DT, true, 1>(p, plan, stream);
        return plan.rows == 16 ? launch_rows<D, DT, false, 1>(p, plan, stream) : launch_rows<D, DT, false, 2>(p, plan, stream);
    }
}

template <Dtype DT>
hipError_t launch_head(const Kv8AttentionParams &p, const Kv8Plan &plan, hipStream_t stream) {
    if (p.cache.head == 64) return launch_typed<64, DT>(p, plan, stream);
    if (p.cache.head == 128) return launch_typed<128, DT>(p, plan, stream);
    return launch_typed<256, DT>(p, plan, stream);
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8AttentionParams &p, Dtype dtype, const Kv8Plan &plan, hipStream_t stream) {
    if (dtype == Dtype::F32) return launch_head<Dtype::F32>(p, plan, stream);
    if (dtype == Dtype::F16) return launch_head<Dtype::F16>(p, plan, stream);
    return launch_head<Dtype::BF16>(p, plan, stream);
}

}  // namespace fortai_hip
