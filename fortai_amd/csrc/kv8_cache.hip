// The 8-bit paged cache: append, read back, copy pages.
//
// One layer of a cache holds, for each page of P tokens and each head,
//   key codes   int8 [P][D]          (a token's codes side by side)
//   value codes int8 [D][P]          (a dim's codes side by side)
// and the two largest magnitudes A of what they stand for: value = code * (A / 127).
// Both orders are the ones in which the attention's matrix instructions take
// their operands, 16 bytes a lane, with no exchange between lanes.
//
// Append: A' = max(A of the tokens the page holds, |x| of the new ones), new
// codes = 127 x / A', and where A' > A the old codes are rounded once more to
// code * A / A'.  Every code is the integer nearest to that quotient in exact
// arithmetic, ties to even, so it depends neither on the compiler's division nor
// on how a prompt was cut into calls inside a page that does not grow.  One
// workgroup owns a page and head (keys or values), so that no two write a word.
//
// Bound by memory for prompts, by the chain of dependent loads (rows, table, A,
// values) for single tokens.  A wave takes blocks of 16 tokens x 64 dims, a lane
// 4 x 4 of them: reads of 256 (fp32) or 128 bytes in a row and, for both orders,
// writes of whole words with the transpose inside the lane.
#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kPageThreads = 256;
constexpr int kPageWaves = kPageThreads / 64;
constexpr int kBlocksPerWave = 4;  // 64 tokens x 256 dims over 4 waves

// round(|v| n / a) for finite v, ties to even, of the exact quotient; v n and
// (2 k + 1) a are exact in 64 bits (7 + 24 and 8 + 24 bits).
// inverse: n / a rounded to fp32, so |v| inverse is off by at most 127 * 2^-23.
__device__ __forceinline__ int nearest_code(float v, float n, float a, float inverse) {
    v = fabsf(v);
    if (a < 1e-30f) {  // n / a may overflow fp32; the fp64 quotient cannot round onto a tie that it is not
        return a > 0.0f ? static_cast<int>(__builtin_rint(static_cast<double>(v) * n / a)) : 0;
    }
    const float y = v * inverse, whole = floorf(y), part = y - whole;
    int k = static_cast<int>(whole) + (part > 0.5f ? 1 : 0);
    if (fabsf(part - 0.5f) < 2e-4f) {
        k = static_cast<int>(whole);
        const double twice = 2.0 * static_cast<double>(v) * n, border = (2.0 * k + 1.0) * static_cast<double>(a);
        if (twice > border || (twice == border && (k & 1))) ++k;
    }
    return min(k, 127);
}

// An infinity stands for the largest magnitude, NaN for zero.
__device__ __forceinline__ uint32_t code_byte(float x, float a, float inverse) {
    if (!(fabsf(x) <= 3.402823466e38f)) return x != x ? 0u : (x > 0.0f ? 127u : 0x81u);
    const int k = nearest_code(x, 127.0f, a, inverse);
    return static_cast<uint32_t>(x < 0.0f ? -k : k) & 0xffu;
}

__device__ __forceinline__ uint32_t requantized_byte(uint32_t byte, float was, float a, float ratio) {
    const int c = static_cast<int8_t>(byte);
    const int k = nearest_code(static_cast<float>(c), was, a, ratio);
    return static_cast<uint32_t>(c < 0 ? -k : k) & 0xffu;
}

template <Dtype DT, bool VEC>
__global__ __launch_bounds__(kPageThreads) void kv8_append_kernel(Kv8View cache, Kv8Rows batch,
    const typename Element<DT>::type *__restrict__ keys, int64_t key_pitch,
    const typename Element<DT>::type *__restrict__ values, int64_t value_pitch) {
    __shared__ float wave_top[kPageWaves];
    const int seq = blockIdx.z >> 1, head = blockIdx.y;
    const bool is_value = blockIdx.z & 1;
    const int P = cache.page_tokens, D = cache.head;
    int begin, count;
    batch.range(seq, &begin, &count);
    const int length = batch.length(seq);
    const int from = max(length, 0), until = length + count;  // the new tokens
    const int first = (from / P + static_cast<int>(blockIdx.x)) * P;
    const int new_from = max(from, first) - first, new_until = min(until, first + P) - first;  // slots of this page
    if (new_from >= new_until) return;
    const int id = batch.page(seq, first / P, cache.pages);
    if (id < 0) return;
    const int old = length > first ? new_from : 0;  // slots [0, old) hold tokens already
    const size_t which = static_cast<size_t>(id) * cache.kv_heads + head;
    float *top_at = (is_value ? cache.value_max : cache.key_max) + which;
    uint32_t *codes = reinterpret_cast<uint32_t *>((is_value ? cache.values : cache.keys) + which * P * D);
    const float was = old > 0 ? *top_at : 0.0f;
    const typename Element<DT>::type *x = (is_value ? values : keys) + static_cast<int64_t>(head) * D;
    const int64_t pitch = is_value ? value_pitch : key_pitch;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int dim_blocks = D / 64, blocks = (P / 16) * dim_blocks;
    f32x4_t v[kBlocksPerWave][4];  // [block][token of the four][dim of the four]
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < kBlocksPerWave; ++b) {
        const int block = b * kPageWaves + wave;
        const int slot = (block / dim_blocks) * 16 + (lane >> 4) * 4, d = (block % dim_blocks) * 64 + (lane & 15) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[b][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (block < blocks && slot + i >= new_from && slot + i < new_until)
                v[b][i] = load4<DT, VEC>(x + static_cast<int64_t>(begin + first + slot + i - length) * pitch + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float m = fabsf(v[b][i][j]);
                if (m <= 3.402823466e38f) top = fmaxf(top, m);
            }
        }
    }
    top = wave_max(top);
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    float a = was;
#pragma unroll
    for (int w = 0; w < kPageWaves; ++w) a = fmaxf(a, wave_top[w]);
    const bool grown = old > 0 && a > was;
    const float inverse = 127.0f / a, ratio = was / a;  // not used where a is zero or tiny
    if (threadIdx.x == 0) *top_at = a;

#pragma unroll
    for (int b = 0; b < kBlocksPerWave; ++b) {
        const int block = b * kPageWaves + wave;
        const int slot = (block / dim_blocks) * 16 + (lane >> 4) * 4, d = (block % dim_blocks) * 64 + (lane & 15) * 4;
        const bool some_new = slot + 3 >= new_from && slot < new_until;
        if (block >= blocks || (!some_new && !(grown && slot < old))) continue;
        if (!is_value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t *at = codes + (static_cast<size_t>(slot + i) * D + d) / 4;
                if (slot + i >= new_from && slot + i < new_until) {
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w |= code_byte(v[b][i][j], a, inverse) << (8 * j);
                    *at = w;
                } else if (grown && slot + i < old) {
                    const uint32_t c = *at;
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w |= requantized_byte(c >> (8 * j), was, a, ratio) << (8 * j);
                    *at = w;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t *at = codes + (static_cast<size_t>(d + j) * P + slot) / 4;
                const bool all_new = slot >= new_from && slot + 3 < new_until;
                const uint32_t c = all_new ? 0u : *at;  // slots that are neither new nor rounded again keep their codes
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t byte = c >> (8 * i);
                    if (slot + i >= new_from && slot + i < new_until) byte = code_byte(v[b][i][j], a, inverse);
                    else if (grown && slot + i < old) byte = requantized_byte(byte, was, a, ratio);
                    w |= (byte & 0xffu) << (8 * i);
                }
                *at = w;
            }
        }
    }
}

// Rows of the cache as values, the transpose of the value codes inside the lane
// as in the append.
template <Dtype DT, bool VEC>
__global__ __launch_bounds__(kPageThreads) void kv8_read_kernel(Kv8View cache, Kv8Rows batch,
    typename Element<DT>::type *__restrict__ keys, int64_t key_pitch, typename Element<DT>::type *__restrict__ values,
    int64_t value_pitch) {
    const int seq = blockIdx.z >> 1, head = blockIdx.y;
    const bool is_value = blockIdx.z & 1;
    const int P = cache.page_tokens, D = cache.head;
    int begin, count;
    batch.range(seq, &begin, &count);
    const int length = batch.length(seq);
    const int from = max(length, 0), until = length + count;
    const int first = (from / P + static_cast<int>(blockIdx.x)) * P;
    const int slot_from = max(from, first) - first, slot_until = min(until, first + P) - first;
    if (slot_from >= slot_until) return;
    const int id = batch.page(seq, first / P, cache.pages);
    const size_t which = static_cast<size_t>(id < 0 ? 0 : id) * cache.kv_heads + head;
    const float scale = id < 0 ? 0.0f : (is_value ? cache.value_max : cache.key_max)[which] / 127.0f;
    const uint32_t *codes = reinterpret_cast<const uint32_t *>((is_value ? cache.values : cache.keys) + which * P * D);
    typename Element<DT>::type *out = (is_value ? values : keys) + static_cast<int64_t>(head) * D;
    const int64_t pitch = is_value ? value_pitch : key_pitch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int dim_blocks = D / 64, blocks = (P / 16) * dim_blocks;
    for (int block = wave; block < blocks; block += kPageWaves) {
        const int slot = (block / dim_blocks) * 16 + (lane >> 4) * 4, d = (block % dim_blocks) * 64 + (lane & 15) * 4;
        if (slot + 3 < slot_from || slot >= slot_until) continue;
        uint32_t w[4];  // keys: of a token, values: of a dim
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = codes[(is_value ? static_cast<size_t>(d + k) * P + slot : static_cast<size_t>(slot + k) * D + d) / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (slot + i < slot_from || slot + i >= slot_until) continue;
            f32x4_t y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t byte = is_value ? w[j] >> (8 * i) : w[i] >> (8 * j);
                y[j] = id < 0 ? 0.0f : static_cast<float>(static_cast<int8_t>(byte)) * scale;
            }
            store4<DT, VEC>(out + static_cast<int64_t>(begin + first + slot + i - length) * pitch + d, y);
        }
    }
}

// Whole pages, every layer and head: 16 KiB of one plane of one pair a
// workgroup, all of it in flight before the first store.  The pairs travel as
// kernel arguments, so that a captured call holds them.
constexpr int kCopyVectors = 4;
constexpr int kCopySlice = kPageThreads * kCopyVectors * 16;
struct PagePairs {
    int32_t from[kKv8PairsPerLaunch], to[kKv8PairsPerLaunch];
};
__global__ __launch_bounds__(kPageThreads) void kv8_copy_pages_kernel(Kv8View cache, size_t layer_codes, size_t layer_tops,
    PagePairs pairs) {
    const int layer = blockIdx.z >> 1;
    const bool is_value = blockIdx.z & 1;
    const size_t from = static_cast<size_t>(pairs.from[blockIdx.y]), to = static_cast<size_t>(pairs.to[blockIdx.y]);
    const size_t bytes = static_cast<size_t>(cache.kv_heads) * cache.page_tokens * cache.head;
    int8_t *plane = (is_value ? cache.values : cache.keys) + layer * layer_codes;
    const u32x4_t *src = reinterpret_cast<const u32x4_t *>(plane + from * bytes);
    u32x4_t *dst = reinterpret_cast<u32x4_t *>(plane + to * bytes);
    const size_t at = static_cast<size_t>(blockIdx.x) * (kCopySlice / 16) + threadIdx.x, end = bytes / 16;
    u32x4_t v[kCopyVectors];
#pragma unroll
    for (int k = 0; k < kCopyVectors; ++k)
        if (at + k * kPageThreads < end) v[k] = __builtin_nontemporal_load(src + at + k * kPageThreads);
#pragma unroll
    for (int k = 0; k < kCopyVectors; ++k)
        if (at + k * kPageThreads < end) __builtin_nontemporal_store(v[k], dst + at + k * kPageThreads);
    if (blockIdx.x == 0) {
        float *tops = (is_value ? cache.value_max : cache.key_max) + layer * layer_tops;
        for (int h = threadIdx.x; h < cache.kv_heads; h += kPageThreads)
            tops[to * cache.kv_heads + h] = tops[from * cache.kv_heads + h];
    }
}

__global__ __launch_bounds__(256) void kv8_clear_kernel(u32x4_t *at, size_t vectors, size_t bytes) {
    const size_t n = static_cast<size_t>(gridDim.x) * blockDim.x;
    for (size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < vectors; i += n) at[i] = u32x4_t{0, 0, 0, 0};
    if (blockIdx.x == 0 && threadIdx.x == 0)
        for (size_t i = vectors * 16; i < bytes; ++i) reinterpret_cast<uint8_t *>(at)[i] = 0;
}

dim3 page_grid(const Kv8View &cache, const Kv8Rows &batch) {
    // the most pages that max_rows tokens can touch, wherever the first one falls
    const int spans = (batch.max_rows + cache.page_tokens - 2) / cache.page_tokens + 1;
    return dim3(spans, cache.kv_heads, 2 * batch.sequences);
}

template <Dtype DT>
void append_typed(const Kv8View &cache, const Kv8Rows &batch, const void *keys, int64_t key_pitch, const void *values,
    int64_t value_pitch, bool vec, hipStream_t stream) {
    typedef typename Element<DT>::type E;
    const dim3 grid = page_grid(cache, batch), block(kPageThreads);
    const E *k = static_cast<const E *>(keys), *v = static_cast<const E *>(values);
    if (vec) hipLaunchKernelGGL((kv8_append_kernel<DT, true>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
    else hipLaunchKernelGGL((kv8_append_kernel<DT, false>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
}

template <Dtype DT>
void read_typed(const Kv8View &cache, const Kv8Rows &batch, void *keys, int64_t key_pitch, void *values,
    int64_t value_pitch, bool vec, hipStream_t stream) {
    typedef typename Element<DT>::type E;
    const dim3 grid = page_grid(cache, batch), block(kPageThreads);
    E *k = static_cast<E *>(keys), *v = static_cast<E *>(values);
    if (vec) hipLaunchKernelGGL((kv8_read_kernel<DT, true>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
    else hipLaunchKernelGGL((kv8_read_kernel<DT, false>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
}

}  // namespace

hipError_t launch_kv8_append(const Kv8View &cache, const Kv8Rows &batch, Dtype dtype, const void *keys, int64_t key_pitch,
    const void *values, int64_t value_pitch, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) append_typed<Dtype::F32>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    else if (dtype == Dtype::F16) append_typed<Dtype::F16>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    else append_typed<Dtype::BF16>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8View &cache, const Kv8Rows &batch, Dtype dtype, void *keys, int64_t key_pitch,
    void *values, int64_t value_pitch, bool vec, hipStream_t stream) {
    if (dtype == Dtype::F32) read_typed<Dtype::F32>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    else if (dtype == Dtype::F16) read_typed<Dtype::F16>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    else read_typed<Dtype::BF16>(cache, batch, keys, key_pitch, values, value_pitch, vec, stream);
    return hipGetLastError();
}

hipError_t launch_kv8_copy_pages(const Kv8View &cache, size_t layer_codes, size_t layer_tops, int layers,
    const int32_t *from, const int32_t *to, int count, hipStream_t stream) {
    const size_t bytes = static_cast<size_t>(cache.kv_heads) * cache.page_tokens * cache.head;
    for (int at = 0; at < count; at += kKv8PairsPerLaunch) {
        const int n = count - at < kKv8PairsPerLaunch ? count - at : kKv8PairsPerLaunch;
        PagePairs pairs = {};
        for (int i = 0; i < n; ++i) {
            pairs.from[i] = from[at + i];
            pairs.to[i] = to[at + i];
        }
        const dim3 grid((bytes + kCopySlice - 1) / kCopySlice, n, 2 * layers);
        hipLaunchKernelGGL(kv8_copy_pages_kernel, grid, dim3(kPageThreads), 0, stream, cache, layer_codes, layer_tops, pairs);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv8_clear(void *storage, size_t bytes, hipStream_t stream) {
    hipLaunchKernelGGL(kv8_clear_kernel, dim3(2048), dim3(256), 0, stream, static_cast<u32x4_t *>(storage), bytes / 16, bytes);
    return hipGetLastError();
}

}  // namespace fortai_hip
