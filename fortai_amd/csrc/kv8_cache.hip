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
// values) for single tokens.  A wave takes a block of 16 tokens x 64 dims, a lane
// 4 x 4 of them: reads of 256 (fp32) or 128 bytes in a row and, for both orders,
// writes of whole words with the transpose inside the lane.  One block a wave, so that
// a page is in flight at once (four blocks one after the other: the read back of
// 2,300 prompt tokens 12.4 us instead of 10.8, an append of them 45 us, 27 KB of code,
// instead of 16).  A token of each of eight sequences: append 6.4 us, read back 5.6.
// Page copies: 1.05 GB in 174 us, 6.0 TB/s.
#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

constexpr int kPageThreads = 256;
constexpr int kAppendWaves = 16;  // 64 tokens x 256 dims, a block of 16 x 64 a wave

// The integer nearest to v n / a, ties to even, of the exact quotient; v >= 0 and
// n <= 127 a, all scaled so that a is in [1/2, 1).  inverse: n / a rounded, so the
// first guess is off by one at most.  The border odd a = (2 k + 1) a is split into
// p + e exactly, and 2 v n - p, which near the border is a difference of two
// products of 32 bits, fits fp32: what is compared is exact where it is close.
__device__ __forceinline__ int nearest_code(float v, float twice_n, float a, float inverse) {
    const float k = floorf(v * inverse), odd = __builtin_fmaf(2.0f, k, 1.0f);
    const float p = odd * a, e = __builtin_fmaf(odd, a, -p), r = __builtin_fmaf(v, twice_n, -p);
    const int i = static_cast<int>(k);
    return i + (r > e || (r == e && (i & 1)) ? 1 : 0);
}

// a page's magnitude as [1/2, 1) and its exponent, and what codes are made with
struct CodeScale {
    float a, inverse;
    int exponent;
    __device__ __forceinline__ explicit CodeScale(float top) {
        exponent = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 0;
        a = top > 0.0f ? __builtin_ldexpf(top, -exponent) : 1.0f;
        inverse = 127.0f / a;
    }
    // An infinity stands for the largest magnitude.  NaN has been made zero.
    __device__ __forceinline__ uint32_t code(float x) const {
        int k = nearest_code(__builtin_ldexpf(fabsf(x), -exponent), 254.0f, a, inverse);
        k = fabsf(x) == __builtin_inff() ? 127 : k;
        return static_cast<uint32_t>(x < 0.0f ? -k : k) & 0xffu;
    }
};

// old codes under a raised magnitude: code * was / a
struct Requantizer {
    float twice_was, a, ratio;
    __device__ __forceinline__ Requantizer(float was, const CodeScale &s)
        : twice_was(__builtin_ldexpf(was, 1 - s.exponent)), a(s.a), ratio(0.5f * twice_was / s.a) {}
    __device__ __forceinline__ uint32_t code(uint32_t byte) const {
        const int c = static_cast<int8_t>(byte);
        const int k = nearest_code(fabsf(static_cast<float>(c)), twice_was, a, ratio);
        return static_cast<uint32_t>(c < 0 ? -k : k) & 0xffu;
    }
    __device__ __forceinline__ uint32_t word(uint32_t w) const {
        return code(w) | code(w >> 8) << 8 | code(w >> 16) << 16 | code(w >> 24) << 24;
    }
};

template <Dtype DT, bool VEC, bool VALUES>
__device__ __forceinline__ void append_page(const Kv8View &cache, const Kv8Rows &batch,
    const typename Element<DT>::type *__restrict__ x, int64_t pitch) {
    __shared__ float wave_top[kAppendWaves];
    const int seq = blockIdx.z >> 1, head = blockIdx.y;
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
    float *top_at = (VALUES ? cache.value_max : cache.key_max) + which;
    uint32_t *codes = reinterpret_cast<uint32_t *>((VALUES ? cache.values : cache.keys) + which * P * D);
    const float was = old > 0 ? *top_at : 0.0f;
    x += static_cast<int64_t>(head) * D + static_cast<int64_t>(begin + first - length) * pitch;  // slot 0's row

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim_blocks = D / 64;
    const int slot = (wave / dim_blocks) * 16 + (lane >> 4) * 4, d = (wave % dim_blocks) * 64 + (lane & 15) * 4;
    f32x4_t v[4];  // [token of the four][dim of the four]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (slot + i >= new_from && slot + i < new_until) v[i] = load4<DT, VEC>(x + static_cast<int64_t>(slot + i) * pitch + d);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float m = fabsf(v[i][j]);
            v[i][j] = m == m ? v[i][j] : 0.0f;
            top = m < __builtin_inff() ? fmaxf(top, m) : top;
        }
    top = wave_max(top);
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    float a = was;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) a = fmaxf(a, wave_top[w]);
    const bool grown = old > 0 && a > was;
    const CodeScale scale(a);
    const Requantizer again(was, scale);
    if (threadIdx.x == 0) *top_at = a;

    const bool some_new = slot + 3 >= new_from && slot < new_until;
    if (!some_new && !(grown && slot < old)) return;
    // the slots of this lane's four that are new, and those rounded again
    uint32_t fresh = 0, rounded = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (slot + i >= new_from && slot + i < new_until) fresh |= 0xffu << (8 * i);
        if (grown && slot + i < old) rounded |= 0xffu << (8 * i);
    }
    uint32_t w[4];  // keys: of a token, values: of a dim
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = VALUES ? scale.code(v[0][i]) | scale.code(v[1][i]) << 8 | scale.code(v[2][i]) << 16 | scale.code(v[3][i]) << 24
                      : scale.code(v[i][0]) | scale.code(v[i][1]) << 8 | scale.code(v[i][2]) << 16 | scale.code(v[i][3]) << 24;
    uint32_t *at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        at[i] = codes + (VALUES ? static_cast<size_t>(d + i) * P + slot : static_cast<size_t>(slot + i) * D + d) / 4;
    if (fresh == 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *at[i] = w[i];
        return;
    }
    // slots that are neither new nor rounded again keep their codes
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const uint32_t mine = i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3];
        uint32_t *to = i == 0 ? at[0] : i == 1 ? at[1] : i == 2 ? at[2] : at[3];
        const uint32_t take = VALUES ? fresh : (fresh >> (8 * i) & 1 ? 0xffffffffu : 0u);
        const uint32_t turn = VALUES ? rounded : (rounded >> (8 * i) & 1 ? 0xffffffffu : 0u);
        if ((take | turn) == 0) continue;
        uint32_t kept = *to;
        if (turn) kept = (again.word(kept) & turn) | (kept & ~turn);
        *to = (mine & take) | (kept & ~take);
    }
}

template <Dtype DT, bool VEC>
__global__ __launch_bounds__(kAppendWaves * 64) void kv8_append_kernel(Kv8View cache, Kv8Rows batch,
    const typename Element<DT>::type *__restrict__ keys, int64_t key_pitch,
    const typename Element<DT>::type *__restrict__ values, int64_t value_pitch) {
    if (blockIdx.z & 1) append_page<DT, VEC, true>(cache, batch, values, value_pitch);
    else append_page<DT, VEC, false>(cache, batch, keys, key_pitch);
}

// Rows of the cache as values, the transpose of the value codes inside the lane
// as in the append.
template <Dtype DT, bool VEC>
__global__ __launch_bounds__(kAppendWaves * 64) void kv8_read_kernel(Kv8View cache, Kv8Rows batch,
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
    const int dim_blocks = D / 64, slot = (wave / dim_blocks) * 16 + (lane >> 4) * 4, d = (wave % dim_blocks) * 64 + (lane & 15) * 4;
    if (slot + 3 < slot_from || slot >= slot_until) return;
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
    const dim3 grid = page_grid(cache, batch), block(cache.page_tokens / 16 * (cache.head / 64) * 64);
    const E *k = static_cast<const E *>(keys), *v = static_cast<const E *>(values);
    if (vec) hipLaunchKernelGGL((kv8_append_kernel<DT, true>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
    else hipLaunchKernelGGL((kv8_append_kernel<DT, false>), grid, block, 0, stream, cache, batch, k, key_pitch, v, value_pitch);
}

template <Dtype DT>
void read_typed(const Kv8View &cache, const Kv8Rows &batch, void *keys, int64_t key_pitch, void *values,
    int64_t value_pitch, bool vec, hipStream_t stream) {
    typedef typename Element<DT>::type E;
    const dim3 grid = page_grid(cache, batch), block(cache.page_tokens / 16 * (cache.head / 64) * 64);
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
