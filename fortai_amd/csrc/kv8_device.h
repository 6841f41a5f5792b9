// What the kernels of the 8-bit cache are handed: one layer's planes and a
// ragged batch of sequences.  Every number that comes from device memory (row
// starts, lengths, page ids) is brought into range before it is used, so that a
// wrong one costs that row or page and reaches no other memory.
#pragma once

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define FORTAI_HD __host__ __device__ __forceinline__
#else
#define FORTAI_HD inline
#endif
#include <stddef.h>
#include <stdint.h>

namespace fortai_hip {

constexpr int kKv8MaxTokens = 1 << 30;  // the longest table: 2^24 pages of 64 tokens
constexpr int kKv8PairsPerLaunch = 448;  // page pairs that fit a launch's arguments beside the rest

struct Kv8View {
    int8_t *keys = nullptr, *values = nullptr;         // [pages][kv_heads][P][D], [pages][kv_heads][D][P]
    float *key_max = nullptr, *value_max = nullptr;    // [pages][kv_heads]
    int pages = 0, page_tokens = 0, kv_heads = 0, head = 0;
};

struct Kv8Rows {
    const int32_t *starts = nullptr;   // [sequences + 1]
    const int32_t *lengths = nullptr;  // [sequences]: tokens before the sequence's first row
    const int32_t *tables = nullptr;   // [sequences][pitch]
    int sequences = 0, rows = 0, max_rows = 0, pitch = 0;

    // the sequence's rows [begin, begin + count) of the batch's arrays
    FORTAI_HD void range(int seq, int *begin, int *count) const {
        int b = starts[seq], e = starts[seq + 1];
        b = b < 0 ? 0 : b > rows ? rows : b;
        e = e < b ? b : e > rows ? rows : e;
        *begin = b;
        *count = e - b < max_rows ? e - b : max_rows;
    }
    FORTAI_HD int length(int seq) const {
        const int n = lengths[seq];
        return n < -kKv8MaxTokens ? -kKv8MaxTokens : n > kKv8MaxTokens ? kKv8MaxTokens : n;
    }
    // the pool's page that holds the sequence's page `index`, or -1
    FORTAI_HD int page(int seq, int index, int pages) const {
        if (index < 0 || index >= pitch) return -1;
        const int id = tables[static_cast<int64_t>(seq) * pitch + index];
        return id >= 0 && id < pages ? id : -1;
    }
};

}  // namespace fortai_hip
