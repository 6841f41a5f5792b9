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

constexpr int kKv8MaxSplits = 256;       // workgroups that may share a sequence's head
constexpr int kKv8PartialRows = 16384;   // rows of partial results that a cache has room for


struct Kv8View {
    int8_t *keys = nullptr, *values = nullptr;         // [pages][kv_heads][P][D], [pages][kv_heads][D][P]
    float *key_max = nullptr, *value_max = nullptr;    // [pages][kv_heads]
    int pages = 0, page_tokens = 0, kv_heads = 0, head = 0;
};

// A word that no kernel writes while this one runs: where its address is the same
// for a whole wave it comes through the scalar cache.
FORTAI_HD int32_t read_only(const int32_t *p) {
#ifdef __HIP_DEVICE_COMPILE__
    return *(const __attribute__((address_space(4))) int32_t *)(p);
#else
    return *p;
#endif
}

struct Kv8Rows {
    const int32_t *starts = nullptr;   // [sequences + 1]
    const int32_t *lengths = nullptr;  // [sequences]: tokens before the sequence's first row
    const int32_t *tables = nullptr;   // [sequences][pitch]
    int sequences = 0, rows = 0, max_rows = 0, pitch = 0;

    // the sequence's rows [begin, begin + count) of the batch's arrays
    FORTAI_HD void range(int seq, int *begin, int *count) const {
        int b = read_only(starts + seq), e = read_only(starts + seq + 1);
        b = b < 0 ? 0 : b > rows ? rows : b;
        e = e < b ? b : e > rows ? rows : e;
        *begin = b;
        *count = e - b < max_rows ? e - b : max_rows;
    }
    FORTAI_HD int length(int seq) const {
        const int n = read_only(lengths + seq);
        return n < -kKv8MaxTokens ? -kKv8MaxTokens : n > kKv8MaxTokens ? kKv8MaxTokens : n;
    }
    // the table's word for the sequence's page `index`, or for the nearest that the table has
    FORTAI_HD int page_word(int seq, int index) const {
        const int at = index < 0 ? 0 : index >= pitch ? pitch - 1 : index;
        return read_only(tables + static_cast<int64_t>(seq) * pitch + at);
    }
    // the pool's page that holds the sequence's page `index`, or -1
    FORTAI_HD int page(int seq, int index, int pages) const {
        const int id = page_word(seq, index);
        return index >= 0 && index < pitch && id >= 0 && id < pages ? id : -1;
    }
};

// How an attention call is cut: `rows` rows of a kv head a workgroup, row_tiles
// such tiles, `splits` workgroups over the cached tokens of each.
struct Kv8Plan {
    int rows = 0, row_tiles = 0, splits = 0;
};

// fp32 queries always have 8 rows in an instruction's 16 columns (each twice, for the
// two halves of its numbers), others where 8 are enough.  More than twice as many rows
// take the kernel with four times as many a workgroup, if the cached tokens are so many
// that the smaller workgroups would have four tiles of 64 a SIMD.  Heads of 256, 16 bits:
// 40 rows over 30,000 tokens, 5.5 tiles a SIMD, 36.4 us against 39.4 (64 rows, which fill
// the smaller workgroups, 37.6 against 34.8); 256 rows over 1,000 tokens, one tile a SIMD,
// 26.0 against 22.3; 8,000 behind 7,000 413 against 560.  fp32: 64 rows over 30,000
// tokens 42.7 against 45.9, 8,000 behind 7,000 661 against 958; where many rows are split
// over few tokens their join costs more than either (1,000 behind 1,000, split in four,
// 54.7 against 27.5 unsplit).
// Tokens are split until there are two workgroups a CU for heads of 256 (more for
// smaller ones, which take less LDS), as far as every one has a tile for each of its
// four waves (two tiles where the waves share them) and the partial results fit: one workgroup a CU
// costs 30.5 us where two cost 25.9 (eight sequences of up to 8190 tokens); one tile a
// wave costs 13.2 us where three cost 17.0 (600 tokens).
inline Kv8Plan kv8_plan(bool fp32, int head, int sequences, int kv_heads, int64_t rows, int64_t max_length) {
    Kv8Plan p;
    const int64_t heads = static_cast<int64_t>(kv_heads) * sequences;
    const int few = fp32 || rows <= 8 ? 8 : 16;
    const bool much = rows > 2 * few && (rows + few - 1) / few * heads >= 4096 / ((max_length + 63) / 64 + 1);
    p.rows = much ? 4 * few : few;
    p.row_tiles = static_cast<int>((rows + p.rows - 1) / p.rows);
    const int64_t base = p.row_tiles * heads, fill = 512 * (256 / head), least = much ? 128 : 256;
    const int64_t wanted = (fill + base - 1) / base, useful = (max_length + least - 1) / least;
    const int64_t room = kKv8PartialRows / (base * p.rows);
    int64_t s = wanted < useful ? wanted : useful;
    s = s < room ? s : room;
    s = s < kKv8MaxSplits ? s : kKv8MaxSplits;
    p.splits = s < 1 ? 1 : static_cast<int>(s);
    return p;
}

}  // namespace fortai_hip
