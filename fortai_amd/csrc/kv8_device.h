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
constexpr int kKv8PartialRows = 16384;   // rows of partial results that a call may have
constexpr int kKv8SharedRows = 32768;    // that one with shared tokens may have: what a cache has room for (with as
                                         // many as the other, two groups of 132 rows over up to 24,000 tokens had
                                         // 204 workgroups, not 456, and took 61 us, not 41)


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
inline Kv8Plan kv8_plan(bool fp32, int head, int sequences, int kv_heads, int64_t rows, int64_t max_length,
    int64_t partial_rows = kKv8PartialRows, int workgroups = 512, int least_rows = 8) {
    Kv8Plan p;
    const int64_t heads = static_cast<int64_t>(kv_heads) * sequences;
    const int few = fp32 || (rows <= 8 && least_rows <= 8) ? 8 : 16;
    const bool much = rows > 2 * few && (rows + few - 1) / few * heads >= 4096 / ((max_length + 63) / 64 + 1);
    p.rows = much ? 4 * few : few;
    p.row_tiles = static_cast<int>((rows + p.rows - 1) / p.rows);
    const int64_t base = p.row_tiles * heads, fill = workgroups * (256 / head), least = much ? 128 : 256;
    const int64_t wanted = (fill + base - 1) / base, useful = (max_length + least - 1) / least;
    const int64_t room = partial_rows / (base * p.rows);
    int64_t s = wanted < useful ? wanted : useful;
    s = s < room ? s : room;
    s = s < kKv8MaxSplits ? s : kKv8MaxSplits;
    p.splits = s < 1 ? 1 : static_cast<int>(s);
    return p;
}

// How a call is cut whose sequences share tokens: the groups' tokens and the sequences'
// own, which have their partial results behind the groups' from row own_at on.  shares
// is false where these do not fit, and where the call would lose by it.
struct Kv8SharedPlan {
    Kv8Plan own, group;
    int64_t own_at = 0;
    bool shares = false;
};

// About how long a plan's workgroups take, in turns of the kernels for few rows (four tiles, one a wave): those for many
// rows take a tile at a time in 0.55 (32 rows) or 0.7 (64) of one, and 1.5 to begin; two a CU take 1.2 times as long.
inline double kv8_turns(const Kv8Plan &p, int64_t blocks, int64_t tokens, int head) {
    const bool few = p.rows <= 16;
    const int64_t tiles = (tokens + 63) / 64, workgroups = blocks * p.splits, chip = 512 * (256 / head);
    const int64_t turns = (tiles + p.splits * (few ? 4 : 1) - 1) / (p.splits * (few ? 4 : 1));
    const double each = 0.7 + (few ? turns : p.rows == 32 ? 1.5 + 0.55 * turns : 1.5 + 0.7 * turns);
    return each * (2 * workgroups > chip ? 1.2 : 1.0) * (workgroups > chip ? static_cast<double>(workgroups) / chip : 1.0);
}

// The groups' tokens are split for one workgroup a CU (half as many partial results to write and join) unless that
// leaves one more than 12 tiles: 4 kv heads of 256 behind 8000 tokens, eight sequences' rows in fp32 17.9 us against
// 23.4 for two a CU, 32 sequences' 33.6 against 37.5; 5 rows of 4 in bf16 behind 24,000 (11.7 tiles) 44.0 against 43.6,
// two groups of 8 (18 tiles) 61 against 41.
inline Kv8SharedPlan kv8_shared_plan(bool fp32, int head, int sequences, int groups, int kv_heads, int64_t rows, int64_t group_rows,
    int64_t max_own, int64_t max_shared) {
    Kv8SharedPlan p;
    const auto blocks = [&](const Kv8Plan &plan, int who) { return static_cast<int64_t>(who) * plan.row_tiles * kv_heads; };
    const auto partial = [&](const Kv8Plan &plan, int who) { return blocks(plan, who) * plan.rows * plan.splits; };
    const int64_t tiles = (max_shared + 63) / 64;
    const auto cut = [&](int least_rows) {
        // the sequences' own tokens are few: what they leave of the workspace is the groups'
        p.own = kv8_plan(fp32, head, sequences, kv_heads, rows, max_own, kKv8SharedRows / 4, 512, least_rows);
        const int64_t own = partial(p.own, sequences);
        const int64_t room = own < kKv8SharedRows ? kKv8SharedRows - own - 63 : 0;
        p.group = kv8_plan(fp32, head, groups, kv_heads, group_rows, max_shared, room, 256);
        if (tiles > 12 * p.group.splits) {
            p.group = kv8_plan(fp32, head, groups, kv_heads, group_rows, max_shared, room);
            // no more workgroups than the chip holds: a few more wait until the first ones end (four sequences of 20 rows of
            // 4 kv heads in fp32 behind 24,000 tokens: 516 workgroups 60.7 us, 504 50)
            const int64_t most = 512 * (256 / head) / blocks(p.group, groups);
            if (most > 0 && most < p.group.splits) p.group.splits = static_cast<int>(most);
        } else if (p.group.rows <= 16) {
            // up to a quarter more workgroups where that saves their last turn of four tiles (four sequences of 20 rows in
            // fp32 behind 8000 tokens of 2 kv heads: 15 splits of 2.08 turns 24.4 us, 16 20.2)
            const int64_t turns = tiles / (4 * p.group.splits), splits = turns > 0 ? (tiles + 4 * turns - 1) / (4 * turns) : 0;
            if (splits > p.group.splits && 4 * splits <= 5 * static_cast<int64_t>(p.group.splits) && splits <= kKv8MaxSplits &&
                splits * blocks(p.group, groups) * p.group.rows <= room)
                p.group.splits = static_cast<int>(splits);
        }
    };
    cut(8);
    // groups of up to 16 rows and sequences of up to 8 are one launch where both have workgroups of 16: three answers to
    // a question of 1000 tokens (16 bits, 4 rows of 4 kv heads) 13.5 us, in two launches 22
    if (p.own.rows == 8 && p.group.rows == 16) cut(16);
    const int64_t own = partial(p.own, sequences);
    p.own_at = (partial(p.group, groups) + 63) / 64 * 64;
    // Where the plain call is one launch and so few tokens are shared, the join costs more than they do: 2 to 46 sequences
    // behind 64 to 256 tokens 10.6 to 26 us, by themselves 6.7 to 14.  Otherwise sharing has to be as fast, by the turns
    // of both, as nearly as they tell (two sequences of 20 rows of 2 kv heads in bf16 behind 24,000 tokens 29 us, by
    // themselves 24; where they tell too much it costs up to a fifth, on average of 700 cases nothing).
    const Kv8Plan plain = kv8_plan(fp32, head, sequences, kv_heads, rows, max_shared + max_own);
    const bool little = plain.splits == 1 && max_shared <= 256;
    const bool slower = kv8_turns(p.group, blocks(p.group, groups), max_shared, head) >
        1.3 * kv8_turns(plain, blocks(plain, sequences), max_shared + max_own, head);
    p.shares = max_shared >= 64 && p.own_at + own <= kKv8SharedRows && !little && !slower;
    return p;
}

}  // namespace fortai_hip
