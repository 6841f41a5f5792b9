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
//   S^T [token][row] = K Q^T in v_mfma_i32_16x16x64_i8, q as digits to the base 256
//   O^T [dim][row] += V^T P^T in v_mfma_f32_16x16x32_f16, the codes turned into fp16
// so that key codes are operands as they are and S is exact up to the query's digits.
// A tile is 64 tokens.  Lane (r = lane & 15, g = lane >> 4) of tile part u (0..3)
// feeds key token 16 (r >> 2) + 4 u + (r & 3), so that S leaves the instruction
// with lane group g holding the 16 consecutive tokens 16 g .. 16 g + 15 of row r:
// those are exactly the value codes that lane reads as one 16-byte word per dim
// (pages are [dim][token]), in the order in which the next instruction takes its
// k index.  P never goes through LDS.
//
// Numerics.  SPLIT: the 16 columns are 8 rows twice, for four digits of q (31 bits)
// and for p in two fp16 halves (22 bits): used for fp32 queries, and where no more
// than 8 rows are there to fill the columns.  Without it three digits (23 bits), and
// p's halves are operands one after the other: with two digits and the upper half alone
// five rows over 32,760 tokens take 0.9 us less and 2000 behind 6000 109 us less, but the
// results are off by 2^-12 of themselves and not the same as the same row's in a call of
// fewer.  The numerator's terms are p_j A_v / 127: what is rounded to fp16 is p_j A_v over
// the largest such product so far (times 2^14, away from fp16's subnormals), so that pages
// of very different magnitude lose nothing against each other.  The denominator has a
// maximum of its own, a lane's: a page of zeros counts there, whatever its score, and
// raises no product's.  Both are whole powers of two, with a score's and a
// magnitude's exponent apart, and what a page's weights are held against first is their
// own largest score: any finite score and magnitude will do.  (Magnitudes in the scores'
// maximum instead, up to 2^100: 4 % faster, infinities beyond, and products beside a page
// of zeros lost.)  Products count as zero below 2^-48 of the largest, 2^-37 without SPLIT;
// in the kernel for many rows below 2^-45 and 2^-34.  All sums are fp32.
//
// Few rows (decode steps, drafts): the four waves of a workgroup take tiles in turn, two
// workgroups a CU; `splits` workgroups share a sequence's head, joined by a second
// launch (the last workgroup joining instead: every workgroup writes its L2 back for
// that, 88 us where two launches take 25).  Bound by what a wave has to issue, 560 vector
// instructions a tile and 1,040 around its tiles (queries, join, quotients; counted at
// heads of 256), and, where a wave has one tile or two, by the loads that wait for each
// other on the way there: page word, keys, then values.  Eight sequences of up to 8190 tokens, 16 heads of 256: 25.8 us for 81 MB (values read into registers as they
// are operands, in pieces of 16 bytes out of rows of 64: 12 % more); five rows over
// 32,760 tokens 22.8 us for 33.6 MB; 600 tokens 13.2 us.
#include "fortai_hip_internal.h"
#include "kv8_device.h"
#include "serving_kernels.h"

namespace fortai_hip {

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int kTileTokens = 64;
constexpr int kWaves = 4;
constexpr int kArithmeticMayCross = 6;       // a scheduling barrier for all but vector and scalar arithmetic
constexpr float kLoScale = 2048.0f;          // 2^11: the left-over halves of a split
constexpr float kPScale = 16384.0f;          // 2^14
constexpr float kWideScale = 2048.0f;        // 2^11, where p may reach 2^4

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

// A product that is rounded to fp32 before anything is done with it: the compiler folds
// a multiplication into a conversion to fp16 (one rounding), but not into every use of it,
// and a lower half that is left over from another upper half is off by a whole step.
__device__ __forceinline__ float rounded(float product) {
    asm("" : "+v"(product));
    return product;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kNone = -3e38f;      // a base of nothing; finite, so that differences are
constexpr float kHuge = 4194304.0f;  // 2^22: a whole score below it, plus an exponent, is exact

// What products p_j A_v are held against: 2^(score + value), with a whole number near a
// score and the exponent of a magnitude.  Beside a huge score the two are kept apart:
// their sum would lose the exponent.
struct Base {
    float score, value;
};

// log2 of a over b, exact wherever it matters
__device__ __forceinline__ float above(const Base &a, const Base &b) { return (a.score - b.score) + (a.value - b.value); }

// the larger of this lane's and that of the lane N further on
template <int N>
__device__ __forceinline__ Base larger_of_lanes(const Base &a) {
    const Base b = {xor_lane<N>(a.score), xor_lane<N>(a.value)};
    return above(b, a) > 0.0f ? b : a;
}

// the largest of the four lanes of a row
__device__ __forceinline__ Base largest_of_row(const Base &a, bool some_huge) {
    if (some_huge) return larger_of_lanes<32>(larger_of_lanes<16>(a));
    float sum = a.score + a.value;
    sum = fmaxf(sum, xor_lane<16>(sum));
    sum = fmaxf(sum, xor_lane<32>(sum));
    return Base{sum, 0.0f};
}

// A softmax's denominator, sum 2^base.
struct Denominator {
    float base = kNone, sum = 0.0f;
    __device__ __forceinline__ void add(float other_base, float other_sum) {
        const float d = other_base - base, scale = exp2_fast(-fabsf(d));
        sum = __builtin_fmaf(d > 0.0f ? sum : other_sum, scale, d > 0.0f ? other_sum : sum);
        base = fmaxf(base, other_base);
    }
    template <int N>
    __device__ __forceinline__ void add_lane() { add(xor_lane<N>(base), xor_lane<N>(sum)); }
};

// What turns a sum of products over 2^base into a result: y norm 2^exponent.  No token: 0.
struct Quotient {
    float norm;
    int exponent;
    __device__ __forceinline__ Quotient(const Base &base, const Denominator &l, float scale)
        : norm(l.sum > 0.0f || l.sum != l.sum ? 1.0f / (l.sum * (scale * 127.0f)) : 0.0f),
          exponent(static_cast<int>(fminf(fmaxf((base.score - l.base) + base.value, -1000.0f), 1000.0f))) {}
    __device__ __forceinline__ Quotient(float n, int e) : norm(n), exponent(e) {}
    __device__ __forceinline__ f32x4_t operator()(f32x4_t y) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_ldexpf(y[i] * norm, exponent);
        return y;
    }
    __device__ __forceinline__ bool some() const { return norm != 0.0f; }
};

template <Dtype DT>
__device__ __forceinline__ f32x4_t load_gate(const Kv8AttentionParams &p, int64_t row, int head, int dim) {
    typedef typename Element<DT>::type E;
    const E *at = static_cast<const E *>(p.gate) + row * p.q_row + static_cast<int64_t>(head) * p.q_head + dim;
    return p.vec ? load4<DT, true>(at) : load4<DT, false>(at);
}

// Four dims of one row and head, gated and stored.  some: the row saw a token; GATE: what
// load_gate() gave is in *early.
template <Dtype DT, bool GATE = false>
__device__ __forceinline__ void finish(const Kv8AttentionParams &p, f32x4_t y, bool some, int64_t row, int head, int out, int dim,
    const f32x4_t *early = nullptr) {
    typedef typename Element<DT>::type E;
    if (p.gate && some) {
        const f32x4_t g = GATE ? *early : load_gate<DT>(p, row, head, dim);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] / (1.0f + expf(-g[i]));
    }
    E *to = static_cast<E *>(p.out) + row * p.out_row + out;
    if (p.vec) store4<DT, true>(to, y);
    else store4<DT, false>(to, y);
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

// What a workgroup does: rows row0 .. of a kv head, as `split` of `splits` over the tiles
// from first_tile on, with the table of sequence seq; `item` is its place among the partial
// results.
struct Work {
    int seq, kvh, row0, split, splits, first_tile;
    RowTile tile;
    size_t item;
};

// Rows and shared tokens of a group: whole tiles, 0 where its rows are more than the call
// was cut for or its numbers name no sequences.
struct Group {
    int first, begin, rows, shared;
};

__device__ __forceinline__ Group group_at(const Kv8AttentionParams &p, int index) {
    Group g;
    const int s0 = read_only(p.sharing.starts + index), s1 = read_only(p.sharing.starts + index + 1);
    const int tokens = min(read_only(p.sharing.shared + index), p.batch.pitch * p.cache.page_tokens);
    g.first = g.begin = g.rows = g.shared = 0;
    if (s0 < 0 || s1 <= s0 || s1 > p.batch.sequences) return g;
    int last, count;
    p.batch.range(s0, &g.begin, &count);
    p.batch.range(s1 - 1, &last, &count);
    g.first = s0;
    g.rows = max(last + count - g.begin, 0);
    g.shared = g.rows <= p.sharing.max_rows && tokens > 0 ? tokens / kTileTokens * kTileTokens : 0;
    return g;
}

// What sequence seq leaves to its group (*index): every row of it, all among the group's, sees
// all of these tokens.
__device__ __forceinline__ Group shared_by(const Kv8AttentionParams &p, int seq, const RowTile &tile, int *index) {
    Group g = {0, 0, 0, 0};
    *index = read_only(p.sharing.group_of + seq);
    if (*index < 0 || *index >= p.sharing.groups) return g;
    g = group_at(p, *index);
    const int end = read_only(p.sharing.starts + *index + 1), rows = tile.total / p.group;
    if (seq < g.first || seq >= end || tile.length < g.shared || tile.begin < g.begin || tile.begin - g.begin + rows > g.rows) g.shared = 0;
    return g;
}

template <bool SHARING, int ROWS>
__device__ __forceinline__ Work work_of(const Kv8AttentionParams &p) {
    Work w;
    if constexpr (!SHARING) {
        w.seq = blockIdx.z;
        w.kvh = blockIdx.y % p.cache.kv_heads;
        w.row0 = (blockIdx.y / p.cache.kv_heads) * ROWS;
        w.split = blockIdx.x;
        w.splits = p.splits;
        w.first_tile = 0;
        w.tile = row_tile(p, w.seq, w.row0, ROWS);
        w.item = ((static_cast<size_t>(w.seq) * gridDim.y + blockIdx.y) * p.splits) + w.split;
    } else {
        // first the groups' blocks, then the sequences'
        const int block = blockIdx.x + p.first_block;
        const int of_groups = p.sharing.groups * p.shared_row_tiles * p.cache.kv_heads * p.shared_splits;
        const bool group = block < of_groups;
        const int at = group ? block : block - of_groups, tiles = group ? p.shared_row_tiles : p.row_tiles;
        w.splits = group ? p.shared_splits : p.splits;
        w.split = at % w.splits;
        const int rest = at / w.splits, rows = rest / p.cache.kv_heads, who = rows / tiles;
        w.kvh = rest % p.cache.kv_heads;
        w.row0 = (rows % tiles) * ROWS;
        // partial results: the groups' rows, then the sequences'
        w.item = static_cast<size_t>(at) + (group ? 0 : static_cast<size_t>(p.own_at) / ROWS);
        if (group) {
            const Group g = group_at(p, who);
            w.seq = g.first;
            w.first_tile = 0;
            // every row sees all of the tokens
            w.tile = RowTile{g.begin, g.shared > 0 ? g.rows * p.group : 0, g.shared, g.shared, g.shared / kTileTokens};
        } else {
            w.seq = who;
            w.tile = row_tile(p, who, w.row0, ROWS);
            int index;
            w.first_tile = shared_by(p, who, w.tile, &index).shared / kTileTokens;
        }
    }
    return w;
}

// Until at most N of this wave's loads from memory are on their way (gfx9 s_waitcnt:
// vmcnt in bits 3:0 and 15:14, the other counters left alone), with no LDS access
// moved across it.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
    asm volatile("" ::: "memory");
}

// LDS reads done: what they read may be overwritten
__device__ __forceinline__ void wait_lds() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// 16 bytes a lane from base + offset (+ INST) to LDS at `to`, lane after lane.
// Written out because the compiler, which cannot tell one buffer's loads from
// another's, would have every LDS read wait for all of them; wait_loads() says which
// have to be there.  There is no destination register.
// m0 is a register that the compiler keeps for itself and warns about: it holds nothing
// across a statement that names it, which is all that is asked.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int INST>
__device__ __forceinline__ void load_to_lds(uint32_t to, uint64_t base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
                 :
                 : "s"(to), "v"(offset), "s"(base), "n"(INST)
                 : "m0", "memory");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)(p)));
}

__device__ __forceinline__ float read_only(const float *p) {
    return *(const __attribute__((address_space(4))) float *)(p);
}

// Queries of a workgroup's rows into LDS as int8 operands, [set][chunk][lane][16]:
// a row scaled by a power of two to magnitudes below 1, times 127, as digits to the
// base 256, the leading one in [-127, 127].  A digit a set in the row's column: three
// (2^-24 of that power of two: bf16 elements down to 2^-9 of the row's largest are
// exact, fp16 ones to 2^-6); with SPLIT four, two a set in columns r and r + 8.
// 16 threads a row, 32 where there are no more than 8 rows; `thread` of THREADS.
template <bool SPLIT>
constexpr int kSets = SPLIT ? 2 : 3;

template <int D, Dtype DT, bool SPLIT, int THREADS>
__device__ __forceinline__ void stage_queries(const Kv8AttentionParams &p, const RowTile &tile, int row0, int kvh, int thread,
    uint32_t *operands, float *factors) {
    typedef typename Element<DT>::type E;
    constexpr int kRows = SPLIT ? 8 : 16, kS = kSets<SPLIT>, kDigits = SPLIT ? 2 * kS : kS;
    constexpr float kOne = 127.0f * (kDigits == 4 ? 16777216.0f : 65536.0f);
    constexpr int kThreads = D >= 128 && kRows == 8 ? 32 : 16, kSteps = D / 4 / kThreads;
#pragma unroll 1
    for (int base = 0; base < kRows; base += THREADS / kThreads) {
        const int local = base + thread / kThreads, part = thread % kThreads, row = row0 + local;
        if (local >= kRows) break;
        const bool there = row < tile.total;
        const int token = there ? row / p.group : 0, head = kvh * p.group + (there ? row % p.group : 0);
        const E *at = static_cast<const E *>(p.q) + static_cast<int64_t>(tile.begin + token) * p.q_row +
            static_cast<int64_t>(head) * p.q_head;
        f32x4_t v[kSteps];
        float top = 0.0f;
        if (p.vec) {
#pragma unroll
            for (int c = 0; c < kSteps; ++c) v[c] = load4<DT, true>(at + 4 * (kThreads * c + part));
        } else {
#pragma unroll
            for (int c = 0; c < kSteps; ++c) v[c] = load4<DT, false>(at + 4 * (kThreads * c + part));
        }
        float poison = 0.0f;  // NaN where an element is not finite: the digits cannot say so
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                top = fmaxf(top, fabsf(v[c][i]));
                poison += v[c][i] * 0.0f;
            }
        top = fmaxf(top, xor_lane<1>(top));
        top = fmaxf(top, xor_lane<2>(top));
        top = fmaxf(top, xor_lane<4>(top));
        top = fmaxf(top, xor_lane<8>(top));
        if constexpr (kThreads == 32) top = fmaxf(top, xor_lane<16>(top));
        poison += xor_lane<1>(poison);
        poison += xor_lane<2>(poison);
        poison += xor_lane<4>(poison);
        poison += xor_lane<8>(poison);
        if constexpr (kThreads == 32) poison += xor_lane<16>(poison);
        const int e = __builtin_amdgcn_frexp_expf(top);
        const float one = p.scale_log2 < 0.0f ? -kOne : kOne;  // so that factors are not negative
        if (part == 0) factors[local] = __builtin_ldexpf(fabsf(p.scale_log2), e) * (1.0f / 127.0f) + poison;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            uint32_t digits[kDigits];
#pragma unroll
            for (int k = 0; k < kDigits; ++k) digits[k] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int x = poison == 0.0f ? static_cast<int>(__builtin_rintf(__builtin_ldexpf(v[c][i], -e) * one)) : 0;
#pragma unroll
                for (int k = kDigits - 1; k >= 0; --k) {
                    const int digit = k > 0 ? static_cast<int8_t>(x) : x;
                    digits[k] |= (static_cast<uint32_t>(digit) & 0xffu) << (8 * i);
                    x = (x - digit) >> 8;
                }
            }
#pragma unroll
            for (int k = 0; k < kDigits; ++k) {
                const int set = SPLIT ? k >> 1 : k, column = SPLIT ? local + 8 * (k & 1) : local;
                const int four = kThreads * c + part;  // of the row's groups of four dims: 16 a chunk, 4 a lane
                operands[(set * (D / 64) + (four >> 4)) * 256 + (((four & 15) >> 2) * 16 + column) * 4 + (four & 3)] = digits[k];
            }
        }
    }
}

// Every wave has its tile's codes brought to LDS of its own by loads that leave no
// trace in registers: 1 KiB a load, whole rows, so that lines are read whole (a
// lane's operands lie in 16 rows: read from memory directly, they took five times as
// many accesses).  What a lane reads from LDS is 16 bytes of row r; the units of 16
// bytes are permuted within a row (by the load's source address) so that the lanes
// that are served together find different banks: 64 banks, 16 lanes at a time, rows
// 0-3 and 12-15 of one g with rows 4-11 of its neighbour.
//
// Keys: token T of the tile in rows of D, unit x at x ^ f(T) with f from T's lane,
//   r(T) = (T / 16) 4 + T % 4.  Values: pages of P tokens one behind the other, dim d
//   in rows of P, unit x at x ^ f(d) (f = 0 for pages of 16 and 32).
template <int D>
__device__ __forceinline__ int key_turn(int r) {
    return D == 256 ? r : D == 128 ? r >> 1 : 3 * (r >> 3);
}

template <int D, bool SPLIT>
struct FewLds {
    static constexpr int kRows = SPLIT ? 8 : 16;  // in an instruction's 16 columns
    union {
        u32x4_t codes[kWaves][kTileTokens * (D / 16)];  // a tile's keys, then its values
        f32x4_t join[kWaves][D / 16][64];               // a wave's results for 16 columns
    } tiles;
    i32x4_t operands[kSets<SPLIT>][D / 64][64];
    float factors[kRows];
    f32x4_t joins[kWaves][kRows];  // a wave's base (score, value) and denominator (base, sum)
};

template <int D, Dtype DT, bool SPLIT, bool SHARING>
__device__ __forceinline__ void attend_few(const Kv8AttentionParams &p, FewLds<D, SPLIT> &memory) {
    typedef typename Element<DT>::type E;
    constexpr int kRows = FewLds<D, SPLIT>::kRows, kS = kSets<SPLIT>;
    constexpr int kChunks = D / 64, kDims = D / 16;
    constexpr int kUnits = D / 16;                  // of a key row
    auto &lds = memory.tiles;
    auto &operands = memory.operands;
    auto &factors = memory.factors;
    auto &joins = memory.joins;

    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    Work work;
    if constexpr (SHARING) work = work_of<true, kRows>(p);
    const int seq = SHARING ? work.seq : blockIdx.z;
    const int split = SHARING ? work.split : blockIdx.x, step = (SHARING ? work.splits : p.splits) * kWaves;
    const int first = (SHARING ? work.first_tile : 0) + split * kWaves + wave;
    const int P = p.cache.page_tokens, shift_p = 31 - __builtin_clz(P), row_shift = shift_p - 4;
    // the pages of a tile's four groups of 16 tokens
    int page0, page1, page2, page3;
    const auto find_page = [&](int token) {
        return __builtin_amdgcn_readfirstlane(p.batch.page(seq, token >> shift_p, p.cache.pages));
    };
    const auto find_pages = [&](int n) {
        page0 = find_page(n * kTileTokens);
        page1 = find_page(n * kTileTokens + 16);
        page2 = find_page(n * kTileTokens + 32);
        page3 = find_page(n * kTileTokens + 48);
    };
    find_pages(first);  // on its way beside the sequence's own numbers
    if constexpr (!SHARING) work = work_of<false, kRows>(p);
    const int kvh = work.kvh, row0 = work.row0;
    const RowTile tile = work.tile;
    if (row0 >= tile.total) return;
    if (split > 0 && work.first_tile + split * kWaves >= tile.tiles) return;  // the join does not look at it
    const bool whole = !SHARING && p.splits == 1;

    const size_t page_stride = static_cast<size_t>(p.cache.kv_heads) * P * D;
    const uint64_t keys = reinterpret_cast<uint64_t>(p.cache.keys) + static_cast<size_t>(kvh) * P * D;
    const uint64_t values = reinterpret_cast<uint64_t>(p.cache.values) + static_cast<size_t>(kvh) * P * D;
    const u32x4_t *value_codes = lds.codes[wave];
    const i32x4_t *key_codes = reinterpret_cast<const i32x4_t *>(value_codes);
    const uint32_t codes_to = __builtin_amdgcn_readfirstlane(lds_address(value_codes));
    // a load takes 1024 / D tokens, D / 64 loads a group of 16, in which the lanes' units turn alike
    uint32_t key_from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        key_from[i] = (lane / kUnits) * D + 16 * ((lane % kUnits) ^ (key_turn<D>(4 * i + (lane / kUnits & 3)) & (kUnits - 1)));
    // value rows are P / 16 units
    const int row_units = P / 16;
    const uint32_t value_from = (lane >> row_shift) * P + 16 * ((lane & (row_units - 1)) ^ (P == 64 ? 3 * (lane >> 5) : 0));
    // a quarter of a tile: 16 D bytes of a page, the tokens' keys or the part of the values' page that is as long
    const auto load_quarter = [&](uint64_t plane, int page, int i, uint32_t from) {
        const uint64_t base = plane + static_cast<uint64_t>(max(page, 0)) * page_stride + ((16 * i) & (P - 1)) * D;
        const uint32_t to = codes_to + i * 16 * D;
        load_to_lds<0>(to, base, from);
        if constexpr (D >= 128) load_to_lds<1024>(to, base, from);
        if constexpr (D >= 256) load_to_lds<2 * 1024>(to, base, from);
        if constexpr (D >= 256) load_to_lds<3 * 1024>(to, base, from);
    };
    const auto load_keys = [&]() {
        load_quarter(keys, page0, 0, key_from[0]);
        load_quarter(keys, page1, 1, key_from[1]);
        load_quarter(keys, page2, 2, key_from[2]);
        load_quarter(keys, page3, 3, key_from[3]);
    };
    const auto load_values = [&]() {
        load_quarter(values, page0, 0, value_from);
        load_quarter(values, page1, 1, value_from);
        load_quarter(values, page2, 2, value_from);
        load_quarter(values, page3, 3, value_from);
    };
    if (first < tile.tiles) load_keys();

    stage_queries<D, DT, SPLIT, kWaves * 64>(p, tile, row0, kvh, threadIdx.x, reinterpret_cast<uint32_t *>(operands), factors);
    lds_barrier();

    const int col = SPLIT ? r & 7 : r;
    const bool low = SPLIT && r >= 8;
    const float share = low ? 1.0f / kLoScale : 1.0f;
    // what the digits of the first and the last set weigh
    const float weight0 = low ? 1.0f / 256.0f : 1.0f, weight = (SPLIT ? weight0 : 1.0f) / 65536.0f;
    const int row = row0 + col;
    const float factor = factors[col];  // of S: softmax scale, log2 e, the query's power of two, 1 / 127^2
    const int position = row < tile.total ? tile.length + row / p.group : -1;  // the last token that the row sees
    f32x4_t o[kDims];
    Base m = {kNone, 0.0f};  // of o
    Denominator l;           // of this lane's tokens
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    // where this lane's operands lie
    const int key_at = (16 * (r >> 2) + (r & 3)) * kUnits, key_turned = key_turn<D>(r) & (kUnits - 1);
    const int value_at = ((g >> row_shift) << row_shift) * D + (r << row_shift) +
        ((g & (row_units - 1)) ^ (P == 64 ? 3 * (r >> 3) : 0));

#pragma unroll 1
    for (int n = first; n < tile.tiles; n += step) {
        const int token = n * kTileTokens + 16 * g;  // the first of this lane's 16
        // the magnitudes of the four groups' pages, asked for together; a page that holds no token yet may hold
        // anything: its magnitudes are not used, and its codes are finite whatever they are
        const auto top_at = [&](const float *tops, int page) {
            return read_only(tops + static_cast<size_t>(max(page, 0)) * p.cache.kv_heads + kvh);
        };
        float key_top0 = top_at(p.cache.key_max, page0), key_top1 = top_at(p.cache.key_max, page1);
        float key_top2 = top_at(p.cache.key_max, page2), key_top3 = top_at(p.cache.key_max, page3);
        float value_top0 = top_at(p.cache.value_max, page0), value_top1 = top_at(p.cache.value_max, page1);
        float value_top2 = top_at(p.cache.value_max, page2), value_top3 = top_at(p.cache.value_max, page3);
        const int next = n + step;
        wait_loads<0>();  // the keys have landed

        i32x4_t s[kS][4];
#pragma unroll
        for (int set = 0; set < kS; ++set)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[set][u] = i32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            i32x4_t k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) k[u] = key_codes[key_at + 4 * u * kUnits + ((4 * c + g) ^ key_turned)];
#pragma unroll
            for (int set = 0; set < kS; ++set) {
                const i32x4_t q = operands[set][c][lane];
#pragma unroll
                for (int u = 0; u < 4; ++u) s[set][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[u], q, s[set][u], 0, 0, 0);
            }
        }
        wait_lds();
        load_values();
        asm volatile("" : "+s"(key_top0), "+s"(key_top1), "+s"(key_top2), "+s"(key_top3));  // not one by one where they
        asm volatile("" : "+s"(value_top0), "+s"(value_top1), "+s"(value_top2), "+s"(value_top3));  // are chosen from
        const auto mine = [&](auto a0, auto a1, auto a2, auto a3) {
            const auto x = g & 1 ? a1 : a0, y = g & 1 ? a3 : a2;
            return g & 2 ? y : x;
        };
        const bool there = mine(page0, page1, page2, page3) >= 0 && token < tile.seen;
        const float key_top = there ? mine(key_top0, key_top1, key_top2, key_top3) : 0.0f;
        const float value_top = there ? mine(value_top0, value_top1, value_top2, value_top3) : 0.0f;
        find_pages(next);
        f16x8_t b[SPLIT ? 2 : 4];  // the weights of tokens 0..7 and 8..15, then their lower halves
        {
            const float f = factor * key_top;
            const int seen = there ? position + 1 - token : 0;  // of this lane's 16 tokens
            float x[16];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // sums of up to 256 products of two digits: exact in fp32
                    float y = static_cast<float>(s[kS - 1][u][i]) * weight;
                    if constexpr (!SPLIT) y = __builtin_fmaf(static_cast<float>(s[1][u][i]), 1.0f / 256.0f, y);
                    y = SPLIT ? __builtin_fmaf(static_cast<float>(s[0][u][i]), weight0, y) : y + static_cast<float>(s[0][u][i]);
                    if constexpr (SPLIT) y = y + xor_lane<8>(y);
                    x[4 * u + i] = y * f;
                }
            if (__any(seen < 16)) {
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = j < seen ? x[j] : -__builtin_inff();
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]);
            const bool some = top > -__builtin_inff();
            const float whole = some ? __builtin_rintf(top) : 0.0f;
            // a page of zeros counts in the denominator, but has no products
            const Base own = {some && value_top > 0.0f ? whole : kNone, static_cast<float>(__builtin_amdgcn_frexp_expf(value_top))};
            const Base now = largest_of_row(own, __any(fabsf(whole) >= kHuge));
            const float higher = above(now, m);
            const float alpha = exp2_fast(-fmaxf(higher, 0.0f));
            if (higher > 0.0f) m = now;
            const float rest = exp2_fast(above(own, m)) * (__builtin_amdgcn_frexp_mantf(value_top) * kPScale);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = exp2_fast(x[j] - whole);
                sum += e;
                const float y = rounded(e * rest);
                _Float16 h = static_cast<_Float16>(y);
                const float left = y - static_cast<float>(h);
                if constexpr (SPLIT) h = low ? static_cast<_Float16>(left * kLoScale) : h;
                else b[2 + (j >> 3)][j & 7] = static_cast<_Float16>(left);
                b[j >> 3][j & 7] = h;
            }
            l.add(some ? whole : kNone, sum);
            if (n != first && __any(alpha != 1.0f)) {
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
            }
        }
        wait_loads<0>();  // the values have landed
        u32x4_t v[kDims];
#pragma unroll
        for (int d = 0; d < kDims; ++d) v[d] = value_codes[value_at + ((16 * d) << row_shift)];
        asm volatile("" ::: "memory");
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            const f16x8_t a0 = codes_to_half(v[d][0], v[d][1]), a1 = codes_to_half(v[d][2], v[d][3]);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b[1], o[d], 0, 0, 0);
            if constexpr (!SPLIT) {
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b[2], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b[3], o[d], 0, 0, 0);
            }
        }
        if (next < tile.tiles) {
            wait_lds();
            load_keys();
        }
    }

    // ---- join the waves
    l.add_lane<16>();
    l.add_lane<32>();
    if (g == 0 && !low) joins[wave][col] = f32x4_t{m.score, m.value, l.base, l.sum};
    lds_barrier();
    Base top = {kNone, 0.0f};
    Denominator total;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const f32x4_t join = joins[w][col];
        const Base other = {join[0], join[1]};
        if (above(other, top) > 0.0f) top = other;
        total.add(join[2], join[3]);
    }
    const float scale = exp2_fast(above(m, top)) * share;
#pragma unroll
    for (int d = 0; d < kDims; ++d) lds.join[wave][d][lane] = o[d] * scale;
    lds_barrier();
    if (low || row >= tile.total) return;
    const size_t item = work.item;
    const int head = kvh * p.group + row % p.group;
    const int64_t at = tile.begin + row / p.group;
    const Quotient quotient(top, total, kPScale);
#pragma unroll 1
    for (int d = wave * kChunks; d < (wave + 1) * kChunks; ++d) {
        f32x4_t y = lds.join[0][d][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) y += lds.join[w][d][lane];
        if constexpr (SPLIT) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) y += lds.join[w][d][lane + 8];
        }
        const int dim = 16 * d + 4 * g;
        if (!whole) *reinterpret_cast<f32x4_t *>(p.partial + (item * kRows + col) * D + dim) = y;
        else finish<DT>(p, quotient(y), quotient.some(), at, head, head * D + dim, dim);
    }
    if (!whole && wave == 0 && g == 0)
        p.partial_ml[item * kRows + col] = f32x4_t{top.score, top.value, total.base, total.sum};
}

template <int D, Dtype DT, bool SPLIT, bool SHARING>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attention_kernel(Kv8AttentionParams p) {
    __shared__ FewLds<D, SPLIT> lds;
    attend_few<D, DT, SPLIT, SHARING>(p, lds);
}

// Many rows (a prompt's chunk): 64 rows a workgroup (32 with SPLIT), which share every
// tile.  For the scores and their weights a wave has 16 (8) of the rows and the whole tile: its queries
// stay in registers, the keys come from LDS (double buffered).  The weights go to the
// other waves through LDS, because for the results a wave has all 64 rows and a
// quarter of the dims: the values that it needs are its own then, which it loads and
// turns into fp16 once for 64 rows.
//
// Scores: f y with y the digits' sum and f > 0 the same for a lane's 16 tokens (one
// page), so that only y is masked and searched for its largest.
//
// 2000 tokens of 16 heads (4 kv heads of 256) behind 6000: 367 to 383 us on three cards, 0.6
// PFLOP/s with a product of three digits or two halves counted once.  Matrix instructions (112 a wave's
// tile) are 54 % of a SIMD's time and its 400 vector instructions the rest: two waves a
// SIMD overlap little.  Where the products had two digits and one half (249 us; the
// 16-row kernel 409) a version in which every wave read the whole tile's values from LDS
// took 265, values by loads to LDS, as the keys, 273, and priority for the products was
// worth 12.
template <int D, bool SPLIT>
struct WideLds {
    static constexpr int kKeyUnits = kTileTokens * (D / 16);
    static constexpr int kHalves = SPLIT ? 1 : 2;  // of a weight, in a column
    union {
        struct {
            u32x4_t keys[2][kKeyUnits];
            f16x8_t weights[kHalves][kWaves][2][64];  // of a wave's rows
            f32x4_t alphas[16];              // of row r of the four waves
        } tile;
        struct {
            u32x4_t first_keys[kKeyUnits];  // loaded meanwhile
            i32x4_t operands[kWaves][kSets<SPLIT>][D / 64][64];
        } start;
        f32x4_t rows[kWaves][D / 16][64];
    } tiles;
    float factors[kWaves][16];
};

template <int D, Dtype DT, bool SPLIT, bool SHARING>
__device__ __forceinline__ void attend_wide(const Kv8AttentionParams &p, WideLds<D, SPLIT> &memory) {
    constexpr int kChunks = D / 64, kUnits = D / 16, kS = kSets<SPLIT>;
    constexpr int kMyRows = SPLIT ? 8 : 16, kRows = kWaves * kMyRows;
    constexpr int kKeyUnits = WideLds<D, SPLIT>::kKeyUnits, kHalves = WideLds<D, SPLIT>::kHalves;
    constexpr int kMine = D / 64;  // a wave's 16s of dims
    auto &lds = memory.tiles;
    auto &factors = memory.factors;

    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const Work work = work_of<SHARING, kRows>(p);
    const int seq = work.seq, kvh = work.kvh, row0 = work.row0, split = work.split, step = work.splits;
    const int first = work.first_tile + split;
    const int P = p.cache.page_tokens, shift_p = 31 - __builtin_clz(P);
    const RowTile tile = work.tile;
    if (row0 >= tile.total) return;
    if (split > 0 && first >= tile.tiles) return;  // the join does not look at it
    const bool whole_rows = !SHARING && p.splits == 1;

    const size_t page_stride = static_cast<size_t>(p.cache.kv_heads) * P * D;
    const uint64_t keys = reinterpret_cast<uint64_t>(p.cache.keys) + static_cast<size_t>(kvh) * P * D;
    const int8_t *values = p.cache.values + static_cast<size_t>(kvh) * P * D;
    // the page of tile n's tokens 16 g .. 16 g + 15: its word of the table, looked at once it is there (where the
    // table ends, tile.seen ends too)
    const auto page_id = [&](int n) { return p.batch.page_word(seq, (n * kTileTokens + 16 * g) >> shift_p); };
    const auto checked = [&](int id) { return id >= 0 && id < p.cache.pages ? id : -1; };
    const uint32_t key_from = (lane / kUnits) * D + 16 * ((lane % kUnits) ^ (key_turn<D>(4 * wave + (lane / kUnits & 3)) & (kUnits - 1)));
    const uint32_t keys_to = __builtin_amdgcn_readfirstlane(lds_address(lds.tile.keys[0]));
    // this wave's 16 tokens of a tile
    const auto load_keys = [&](int page, int buffer) {
        const int mine = __builtin_amdgcn_readlane(page, 16 * wave);
        const uint64_t base = keys + static_cast<uint64_t>(max(mine, 0)) * page_stride + ((16 * wave) & (P - 1)) * D;
        const uint32_t to = keys_to + (buffer * kKeyUnits + wave * 16 * kUnits) * 16;
        load_to_lds<0>(to, base, key_from);
        if constexpr (D >= 128) load_to_lds<1024>(to, base, key_from);
        if constexpr (D >= 256) load_to_lds<2 * 1024>(to, base, key_from);
        if constexpr (D >= 256) load_to_lds<3 * 1024>(to, base, key_from);
    };
    // this wave's dims of a tile's values as they are operands: the lane's 16 tokens of dim r of each 16
    u32x4_t codes[kMine];
    const auto load_values = [&](int page) {
        const int8_t *from = values + static_cast<size_t>(max(page, 0)) * page_stride +
            static_cast<size_t>(wave * (D / 4) + r) * P + ((16 * g) & (P - 1));
#pragma unroll
        for (int i = 0; i < kMine; ++i) codes[i] = *reinterpret_cast<const u32x4_t *>(from + 16 * i * P);
    };
    float key_top, value_top;  // of this lane's page
    const auto load_tops = [&](int page) {
        const size_t at = static_cast<size_t>(max(page, 0)) * p.cache.kv_heads + kvh;
        key_top = p.cache.key_max[at];
        value_top = p.cache.value_max[at];
    };
    int page = checked(page_id(first)), next_id = -1;  // the page of this tile, and the word that says the next one's
    if (first < tile.tiles) {
        load_keys(page, 0);
        load_tops(page);
        next_id = page_id(first + step);
        load_values(page);
    }
    stage_queries<D, DT, SPLIT, 64>(p, tile, row0 + kMyRows * wave, kvh, lane, reinterpret_cast<uint32_t *>(lds.start.operands[wave]),
        factors[wave]);
    wait_lds();  // its own wave's rows only
    i32x4_t q[kS][kChunks];
#pragma unroll
    for (int set = 0; set < kS; ++set)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) q[set][c] = lds.start.operands[wave][set][c][lane];
    const int col = SPLIT ? r & 7 : r, row = row0 + kMyRows * wave + col;
    const bool low = SPLIT && r >= 8;
    const float factor = factors[wave][col] * (SPLIT ? 1.0f : 1.0f / 65536.0f);  // per unit of the last digit
    const float weight0 = low ? 1.0f / 256.0f : 1.0f;  // of a first digit, where they are four
    const int position = row < tile.total ? tile.length + row / p.group : -1;  // the last token that the row sees
    f32x4_t o[kWaves][kMine];  // of row r of every wave's
    Base m = {kNone, 0.0f};
    Denominator l;  // of this lane's tokens
#pragma unroll
    for (int t = 0; t < kWaves; ++t)
#pragma unroll
        for (int i = 0; i < kMine; ++i) o[t][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int key_at = (16 * (r >> 2) + (r & 3)) * kUnits, key_turned = key_turn<D>(r) & (kUnits - 1);

    int buffer = 0;
#pragma unroll 1
    for (int n = first; n < tile.tiles; n += step) {
        const bool more = n + step < tile.tiles;
        wait_loads<kMine>();  // all but the values, which were asked for last
        lds_barrier();  // every wave's keys are there, and its products with the tile before done
        const int token = n * kTileTokens + 16 * g;  // the first of this lane's 16
        const bool there = page >= 0 && token < tile.seen;
        const float k_top = there ? key_top : 0.0f, v_top = there ? value_top : 0.0f;
        page = checked(next_id);
        if (more) {
            load_keys(page, buffer ^ 1);
            load_tops(page);
            next_id = page_id(n + 2 * step);
        }

        const i32x4_t *key_codes = reinterpret_cast<const i32x4_t *>(lds.tile.keys[buffer]);
        i32x4_t s[kS][4], k[2][4];
        const auto read_keys = [&](int c) {
#pragma unroll
            for (int u = 0; u < 4; ++u) k[c & 1][u] = key_codes[key_at + 4 * u * kUnits + ((4 * c + g) ^ key_turned)];
        };
#pragma unroll
        for (int set = 0; set < kS; ++set)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[set][u] = i32x4_t{0, 0, 0, 0};
        read_keys(0);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            if (c + 1 < kChunks) read_keys(c + 1);
            __builtin_amdgcn_sched_barrier(kArithmeticMayCross);
#pragma unroll
            for (int set = 0; set < kS; ++set)
#pragma unroll
                for (int u = 0; u < 4; ++u) s[set][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[c & 1][u], q[set][c], s[set][u], 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        // digits' sums: up to 256 * 127^2 the leading one's, which leaves room for one more digit in 32 bits; four digits
        // are two of the row's column and two of the one 8 further on
        float y[16];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (SPLIT) {
                    const float half = __builtin_fmaf(static_cast<float>(s[0][u][i]), weight0,
                        static_cast<float>(s[1][u][i]) * (weight0 / 65536.0f));
                    y[4 * u + i] = half + xor_lane<8>(half);
                } else {
                    const float last = static_cast<float>(s[1][u][i] * 256 + s[kS - 1][u][i]);
                    y[4 * u + i] = __builtin_fmaf(static_cast<float>(s[0][u][i]), 65536.0f, last);
                }
            }
        const int seen = there ? position + 1 - token : 0;  // of this lane's 16 tokens
        if (__any(seen < 16)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = j < seen ? y[j] : -__builtin_inff();
        }
        // not 0 or NaN times infinity where masked
        const float product = seen > 0 ? factor * k_top : 0.0f, f = product == 0.0f ? 1.2e-38f : product;
        float top = y[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, y[j]);
        top *= f;
        const bool some = top > -__builtin_inff();
        const float whole = some ? __builtin_rintf(top) : 0.0f;
        const bool some_huge = __any(fabsf(whole) >= kHuge);
        float scale = f;
        if (some_huge) {  // the same rounded products as the largest one: exact ones may lie far above it
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] *= f;
            scale = 1.0f;
        }
        // a page of zeros counts in the denominator, but has no products
        const Base own = {some && v_top > 0.0f ? whole : kNone, static_cast<float>(__builtin_amdgcn_frexp_expf(v_top))};
        const Base now = largest_of_row(own, some_huge);
        // a new base only where the old one is left behind by more than 2^4
        const float higher = above(now, m);
        const float alpha = higher > 4.0f ? exp2_fast(-higher) : 1.0f;
        if (higher > 4.0f) m = now;
        const float rest = exp2_fast(above(own, m)) * (__builtin_amdgcn_frexp_mantf(v_top) * kWideScale);
        float sum = 0.0f;
        f16x8_t b[kHalves][2];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float e0 = exp2_fast(__builtin_fmaf(y[j], scale, -whole)), e1 = exp2_fast(__builtin_fmaf(y[j + 1], scale, -whole));
            sum += e0 + e1;
            const f32x2_t e = {rounded(e0 * rest), rounded(e1 * rest)};
            f16x2_t h = __builtin_convertvector(e, f16x2_t);
            const f32x2_t left = e - __builtin_convertvector(h, f32x2_t);
            if constexpr (SPLIT) {
                h = low ? __builtin_convertvector(left * kLoScale, f16x2_t) : h;
            } else {
                const f16x2_t rest_of = __builtin_convertvector(left, f16x2_t);
                b[kHalves - 1][j >> 3][j & 7] = rest_of[0];
                b[kHalves - 1][j >> 3][(j & 7) + 1] = rest_of[1];
            }
            b[0][j >> 3][j & 7] = h[0];
            b[0][j >> 3][(j & 7) + 1] = h[1];
        }
        l.add(some ? whole : kNone, sum);
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
            lds.tile.weights[half][wave][0][lane] = b[half][0];
            lds.tile.weights[half][wave][1][lane] = b[half][1];
        }
        if (g == 0) reinterpret_cast<float *>(&lds.tile.alphas[r])[wave] = alpha;
        lds_barrier();  // every wave's weights are there
        __builtin_amdgcn_s_setprio(1);
        f16x8_t weights[kHalves][kWaves][2];
        const f32x4_t alphas = lds.tile.alphas[r];
#pragma unroll
        for (int half = 0; half < kHalves; ++half)
#pragma unroll
            for (int t = 0; t < kWaves; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) weights[half][t][k] = lds.tile.weights[half][t][k][lane];
        if (__any(alphas[0] != 1.0f || alphas[1] != 1.0f || alphas[2] != 1.0f || alphas[3] != 1.0f)) {
#pragma unroll
            for (int t = 0; t < kWaves; ++t)
#pragma unroll
                for (int i = 0; i < kMine; ++i) o[t][i] *= alphas[t];
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const f16x8_t a0 = codes_to_half(codes[i][0], codes[i][1]), a1 = codes_to_half(codes[i][2], codes[i][3]);
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
#pragma unroll
                for (int t = 0; t < kWaves; ++t)
                    o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, weights[half][t][0], o[t][i], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < kWaves; ++t)
                    o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, weights[half][t][1], o[t][i], 0, 0, 0);
            }
        }
        if (more) load_values(page);
        buffer ^= 1;
    }
    __builtin_amdgcn_s_setprio(0);

    l.add_lane<16>();
    l.add_lane<32>();
    const Quotient quotient = !whole_rows ? Quotient(kPScale / kWideScale, 0) : Quotient(m, l, kWideScale);
    lds_barrier();  // the last tile's products are done
#pragma unroll
    for (int t = 0; t < kWaves; ++t)
#pragma unroll
        for (int i = 0; i < kMine; ++i) lds.rows[t][wave * kMine + i][lane] = o[t][i];
    const size_t item = work.item;
    if (!whole_rows && g == 0 && !low)
        p.partial_ml[item * kRows + kMyRows * wave + col] = f32x4_t{m.score, m.value, l.base, l.sum};
    lds_barrier();
    // the rows that the wave has the sums of: a row's dims, four a lane, in as many rows at a time as a wave holds
    constexpr int kLanes = D / 4, kTogether = 64 / kLanes;
    const int four = lane % kLanes, dim = 4 * four;
#pragma unroll 1
    for (int k = 0; k < kMyRows; k += kTogether) {
        const int local = k + lane / kLanes, at = row0 + kMyRows * wave + local;
        const Quotient row_quotient(__shfl(quotient.norm, local), __shfl(quotient.exponent, local));
        if (at >= tile.total) break;
        f32x4_t y = lds.rows[wave][four >> 2][16 * (four & 3) + local];
        if constexpr (SPLIT) y += lds.rows[wave][four >> 2][16 * (four & 3) + local + 8] * (1.0f / kLoScale);
        y = row_quotient(y);
        const int head = kvh * p.group + at % p.group;
        if (!whole_rows) *reinterpret_cast<f32x4_t *>(p.partial + (item * kRows + kMyRows * wave + local) * D + dim) = y;
        else finish<DT>(p, y, row_quotient.some(), tile.begin + at / p.group, head, head * D + dim, dim);
    }
}

template <int D, Dtype DT, bool SPLIT, bool SHARING>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attention_wide_kernel(Kv8AttentionParams p) {
    __shared__ WideLds<D, SPLIT> lds;
    attend_wide<D, DT, SPLIT, SHARING>(p, lds);
}

// Many rows of groups, few of each sequence's: both in one launch, so that the second
// fills what the first leaves.  32 sequences (16 heads, 4 kv heads of 256, fp32) with up to 190
// tokens of their own behind 8000 shared ones: 29 us, where two launches took 28 and 10.
template <int D, Dtype DT, bool FEW_SPLIT, bool WIDE_SPLIT>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attention_both_kernel(Kv8AttentionParams p) {
    __shared__ union {
        FewLds<D, FEW_SPLIT> few;
        WideLds<D, WIDE_SPLIT> wide;
    } lds;
    if (static_cast<int>(blockIdx.x) < p.sharing.groups * p.shared_row_tiles * p.cache.kv_heads * p.shared_splits)
        attend_wide<D, DT, WIDE_SPLIT, true>(p, lds.wide);
    else
        attend_few<D, DT, FEW_SPLIT, true>(p, lds.few);
}

// The splits of one row and head, 64 dims a workgroup: four dims a lane, 16 or 32
// splits side by side, so that up to 128 are on their way at once.
template <int D, Dtype DT, int THREADS>
__global__ __launch_bounds__(THREADS) void kv8_attention_join_kernel(Kv8AttentionParams p, int tile_rows) {
    constexpr int kLanes = 16, kGroups = THREADS / kLanes;
    __shared__ float weight[kKv8MaxSplits];
    __shared__ f32x4_t sums[kGroups][kLanes];
    const int seq = blockIdx.z, kvh = blockIdx.y / (D / 64), slice = blockIdx.y % (D / 64), row = blockIdx.x;
    const int row0 = row / tile_rows * tile_rows;
    const RowTile tile = row_tile(p, seq, row0, tile_rows);
    if (row >= tile.total) return;
    const int together = tile_rows > 16 ? 1 : kWaves;  // tiles that a workgroup's waves take at once
    const int active = min(p.splits, max((tile.tiles + together - 1) / together, 1));
    const size_t y_index = static_cast<size_t>(row / tile_rows) * p.cache.kv_heads + kvh;
    const size_t tiles_y = static_cast<size_t>(p.row_tiles) * p.cache.kv_heads;
    const size_t item = (static_cast<size_t>(seq) * tiles_y + y_index) * p.splits;
    const f32x4_t *ml = p.partial_ml + item * tile_rows + row % tile_rows;

    const int lane = threadIdx.x & 63;
    const int group = threadIdx.x / kLanes, at = threadIdx.x % kLanes, dim = 64 * slice + 4 * at;
    const float *from = p.partial + (item * tile_rows + row % tile_rows) * D + dim;
    const size_t step = static_cast<size_t>(tile_rows) * D;
    // the first four splits of a group, before the weights are known
    f32x4_t early[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        early[k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (group + k * kGroups < active) early[k] = *reinterpret_cast<const f32x4_t *>(from + (group + k * kGroups) * step);
    }
    Base top = {kNone, 0.0f};
    Denominator total;
#pragma unroll 1
    for (int i = lane; i < active; i += 64) {
        const f32x4_t join = ml[static_cast<size_t>(i) * tile_rows];
        const Base other = {join[0], join[1]};
        if (above(other, top) > 0.0f) top = other;
        total.add(join[2], join[3]);
    }
    top = larger_of_lanes<32>(top);
    top = larger_of_lanes<16>(top);
    top = larger_of_lanes<8>(top);
    top = larger_of_lanes<4>(top);
    top = larger_of_lanes<2>(top);
    top = larger_of_lanes<1>(top);
    total.add_lane<32>();
    total.add_lane<16>();
    total.add_lane<8>();
    total.add_lane<4>();
    total.add_lane<2>();
    total.add_lane<1>();
    if (threadIdx.x < 64) {
#pragma unroll 1
        for (int i = lane; i < active; i += 64) {
            const f32x4_t join = ml[static_cast<size_t>(i) * tile_rows];
            const Base other = {join[0], join[1]};
            weight[i] = exp2_fast(above(other, top));
        }
    }
    lds_barrier();
    f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (group + k * kGroups < active) y += early[k] * weight[group + k * kGroups];
#pragma unroll 1
    for (int i = group + 4 * kGroups; i < active; i += kGroups) y += *reinterpret_cast<const f32x4_t *>(from + i * step) * weight[i];
    sums[group][at] = y;
    lds_barrier();
    if (threadIdx.x >= kLanes) return;
    const int used = min(active, kGroups);
#pragma unroll 4
    for (int k = 1; k < used; ++k) y += sums[k][at];
    const Quotient quotient(top, total, kPScale);
    const int head = kvh * p.group + row % p.group;
    finish<DT>(p, quotient(y), quotient.some(), tile.begin + row / p.group, head, head * D + dim, dim);
}

// The same where a row's tokens are its group's, then its own: the partial results of
// both.  One wave does 64 dims where it can have a quarter of the partial results on their
// way at once: four waves of fewer each fill the chip's places twice (32 sequences of 4 kv
// heads, 33 partial results a row: 8.3 us against 10.0; 17 of them 6.5).
template <int D, Dtype DT, int THREADS>
__global__ __launch_bounds__(THREADS) void kv8_shared_join_kernel(Kv8AttentionParams p) {
    constexpr int kLanes = 16, kGroups = THREADS / kLanes, kEarly = THREADS == 64 ? 8 : 4;
    __shared__ float weight[2 * kKv8MaxSplits];
    __shared__ f32x4_t sums[kGroups][kLanes];
    const int seq = blockIdx.z, kvh = blockIdx.y / (D / 64), slice = blockIdx.y % (D / 64), row = blockIdx.x;
    const RowTile tile = row_tile(p, seq, row / p.own_rows * p.own_rows, p.own_rows);
    if (row >= tile.total) return;
    int index;
    const Group g = shared_by(p, seq, tile, &index);
    const auto active = [](int tiles, int splits, int rows) {
        const int together = rows > 16 ? 1 : kWaves;  // tiles that a workgroup's waves take at once
        return min(splits, max((tiles + together - 1) / together, 1));
    };
    const int own = active(tile.tiles - g.shared / kTileTokens, p.splits, p.own_rows);
    const int all = own + (g.shared > 0 ? active(g.shared / kTileTokens, p.shared_splits, p.shared_rows) : 0);
    // place of this row in the first split of either
    const int group_row = (tile.begin - g.begin) * p.group + row;
    const auto place = [&](int who, int tiles, int at, int rows, int splits) {
        return (((static_cast<int64_t>(who) * tiles + at / rows) * p.cache.kv_heads + kvh) * splits) * rows + at % rows;
    };
    const int64_t own_at = p.own_at + place(seq, p.row_tiles, row, p.own_rows, p.splits);
    const int64_t group_at = place(max(index, 0), p.shared_row_tiles, group_row, p.shared_rows, p.shared_splits);
    const auto partial_row = [&](int i) {
        return i < own ? own_at + static_cast<int64_t>(i) * p.own_rows : group_at + static_cast<int64_t>(i - own) * p.shared_rows;
    };

    // the first partial results of a group and the row's gates, before the weights are known
    const int lane = threadIdx.x & 63;
    const int group = threadIdx.x / kLanes, at = threadIdx.x % kLanes, dim = 64 * slice + 4 * at;
    const int head = kvh * p.group + row % p.group;
    f32x4_t early[kEarly], gates = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
        early[k] = *reinterpret_cast<const f32x4_t *>(p.partial + partial_row(min(group + k * kGroups, all - 1)) * D + dim);
    if (p.gate) gates = load_gate<DT>(p, tile.begin + row / p.group, head, dim);
    Base top = {kNone, 0.0f};
    Denominator total;
#pragma unroll 1
    for (int i = lane; i < all; i += 64) {
        const f32x4_t join = p.partial_ml[partial_row(i)];
        const Base other = {join[0], join[1]};
        if (above(other, top) > 0.0f) top = other;
        total.add(join[2], join[3]);
    }
    top = larger_of_lanes<32>(top);
    top = larger_of_lanes<16>(top);
    top = larger_of_lanes<8>(top);
    top = larger_of_lanes<4>(top);
    top = larger_of_lanes<2>(top);
    top = larger_of_lanes<1>(top);
    total.add_lane<32>();
    total.add_lane<16>();
    total.add_lane<8>();
    total.add_lane<4>();
    total.add_lane<2>();
    total.add_lane<1>();
    if (threadIdx.x < 64) {
#pragma unroll 1
        for (int i = lane; i < all; i += 64) {
            const f32x4_t join = p.partial_ml[partial_row(i)];
            const Base other = {join[0], join[1]};
            weight[i] = exp2_fast(above(other, top));
        }
    }
    lds_barrier();
    f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
        if (group + k * kGroups < all) y += early[k] * weight[group + k * kGroups];
#pragma unroll 4
    for (int i = group + kEarly * kGroups; i < all; i += kGroups) y += *reinterpret_cast<const f32x4_t *>(p.partial + partial_row(i) * D + dim) * weight[i];
    sums[group][at] = y;
    lds_barrier();
    if (threadIdx.x >= kLanes) return;
    const int used = min(all, kGroups);
#pragma unroll 4
    for (int k = 1; k < used; ++k) y += sums[k][at];
    const Quotient quotient(top, total, kPScale);
    finish<DT, true>(p, quotient(y), quotient.some(), tile.begin + row / p.group, head, head * D + dim, dim, &gates);
}

// `blocks` blocks from first_block on, of the groups' and the sequences' one after the other
template <int D, Dtype DT, int ROWS>
hipError_t launch_shared_rows(Kv8AttentionParams p, int first_block, int blocks, hipStream_t stream) {
    p.first_block = first_block;
    constexpr bool kSplit = ROWS == 8 || ROWS == 32;
    if constexpr (ROWS > 16) hipLaunchKernelGGL((kv8_attention_wide_kernel<D, DT, kSplit, true>), dim3(blocks), dim3(kWaves * 64), 0, stream, p);
    else hipLaunchKernelGGL((kv8_attention_kernel<D, DT, kSplit, true>), dim3(blocks), dim3(kWaves * 64), 0, stream, p);
    return hipGetLastError();
}

template <int D, Dtype DT>
hipError_t launch_shared_typed(Kv8AttentionParams p, const Kv8SharedPlan &cut, hipStream_t stream) {
    const Kv8Plan &plan = cut.own, &shared = cut.group;
    p.own_at = static_cast<int>(cut.own_at);
    p.splits = plan.splits;
    p.row_tiles = plan.row_tiles;
    p.own_rows = plan.rows;
    p.shared_splits = shared.splits;
    p.shared_row_tiles = shared.row_tiles;
    p.shared_rows = shared.rows;
    const int heads = p.cache.kv_heads;
    const int of_groups = p.sharing.groups * shared.row_tiles * heads * shared.splits, own = p.batch.sequences * plan.row_tiles * heads * plan.splits;
    const auto launch = [&](int rows, int first_block, int blocks) {
        if constexpr (DT == Dtype::F32)
            return rows == 8 ? launch_shared_rows<D, DT, 8>(p, first_block, blocks, stream) : launch_shared_rows<D, DT, 32>(p, first_block, blocks, stream);
        else
            return rows == 8 ? launch_shared_rows<D, DT, 8>(p, first_block, blocks, stream)
                : rows == 16 ? launch_shared_rows<D, DT, 16>(p, first_block, blocks, stream)
                             : launch_shared_rows<D, DT, 64>(p, first_block, blocks, stream);
    };
    const auto launch_both = [&](auto kernel) {
        p.first_block = 0;
        hipLaunchKernelGGL(kernel, dim3(of_groups + own), dim3(kWaves * 64), 0, stream, p);
        return hipGetLastError();
    };
    hipError_t e;
    if (plan.rows == shared.rows) {
        e = launch(plan.rows, 0, of_groups + own);
    } else if (plan.rows <= 16 && shared.rows > 16) {
        if constexpr (DT == Dtype::F32) e = launch_both(kv8_attention_both_kernel<D, DT, true, true>);
        else if (plan.rows == 8) e = launch_both(kv8_attention_both_kernel<D, DT, true, false>);
        else e = launch_both(kv8_attention_both_kernel<D, DT, false, false>);
    } else {
        e = launch(shared.rows, 0, of_groups);
        if (e == hipSuccess) e = launch(plan.rows, of_groups, own);
    }
    if (e != hipSuccess) return e;
    const dim3 rows(p.batch.max_rows * p.group, heads * (D / 64), p.batch.sequences);
    if (plan.splits + shared.splits <= 64) hipLaunchKernelGGL((kv8_shared_join_kernel<D, DT, 64>), rows, dim3(64), 0, stream, p);
    else hipLaunchKernelGGL((kv8_shared_join_kernel<D, DT, 256>), rows, dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <Dtype DT>
hipError_t launch_shared_head(const Kv8AttentionParams &p, const Kv8SharedPlan &plan, hipStream_t stream) {
    if (p.cache.head == 64) return launch_shared_typed<64, DT>(p, plan, stream);
    if (p.cache.head == 128) return launch_shared_typed<128, DT>(p, plan, stream);
    return launch_shared_typed<256, DT>(p, plan, stream);
}

template <int D, Dtype DT, int ROWS>
hipError_t launch_rows(Kv8AttentionParams p, const Kv8Plan &plan, hipStream_t stream) {
    const dim3 grid(plan.splits, plan.row_tiles * p.cache.kv_heads, p.batch.sequences);
    p.splits = plan.splits;
    p.row_tiles = plan.row_tiles;
    constexpr bool kSplit = ROWS == 8 || ROWS == 32;
    if constexpr (ROWS > 16) hipLaunchKernelGGL((kv8_attention_wide_kernel<D, DT, kSplit, false>), grid, dim3(kWaves * 64), 0, stream, p);
    else hipLaunchKernelGGL((kv8_attention_kernel<D, DT, kSplit, false>), grid, dim3(kWaves * 64), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && plan.splits > 1) {
        const dim3 rows(p.batch.max_rows * p.group, p.cache.kv_heads * (D / 64), p.batch.sequences);
        if (plan.splits <= 64) hipLaunchKernelGGL((kv8_attention_join_kernel<D, DT, 256>), rows, dim3(256), 0, stream, p, plan.rows);
        else hipLaunchKernelGGL((kv8_attention_join_kernel<D, DT, 512>), rows, dim3(512), 0, stream, p, plan.rows);
        e = hipGetLastError();
    }
    return e;
}

template <int D, Dtype DT>
hipError_t launch_typed(const Kv8AttentionParams &p, const Kv8Plan &plan, hipStream_t stream) {
    if constexpr (DT == Dtype::F32) {
        return plan.rows == 8 ? launch_rows<D, DT, 8>(p, plan, stream) : launch_rows<D, DT, 32>(p, plan, stream);
    } else {
        return plan.rows == 8 ? launch_rows<D, DT, 8>(p, plan, stream)
            : plan.rows == 16 ? launch_rows<D, DT, 16>(p, plan, stream)
                              : launch_rows<D, DT, 64>(p, plan, stream);
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

hipError_t launch_kv8_shared_attention(const Kv8AttentionParams &p, Dtype dtype, const Kv8SharedPlan &plan, hipStream_t stream) {
    if (dtype == Dtype::F32) return launch_shared_head<Dtype::F32>(p, plan, stream);
    if (dtype == Dtype::F16) return launch_shared_head<Dtype::F16>(p, plan, stream);
    return launch_shared_head<Dtype::BF16>(p, plan, stream);
}

}  // namespace fortai_hip
