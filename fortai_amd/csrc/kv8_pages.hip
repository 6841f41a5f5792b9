// Page bookkeeping of the 8-bit cache, on the host: which pages a sequence's
// tokens lie in, shared between sequences that forked, copied when one of them
// writes.  No GPU is touched here; what has to be moved is handed back as pairs
// for fortai_hip_kv8_copy_pages.  (include/fortai_hip_backend.h,
// fortai_hip_kv8_pages_*.)
//
// The lowest free page is given out first, so that a pool that is used lightly
// stays at its lower end and compaction has little to move.
#include "../../include/fortai_hip_backend.h"

#include <cstdint>
#include <functional>
#include <new>
#include <queue>
#include <vector>

struct fortai_hip_kv8_pages {
    int pages = 0, page_tokens = 0, pitch = 0;
    std::vector<int32_t> users;  // sequences that hold a page
    std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free_pages;
    std::vector<std::vector<int32_t>> tables;
    std::vector<int64_t> lengths;

    bool has(int sequence) const { return sequence >= 0 && static_cast<size_t>(sequence) < tables.size(); }
    int64_t pages_of(int64_t tokens) const { return (tokens + page_tokens - 1) / page_tokens; }
    int32_t take() {
        const int32_t p = free_pages.top();
        free_pages.pop();
        users[p] = 1;
        return p;
    }
    void give(int32_t p) {
        if (--users[p] == 0) free_pages.push(p);
    }
};

extern "C" {

int fortai_hip_kv8_pages_create(int pages, int page_tokens, int sequences, int table_pitch, fortai_hip_kv8_pages **out) {
    if (!out) return FORTAI_HIP_INVALID;
    *out = nullptr;
    if (pages < 1 || (page_tokens != 16 && page_tokens != 32 && page_tokens != 64) || sequences < 1 || table_pitch < 1 ||
        table_pitch > (1 << 24))
        return FORTAI_HIP_INVALID;
    fortai_hip_kv8_pages *p = nullptr;
    try {
        p = new fortai_hip_kv8_pages;
        p->pages = pages;
        p->page_tokens = page_tokens;
        p->pitch = table_pitch;
        p->users.assign(pages, 0);
        std::vector<int32_t> all(pages);
        for (int i = 0; i < pages; ++i) all[i] = i;
        // ascending order is a heap already; giving a page back never allocates (the capacity stays)
        p->free_pages = decltype(p->free_pages)(std::greater<int32_t>(), std::move(all));
        p->tables.resize(sequences);
        p->lengths.assign(sequences, 0);
    } catch (...) {
        delete p;
        return FORTAI_HIP_RUNTIME_ERROR;
    }
    *out = p;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_pages_destroy(fortai_hip_kv8_pages *p) {
    delete p;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_pages_extend(fortai_hip_kv8_pages *p, int sequence, int tokens, int32_t *from, int32_t *to, int *copies) {
    if (!p || !p->has(sequence) || tokens < 0 || !from || !to || !copies) return FORTAI_HIP_INVALID;
    *copies = 0;
    if (tokens == 0) return FORTAI_HIP_OK;
    std::vector<int32_t> &table = p->tables[sequence];
    const int64_t length = p->lengths[sequence], need = p->pages_of(length + tokens);
    const bool inside = length % p->page_tokens != 0;  // the next token goes into a page that holds tokens already
    const bool shared = inside && p->users[table.back()] > 1;
    const int64_t fresh = need - static_cast<int64_t>(table.size()) + (shared ? 1 : 0);
    if (need > p->pitch || fresh > static_cast<int64_t>(p->free_pages.size())) return FORTAI_HIP_INVALID;
    try {
        table.reserve(static_cast<size_t>(need));
    } catch (...) {
        return FORTAI_HIP_RUNTIME_ERROR;
    }
    if (shared) {
        const int32_t own = p->take();
        *from = table.back();
        *to = own;
        *copies = 1;
        p->give(table.back());
        table.back() = own;
    }
    while (static_cast<int64_t>(table.size()) < need) table.push_back(p->take());
    p->lengths[sequence] = length + tokens;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_pages_fork(fortai_hip_kv8_pages *p, int sequence, int fork, int64_t length) {
    if (!p || !p->has(sequence) || !p->has(fork) || sequence == fork || length < 0 || length > p->lengths[sequence] ||
        p->lengths[fork] != 0)
        return FORTAI_HIP_INVALID;
    const size_t count = static_cast<size_t>(p->pages_of(length));
    try {
        p->tables[fork].assign(p->tables[sequence].begin(), p->tables[sequence].begin() + count);
    } catch (...) {
        p->tables[fork].clear();
        return FORTAI_HIP_RUNTIME_ERROR;
    }
    for (int32_t id : p->tables[fork]) ++p->users[id];
    p->lengths[fork] = length;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_pages_truncate(fortai_hip_kv8_pages *p, int sequence, int64_t length) {
    if (!p || !p->has(sequence) || length < 0 || length > p->lengths[sequence]) return FORTAI_HIP_INVALID;
    std::vector<int32_t> &table = p->tables[sequence];
    const size_t keep = static_cast<size_t>(p->pages_of(length));
    while (table.size() > keep) {
        p->give(table.back());
        table.pop_back();
    }
    p->lengths[sequence] = length;
    return FORTAI_HIP_OK;
}

int fortai_hip_kv8_pages_compact(fortai_hip_kv8_pages *p, int32_t *from, int32_t *to, int capacity, int *copies) {
    if (!p || !copies || capacity < 0 || (capacity > 0 && (!from || !to))) return FORTAI_HIP_INVALID;
    *copies = 0;
    const int live = p->pages - static_cast<int>(p->free_pages.size());
    std::vector<int32_t> moved, rest;
    try {
        moved.assign(p->pages, -1);
        rest.reserve(p->pages);
    } catch (...) {
        return FORTAI_HIP_RUNTIME_ERROR;
    }
    // live pages from the upper end on into the lowest holes, until all lie below `live`
    int hole = 0, n = 0;
    for (int page = p->pages - 1; page >= live && n < capacity; --page) {
        if (p->users[page] == 0) continue;
        while (p->users[hole] != 0 || moved[hole] == -2) ++hole;
        from[n] = page;
        to[n] = hole;
        moved[page] = hole;
        moved[hole] = -2;  // taken by this move
        ++n;
    }
    for (int k = 0; k < n; ++k) {
        p->users[to[k]] = p->users[from[k]];
        p->users[from[k]] = 0;
    }
    if (n > 0) {
        for (auto &table : p->tables)
            for (int32_t &id : table)
                if (moved[id] >= 0) id = moved[id];
        for (int page = 0; page < p->pages; ++page)
            if (p->users[page] == 0) rest.push_back(page);
        p->free_pages = decltype(p->free_pages)(std::greater<int32_t>(), std::move(rest));
    }
    *copies = n;
    return FORTAI_HIP_OK;
}

int64_t fortai_hip_kv8_pages_length(const fortai_hip_kv8_pages *p, int sequence) {
    return p && p->has(sequence) ? p->lengths[sequence] : -1;
}

int fortai_hip_kv8_pages_free_count(const fortai_hip_kv8_pages *p) {
    return p ? static_cast<int>(p->free_pages.size()) : -1;
}

int fortai_hip_kv8_pages_tables(const fortai_hip_kv8_pages *p, const int *sequences, int count, int32_t *tables, int table_pitch) {
    if (!p || count < 0 || table_pitch < 1 || (count > 0 && (!sequences || !tables))) return FORTAI_HIP_INVALID;
    for (int i = 0; i < count; ++i)
        if (!p->has(sequences[i]) || p->tables[sequences[i]].size() > static_cast<size_t>(table_pitch))
            return FORTAI_HIP_INVALID;
    for (int i = 0; i < count; ++i) {
        const std::vector<int32_t> &table = p->tables[sequences[i]];
        int32_t *row = tables + static_cast<size_t>(i) * table_pitch;
        for (int k = 0; k < table_pitch; ++k) row[k] = static_cast<size_t>(k) < table.size() ? table[k] : -1;
    }
    return FORTAI_HIP_OK;
}

// The tokens of `count` sequences in a row are compared with those of a group's first one;
// a sequence joins while that leaves more tokens that need not be read again.
int fortai_hip_kv8_pages_groups(const fortai_hip_kv8_pages *p, const int *sequences, int count, int32_t *starts, int32_t *shared,
    int32_t *group_of, int *groups) {
    if (!p || !groups || count < 0 || !starts || (count > 0 && (!sequences || !shared || !group_of))) return FORTAI_HIP_INVALID;
    *groups = 0;
    for (int i = 0; i < count; ++i)
        if (!p->has(sequences[i])) return FORTAI_HIP_INVALID;
    constexpr int64_t kLeast = 64;  // tokens: what attention shares is whole tiles of 64
    int n = 0, first = 0;
    while (first < count) {
        const std::vector<int32_t> &table = p->tables[sequences[first]];
        int64_t common = p->lengths[sequences[first]];
        int end = first + 1;
        while (end < count) {
            const std::vector<int32_t> &other = p->tables[sequences[end]];
            size_t same = 0;
            while (same < table.size() && same < other.size() && table[same] == other[same]) ++same;
            int64_t tokens = static_cast<int64_t>(same) * p->page_tokens;
            if (tokens > p->lengths[sequences[end]]) tokens = p->lengths[sequences[end]];
            if (tokens > common) tokens = common;
            const int64_t members = end - first;
            if (tokens < kLeast || (members > 1 && tokens * members < common * (members - 1))) break;
            common = tokens;
            ++end;
        }
        const bool alone = end == first + 1;
        // sequences that share nothing lie together in groups of no shared tokens
        if (!alone || n == 0 || shared[n - 1] != 0) {
            starts[n] = first;
            shared[n] = alone ? 0 : static_cast<int32_t>(common);
            ++n;
        }
        for (int i = first; i < end; ++i) group_of[i] = n - 1;
        first = end;
    }
    starts[n] = count;
    *groups = n;
    return FORTAI_HIP_OK;
}

}  // extern "C"
