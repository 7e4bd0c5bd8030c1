// How a step's attention over a paged cache is cut into workgroups (host).
//
// A sequence's rows (new tokens x query heads of a kv head) are cut into tiles of
// 16 (the kernel for few rows) or 128 (for many); a tile's rows see the key
// positions [0, first tokens) and [window's start, last row's position], counted
// in the kernel's steps.  Where there are fewer tiles than the card has room for,
// the tiles' steps are split, each tile by itself and as far as all workgroups
// find room at once, or (few rows of different sequences) into even shares through
// all of them; what the splits leave is merged.
//
// Which kernel: a tile of 16 rows reads the keys for itself alone, one of 128 is
// slow to begin and to end.  One sequence of 32 query heads on 8, 128 dims, 4000 positions
// before, f16, few / many us: 100 rows 18.1 / 24.7, 128 17.7 / 25.2, 192 22.0 / 29.3, 256 23.7 / 30.0; eight such
// sequences: 100 rows 59.4 / 72.1, 200 106 / 82.5; f32: 128 rows 35.9 / 35.4, 256 58.5 / 48.7.  Where the kernel for many
// runs anyway it takes middling sequences along: eight of 112 to 200 rows 82.5 us, the smaller ones in a launch of their own 107.
// 64 and 256 dims take the same numbers; they were not measured there.
#pragma once
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "paged.hpp"

namespace barq {

constexpr int64_t PAGED_FEW_ROWS = 16, PAGED_MANY_ROWS = 128;   // of a tile

struct PagedShape {
    int G = 1, n_kv = 1;          // query heads of a kv head, kv heads
    int64_t window = 0, n_sink = 0;
    int few_step = 32, many_step = 64;   // positions of a kernel's step
    // rows from which a sequence's tiles are the large ones: many_from, or alone_from if the smaller tiles of all sequences
    // below that take at most alone_tiles workgroups; beside_from where another sequence has that many
    int64_t many_from = 129, alone_from = 257, alone_tiles = 256, beside_from = 65;
    int64_t few_target = 512, many_target = 512;    // workgroups that the card holds at once
    int64_t few_least = 4, many_least = 4;          // steps that a split has at least
    int64_t few_start = 4;        // steps that an item's beginning and end take the time of (2 and 8 measured 1 to 2 % worse)
    int64_t step_bytes = 16384;   // of K and V in a step of few rows
    // bytes of K and V that few rows read from which they pass the caches by: 16 sequences' 256 / 192 / 160 / 128 / 96 MB
    // take 49.9 / 40.0 / 35.2 / 29.3 / 27.0 us so, 53.0 / 42.0 / 36.5 / 27.2 / 22.2 otherwise (the same pages again and again:
    // what a model's other layers leave of them in the caches was not measured).  Counted by lengths: a page that sequences share
    // counts for each, 16 / 32 / 64 sequences of 4000 positions on the same pages take 23.6 / 38.8 / 64.1 us so, 21.9 / 32.5 / 53.9 otherwise
    int64_t once_from = 160 << 20;
    size_t part_rows = 0;         // partial states there is room for, for each kv head
};

struct PagedSeq {
    int64_t q_len, kv_len, table;
};

struct PagedPlan {
    std::vector<PagedItem> few, many;
    std::vector<PagedMerge> merges;
    size_t n_few = 0;             // workgroups for few rows: items 0 .. n_few - 1, and what follows each of them
    bool once = false;            // whether few rows' keys and values are read as passing by
};

struct PagedLimits {
    size_t max_seqs, max_tokens, max_pages, n_pages, page_size;
};

enum class PagedFault { none, dim, invalid };

// What is wrong with a step's arrays (said in msg), none if nothing is; then tokens, and entries of the page table.
// stamp has one value a page, none of them `number`: the pages that take new tokens get it.
inline PagedFault paged_check(const PagedLimits& lim, size_t n_seqs, const int32_t* q_len, const int32_t* kv_len,
                              const int32_t* pages, size_t stride, uint32_t* stamp, uint32_t number, size_t& tokens,
                              size_t& entries, char* msg, size_t room) {
    constexpr int32_t most = 0x7ffff000;   // positions: a step past the last one stays an int
    tokens = entries = 0;
    if (n_seqs > lim.max_seqs) {
        snprintf(msg, room, "%zu sequences, the batch has room for %zu", n_seqs, lim.max_seqs);
        return PagedFault::dim;
    }
    if (n_seqs && (!q_len || !kv_len || !pages)) {
        snprintf(msg, room, "null array");
        return PagedFault::invalid;
    }
    for (size_t s = 0; s < n_seqs; s++) {
        if (q_len[s] < 0 || kv_len[s] < q_len[s] || kv_len[s] > most) {
            snprintf(msg, room, "sequence %zu: %d new tokens, kv_len %d (with them; at most 2^31 - 4096)", s, q_len[s], kv_len[s]);
            return PagedFault::dim;
        }
        const size_t n = ((size_t)kv_len[s] + lim.page_size - 1) / lim.page_size;
        if (n > lim.max_pages || n > stride) {
            snprintf(msg, room, "sequence %zu needs %zu pages: the batch has room for %zu, the table has %zu", s, n, lim.max_pages, stride);
            return PagedFault::dim;
        }
        tokens += (size_t)q_len[s];
        entries += n;
        const size_t written = ((size_t)kv_len[s] - (size_t)q_len[s]) / lim.page_size;
        for (size_t i = 0; i < n; i++) {
            const int32_t id = pages[s * stride + i];
            if (id < -1 || (id >= 0 && (size_t)id >= lim.n_pages)) {
                snprintf(msg, room, "sequence %zu: page %zu is %d, the cache has %zu (-1: none)", s, i, id, lim.n_pages);
                return PagedFault::invalid;
            }
            if (id >= 0 && q_len[s] && i >= written) {
                if (stamp[id] == number) {
                    snprintf(msg, room, "sequence %zu: page %d takes new tokens in two places", s, id);
                    return PagedFault::invalid;
                }
                stamp[id] = number;
            }
        }
    }
    if (tokens > lim.max_tokens) {
        snprintf(msg, room, "%zu new tokens, the batch has room for %zu", tokens, lim.max_tokens);
        return PagedFault::dim;
    }
    return PagedFault::none;
}

// The most groups of new tokens.
inline size_t paged_max_groups(size_t max_seqs, size_t max_tokens) { return std::min(max_tokens, max_tokens / PAGE_BLOCK + 2 * max_seqs); }

// A sequence's new tokens, the batch's t0 .. on, cut where a block ends.
inline PagedGroup* paged_groups(int32_t t0, int32_t q_len, int32_t kv_len, const int32_t* ids, int log_page, PagedGroup* g) {
    for (int32_t j = kv_len - q_len; j < kv_len;) {
        const int32_t n = std::min(PAGE_BLOCK - j % PAGE_BLOCK, kv_len - j), id = ids[j >> log_page];
        *g++ = {t0, n, id < 0 ? -1 : (id << log_page) + (j & ((1 << log_page) - 1)), j};
        t0 += n;
        j += n;
    }
    return g;
}

// The most items and merges that a plan of these limits has.
inline size_t paged_max_tiles(size_t max_seqs, size_t max_tokens, size_t G) { return (max_tokens * G + 15) / 16 + max_seqs; }

// The kernels' steps and numbers of workgroups for a type and head_dim.
inline void paged_shape_for(PagedShape& sh, bool f16, size_t hd) {
    sh.few_step = f16 ? 32 : 16;
    sh.many_step = f16 ? 64 : 32;
    if (!f16) sh.alone_from = sh.many_from;
    sh.step_bytes = 128 * (int64_t)hd;
    // by the kernels' registers: one, two, three workgroups a CU (f32 rows of 64 dims have room for four, not used)
    sh.few_target = hd == 256 ? 256 : hd == 128 ? 512 : 768;
    sh.many_target = hd == 256 ? 256 : 512;
}

// Partial states to have room for (of each kv head): 64 MiB of them with 128 dims at most.  (So many kv heads that a tile's states find no
// room are as many workgroups, and nothing is split.)
inline size_t paged_part_rows(const PagedShape& sh, size_t max_tokens) {
    const size_t splits = 2 * (size_t)std::max(sh.few_target, sh.many_target) / sh.n_kv + 2;
    return std::min(max_tokens * sh.G * splits, (size_t)131072 / sh.n_kv);
}

// Cuts tiles into shares of equal time for `slots` workgroups, one after another through the tiles, so that a workgroup may end
// one tile and begin the next; an item takes its steps' time and `start` besides.  cut: the workgroups' first items, n of
// them, then what they go on with; part is the tile's number.  false: no better than `worst`, the longest time without that.
// Where each tile is cut by itself up to half of the slots may stay empty: 33 / 40 / 48 sequences of 3000, 3000 and 1500
// positions (8 kv heads, 128 dims, 64 slots) 99 / 104 / 66 us, with shares 73 / 86 / 64.  Tiles that read the same keys are
// not cut so: side by side one reads them for the others too (eight sequences of 25 tokens 60 us, with shares 99).
inline bool paged_shares(const std::vector<PagedItem>& tiles, int64_t steps, int64_t slots, int64_t least, int64_t start, int64_t worst,
                         std::vector<PagedItem>& cut, size_t& n) {
    std::vector<PagedItem> row;   // the shares one behind the other
    std::vector<char> first;      // whether an item begins one
    int64_t share = std::max((steps + start * ((int64_t)tiles.size() + slots) + slots - 1) / slots, start + least);
    for (bool fits = false; !fits; share += std::max<int64_t>(share / 32, 1)) {
        if (share * 16 > worst * 15) return false;   // (a sixteenth at least, or it is not worth it)
        row.clear();
        first.clear();
        n = 0;
        int64_t left = 0;   // of the share
        for (size_t t = 0; t < tiles.size(); t++) {
            const int64_t end = tiles[t].v1;
            for (int64_t v = 0; v < end;) {
                first.push_back(left < start + least);
                if (first.back()) {
                    left = share;
                    n++;
                }
                int64_t take = std::min(end - v, left - start);
                if (take < end - v) {
                    take -= take % least;   // (the waves' steps alike)
                    if (end - v - take < least) take = end - v;
                }
                row.push_back(tiles[t]);
                row.back().v0 = (int32_t)v;
                row.back().v1 = (int32_t)(v + take);
                row.back().part = (int32_t)t;
                v += take;
                left -= take + start;
            }
        }
        fits = (int64_t)n <= slots;
    }
    cut.resize(row.size());
    size_t head = 0, rest = n, last = 0;
    for (size_t i = 0; i < row.size(); i++) {
        const size_t at = first[i] ? head++ : rest++;
        cut[at] = row[i];
        if (!first[i]) cut[last].next = (int32_t)at;
        last = at;
    }
    return true;
}

inline void paged_plan(const PagedShape& sh, const std::vector<PagedSeq>& seqs, PagedPlan& p) {
    p.few.clear();
    p.many.clear();
    p.merges.clear();
    p.n_few = 0;
    int64_t steps[2] = {0, 0}, q0 = 0, small = 0, longest = 0;
    bool apart = true;   // no two tiles of few rows are of one sequence (sequences may share pages)
    for (const PagedSeq& s : seqs) {
        longest = std::max(longest, s.q_len * sh.G);
        if (s.q_len * sh.G < sh.alone_from) small += (s.q_len * sh.G + PAGED_FEW_ROWS - 1) / PAGED_FEW_ROWS;
    }
    int64_t many_from = small * sh.n_kv <= sh.alone_tiles ? sh.alone_from : sh.many_from;
    if (longest >= many_from) many_from = sh.beside_from;
    for (const PagedSeq& s : seqs) {
        const int64_t rows = s.q_len * sh.G, past = s.kv_len - s.q_len;
        const bool many = rows >= many_from;
        const int64_t tile = many ? PAGED_MANY_ROWS : PAGED_FEW_ROWS, unit = many ? sh.many_step : sh.few_step;
        for (int64_t r = 0; r < rows; r += tile) {
            PagedItem it{};
            it.q0 = (int32_t)q0;
            it.past = (int32_t)past;
            it.kv_len = (int32_t)s.kv_len;
            it.table = (int32_t)s.table;
            it.row0 = (int32_t)r;
            it.rows = (int32_t)std::min(tile, rows - r);
            const int64_t first = past + r / sh.G, end = past + (r + it.rows - 1) / sh.G + 1;
            const int64_t low = sh.window ? std::max<int64_t>(first - sh.window + 1, 0) / unit : 0;
            it.a = (int32_t)std::min((std::min(sh.n_sink, end) + unit - 1) / unit, low);
            it.b = (int32_t)low;
            it.v1 = (int32_t)(it.a + (end + unit - 1) / unit - low);
            it.part = -1;
            it.next = -1;
            apart &= many || rows <= tile;
            steps[many] += it.v1;
            (many ? p.many : p.few).push_back(it);
        }
        q0 += s.q_len;
    }
    p.once = apart && steps[0] * sh.n_kv * sh.step_bytes >= sh.once_from;
    size_t part = 0;
    for (int kind = 0; kind < 2; kind++) {
        std::vector<PagedItem>& items = kind ? p.many : p.few;
        const int64_t target = std::max<int64_t>((kind ? sh.many_target : sh.few_target) / sh.n_kv, 1);
        const int64_t least = kind ? sh.many_least : sh.few_least;
        if (!items.empty() && (int64_t)items.size() < target) {
            // steps of a split: the fewest (at least `least`) with which the splits all find room at once
            int64_t each = std::max((steps[kind] + target - 1) / target, least);
            const auto splits = [&](int64_t e) {
                int64_t n = 0;
                for (const PagedItem& it : items) n += (it.v1 + e - 1) / e;
                return n;
            };
            for (int64_t n; (n = splits(each)) > target;) {
                const int64_t more = each * n / target;   // (about as many splits too many as steps too few)
                if (n == (int64_t)items.size()) break;
                each = std::max(each + 1, std::min(more, each + each / 8));
            }
            std::vector<PagedItem> cut;
            int64_t longest = 0;
            for (const PagedItem& it : items) {
                const int64_t n = (it.v1 + each - 1) / each;
                longest = std::max(longest, (it.v1 + n - 1) / n);
            }
            if (!kind && apart && paged_shares(items, steps[0], target, least, sh.few_start, longest + sh.few_start, cut, p.n_few)) {
                std::vector<int32_t> n(items.size(), 0);
                size_t rows = 0;
                for (const PagedItem& c : cut) n[c.part]++;
                for (size_t t = 0; t < items.size(); t++) rows += n[t] > 1 ? (size_t)n[t] * items[t].rows : 0;
                if (rows <= sh.part_rows) {
                    std::vector<int32_t> at(items.size(), -1);
                    for (size_t t = 0; t < items.size(); t++) {
                        if (n[t] < 2) continue;
                        const PagedItem& it = items[t];
                        p.merges.push_back({it.q0, it.row0, it.rows, (int32_t)part, n[t], {0, 0, 0}});
                        at[t] = (int32_t)part;
                        part += (size_t)n[t] * it.rows;
                    }
                    for (PagedItem& c : cut) {
                        int32_t& to = at[c.part];
                        c.part = to;
                        if (to >= 0) to += c.rows;
                    }
                    items.swap(cut);
                    continue;
                }
                cut.clear();
            }
            for (const PagedItem& it : items) {
                int64_t n = std::max<int64_t>((it.v1 + each - 1) / each, 1);
                n = std::min<int64_t>(n, (int64_t)((sh.part_rows - part) / (size_t)it.rows));
                if (n < 2) {
                    cut.push_back(it);
                    continue;
                }
                p.merges.push_back({it.q0, it.row0, it.rows, (int32_t)part, (int32_t)n, {0, 0, 0}});
                for (int64_t i = 0; i < n; i++) {
                    PagedItem c = it;
                    c.v0 = (int32_t)(it.v1 * i / n);
                    c.v1 = (int32_t)(it.v1 * (i + 1) / n);
                    c.part = (int32_t)part;
                    part += (size_t)it.rows;
                    cut.push_back(c);
                }
            }
            items.swap(cut);
        }
        // the longest first: the last workgroups to start are short ones
        std::stable_sort(items.begin(), items.end(), [](const PagedItem& x, const PagedItem& y) {
            return x.v1 - x.v0 > y.v1 - y.v0;
        });
        if (!kind) p.n_few = items.size();
    }
}

}  // namespace barq
