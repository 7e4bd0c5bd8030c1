// Attention over a 4-bit KV cache on the host: which kernel a call takes and
// how its rows and positions are cut into workgroups.
#pragma once
#include <stddef.h>

namespace barq {

constexpr int Q4P_NW = 4;               // waves of a workgroup of attn_q4_prompt_kernel
constexpr int Q4P_ROWS = 16 * Q4P_NW;   // its query rows

// Rows of a kv head from which it is used (64 and 128 dims).  us, attn_q4_kernel
// / this one, with the merge: 32/8 heads of 128, 16 / 24 / 32 rows (64 / 96 / 128 of a
// kv head) after 1000 10.9 / 13.5, 13.6 / 14.0, 17.0 / 15.0, after 8000 23 / 23,
// 26 / 29, 31 / 31, from position 0 7.8 / 6.5 each; of 64, 16 / 24 rows after 1000
// 8.8 / 10.5, 9.6 / 10.8.
constexpr int Q4P_MIN_ROWS = 128;

struct Q4Plan {
    bool prompt;     // attn_q4_prompt_kernel
    int G, groups;   // query heads that share a kv head (1 when they do not divide), and how many such groups
    int tiles;       // workgroups' row tiles
    int n_split, chunk;   // splits of the positions, positions of one
};

inline Q4Plan q4_plan(size_t n_head, size_t n_head_kv, size_t hd, size_t q_len, size_t kv_len, size_t cus) {
    constexpr size_t STEP = 32, TURN = 128;
    Q4Plan p;
    const bool even = n_head % n_head_kv == 0;
    p.G = even ? (int)(n_head / n_head_kv) : 1;
    p.groups = even ? (int)n_head_kv : (int)n_head;
    const size_t rows = q_len * p.G;
    p.prompt = hd <= 128 && rows >= Q4P_MIN_ROWS;
    const size_t per = p.prompt ? (size_t)Q4P_ROWS : 16, unit = p.prompt ? 4 * STEP : TURN;
    p.tiles = (int)((rows + per - 1) / per);
    // About two workgroups a CU, and no splits from one and a half on.  us with
    // targets of 1 / 1.5 / 2 / 3 a CU: 32/8 heads of 128, one row after 65535 28.4 / 30.0
    // / 25.6 / 27.5, 10 after 10000 20.3 / 21.2 / 20.1 / 21.6, 64 after 4000 33.4 /
    // 35.4 / 31.2 / 31.0, 512 after 1536 91 / 71 / 71 / 66, 1000 after 1500 (504
    // workgroups unsplit) 121 / 121 / 142 / 142; 200 after 800 of 64 23.7 / 19.8 / 19.7 / 21.6
    const size_t wg = (size_t)p.groups * p.tiles;
    size_t ns = 2 * wg >= 3 * cus ? 1 : (2 * cus + wg - 1) / wg;
    const size_t most = (kv_len + unit - 1) / unit;
    if (ns > most) ns = most;
    if (ns > 1024) ns = 1024;   // the merge's limit
    // At most 2^21 positions a split (byte offsets in 32 bits: 2^28 of 256 dims), so
    // that no cache below 2^31 positions takes more than the merge's limit.
    const size_t least = (kv_len + ((size_t)1 << 21) - 1) >> 21;
    if (ns < least) ns = least;
    size_t ch = (kv_len + ns - 1) / ns;
    ch = (ch + unit - 1) / unit * unit;
    p.chunk = (int)ch;
    p.n_split = (int)((kv_len + ch - 1) / ch);
    return p;
}

// Whether the call's launches, the merge's among them, stay below 2^32 threads (a
// larger grid is cut without an error).
inline bool q4_fits(const Q4Plan& p, size_t n_head, size_t hd, size_t q_len) {
    const size_t most = ((size_t)1 << 32) - 1;
    const size_t merge = ((n_head * hd + 255) / 256 * q_len + 3) / 4;   // workgroups
    return (size_t)p.n_split * p.tiles * p.groups <= most / (64 * Q4P_NW) && (p.n_split == 1 || merge <= most / 256);
}

// Where the split that begins at start ends, for a row tile that sees `visible`
// positions (below start where it sees none of the split).  Without start + chunk,
// which may pass 2^31 in the last split.
constexpr int q4_range_end(int start, int chunk, int visible) { return visible - start < chunk ? visible : start + chunk; }

// What a wave of attn_q4_kernel fetches while it works on the step at `at` (of
// n positions, a step every `turn`): the next one, or behind the last the end
// of the range's whole tiles.  There the scalar offset is the descriptor's limit
// itself, and every address is out of bounds and reads as zero (the bounds
// check subtracts the scalar offset from the limit; it need not go below zero).
constexpr int q4_ahead(int at, int turn, int n) { return at + turn < n ? at + turn : (n + 7) / 8 * 8; }

}  // namespace barq
