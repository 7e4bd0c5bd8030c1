// The paged KV cache: how K and V lie in a page, and what the host hands the
// kernels about a step's sequences.
//
// A pool holds n_pages pages of page_size positions (a power of two, 16 at
// least) for every layer; page p of a layer holds them for all kv heads.  A
// block is 16 positions of one kv head, 16 * HD elements in a row:
//   K  [HD / E][16 positions][E dims]      E = 16 / sizeof(element): 8 in f16, 4 in f32
//   V  [16 / E][HD dims][E positions]
// so that 16 bytes are what one lane of an MFMA operand wants of either: E dims
// of a position of K, E positions of a dim of V (already transposed for P V),
// and neighbouring lanes' pieces lie side by side.  A page's blocks of a kv head
// follow each other, its kv heads too.
//
// A finite element beyond +-65504 is kept as +-65504 in f16 (the others are
// rounded to the nearest, ties to even); NaN and the infinities are kept as NaN
// in either type.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace barq {

constexpr int PAGE_BLOCK = 16;            // positions of a block
constexpr int PAGED_MERGE_WAVE = 8;       // partial states of a row that one wave joins; more: four of them
constexpr size_t PAGE_MAX = 1u << 16;     // positions of a page

// One workgroup's share of the attention of a step: rows of one sequence (row r
// is its new token r / G and query head r % G of the kv head at hand) against
// some of the key steps they see.
struct PagedItem {
    int32_t q0;      // the sequence's first new token among the batch's
    int32_t past;    // that token's position
    int32_t kv_len;
    int32_t table;   // where the sequence's page ids begin
    int32_t row0, rows;
    int32_t a, b;    // key step v (of a kernel's unit of positions) is v below a, v - a + b from there on: the first
                     // tokens that stay visible, then the window
    int32_t v0, v1;  // this item's steps
    int32_t part;    // its first row among the partial states, -1: it writes the output itself
    int32_t next;    // the item that the same workgroup takes after this one, -1: none (few rows)
    int32_t pad[4];
};
static_assert(sizeof(PagedItem) == 64, "items are fetched as 64 bytes");

// Rows whose steps several items share: their partial states lie rows apart.
struct PagedMerge {
    int32_t q0, row0, rows, part, n_split, pad[3];
};
static_assert(sizeof(PagedMerge) == 32, "");

// What a replayed graph reads anew (a call outside a capture passes it along).
struct PagedCounts {
    int32_t n_tokens, few, many, merges;
    int32_t groups;
    int32_t pad[11];
};
static_assert(sizeof(PagedCounts) == 64, "");

// New tokens t0 .. t0 + n - 1 of a sequence whose positions pos .. pos + n - 1 lie in one block, in the pool's rows
// row .. row + n - 1 (row: page * page_size + slot; -1: none).
struct PagedGroup {
    int32_t t0, n, row, pos;
};
static_assert(sizeof(PagedGroup) == 16, "");

}  // namespace barq
