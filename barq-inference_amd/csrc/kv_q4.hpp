// The KV cache held in 4 bits: Q4_0 blocks (32 dims share one f16 scale d,
// element = (code - 8) * d, code 0 .. 15) laid out for the attention kernels.
//
// Positions are grouped in tiles of 8.  Per layer and kv head, with HD dims
// and NB = HD / 32 blocks a row:
//   K codes   [position][4][NB] dwords: dword (kq, b) holds dims 32 b + 8 kq
//             .. + 7 of the position, dim e of them in bits 4 (e / 2) + 16 (e %
//             2): the 8 contraction slots that lane group kq of a 16x16x32
//             MFMA gives block b, so a lane loads its part of a row in one piece
//   V codes   [tile][16][HD / 16] dwords: dword (i, c) holds dim 16 c + i of
//             the tile's 8 positions, position e in bits 4 (e / 2) + 16 (e % 2),
//             so V is already transposed for P V
//             (a dword masked by 0x000F000F << 4 j holds codes 2 j and 2 j + 1
//             as a packed pair)
//   scales    [tile][NB][8] f16, K's and V's alike: a lane's 8 positions of a
//             block are 16 bytes
// A position takes HD / 2 + 2 NB bytes of K and as many of V: 144 bytes with
// 128 dims against 1024 in f32.
//
// Scale and codes of a block: t = its first element of the largest |x|, d =
// t / -8 rounded to f16 and kept within +-8188 (so that every value (code - 8)
// * d is within f16's range, which attention relies on; |x| beyond 65504
// saturates), code = the nearest one under d, the larger one on a border.  A
// block with a NaN or an infinity gets the scale NaN and reads as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace barq {

constexpr int KV_TILE = 8;             // positions of a tile
constexpr float Q4_D_MAX = 8188.0f;    // 8 * 8188 = 65504

// One layer of a 4-bit cache (or of a staging area laid out alike).
struct Q4View {
    uint8_t* kc;       // codes
    uint8_t* vc;
    uint8_t* ks;       // scales
    uint8_t* vs;
    size_t code_head;  // bytes between kv heads
    size_t scale_head;
};

// bit of code e of a dword's eight
__host__ __device__ constexpr int q4_bit(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

inline size_t q4_tiles(size_t positions) { return (positions + KV_TILE - 1) / KV_TILE; }
// bytes of one kv head's codes / scales (K's, and V's again)
inline size_t q4_code_bytes(size_t positions, size_t hd) { return q4_tiles(positions) * KV_TILE * (hd / 2); }
inline size_t q4_scale_bytes(size_t positions, size_t hd) { return q4_tiles(positions) * KV_TILE * (hd / 32) * 2; }
inline bool q4_head_dim(size_t hd) { return hd == 64 || hd == 128 || hd == 256; }

}  // namespace barq
