// Eviction on the host: how many kv heads' rows one launch moves.
#pragma once
#include <stddef.h>

namespace barq {

// Threads per kv head that move m rows of hd dims: f32 rows (K's and V's),
// 16 bytes each where a row is whole ones, and 4-bit rows (kv_evict.hip has the
// three kinds).
inline double evict_threads(bool q4, double m, size_t hd) {
    if (!q4) return 2.0 * m * (double)(hd % 4 == 0 ? hd / 4 : hd);
    const double tiles = (double)(((size_t)m + 7) / 8), nb = (double)(hd / 32);
    return 16.0 * tiles + m * nb + 2.0 * tiles * nb;
}

// kv heads of a launch, whose threads must be fewer than 2^32 (a larger grid is
// cut without an error): all of them in any ordinary call, 0 if one alone has too many.
inline size_t evict_heads(bool q4, size_t n_kv, size_t m, size_t hd) {
    const double most = 4294967296.0 - 1024.0;   // (each kind's last workgroup may be short)
    const double heads = most / evict_threads(q4, (double)m, hd);
    return heads < (double)n_kv ? (size_t)heads : n_kv;
}

}  // namespace barq
