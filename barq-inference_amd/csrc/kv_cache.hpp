// The device KV cache behind barq_rocm_kv_cache (kv_cache.cpp, attention.cpp).
#pragma once
#include "../../include/barq_rocm.h"

#include <vector>

#include "kv_q4.hpp"

// BARQ_TYPE_F32: K and V each [n_layers][n_head_kv][max_size][head_dim] f32.
// BARQ_TYPE_Q4_0: kv_q4.hpp's codes in k and v, its scales in ks and vs, each
// [n_layers][n_head_kv][tiles of max_size].  Per-layer lengths live on the
// host (the reference's per-layer vectors grow independently; size() follows
// layer 0).
struct barq_rocm_kv_cache {
    int device = 0;
    int type = BARQ_TYPE_F32;
    size_t max_size = 0, n_layers = 0, n_head_kv = 0, head_dim = 0;
    float* k = nullptr;   // f32 rows (null in a 4-bit cache)
    float* v = nullptr;
    uint8_t* q4 = nullptr;   // one allocation: K codes, V codes, K scales, V scales
    std::vector<size_t> len;
    size_t size = 0;

    size_t head_stride() const { return max_size * head_dim; }
    size_t layer_stride() const { return n_head_kv * head_stride(); }
    size_t code_bytes() const { return n_layers * n_head_kv * barq::q4_code_bytes(max_size, head_dim); }
    size_t scale_bytes() const { return n_layers * n_head_kv * barq::q4_scale_bytes(max_size, head_dim); }
    barq::Q4View view(size_t layer) const {
        barq::Q4View w;
        w.code_head = barq::q4_code_bytes(max_size, head_dim);
        w.scale_head = barq::q4_scale_bytes(max_size, head_dim);
        w.kc = q4 + layer * n_head_kv * w.code_head;
        w.vc = w.kc + code_bytes();
        w.ks = q4 + 2 * code_bytes() + layer * n_head_kv * w.scale_head;
        w.vs = w.ks + scale_bytes();
        return w;
    }
};
