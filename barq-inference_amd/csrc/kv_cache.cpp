// C ABI of what a KV cache offers beyond the reference's (include/barq_rocm.h):
// reading its rows whatever it holds them as.
#include "../../include/barq_rocm.h"

#include <hip/hip_runtime.h>

#include "api_internal.hpp"
#include "kv_cache.hpp"
#include "launch.hpp"

using namespace barq_api;

extern "C" {

int barq_rocm_kv_cache_read(barq_rocm_handle* h, const barq_rocm_kv_cache* c, size_t layer, size_t first, size_t n,
                            float* k, float* v, int mem) {
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_handle(h));
    if (!c) return fail(BARQ_E_INVALID, "kv_cache_read: null cache");
    if (layer >= c->n_layers) return fail(BARQ_E_INVALID, "kv_cache_read: layer %zu of %zu", layer, c->n_layers);
    if (n > c->len[layer] || first > c->len[layer] - n)
        return fail(BARQ_E_DIM, "kv_cache_read: positions %zu .. +%zu, layer %zu holds %zu", first, n, layer, c->len[layer]);
    if (n == 0) return ok();
    if (!k && !v) return fail(BARQ_E_INVALID, "kv_cache_read: null buffer");
    if (h->device != c->device) return fail(BARQ_E_INVALID, "kv_cache_read: cache is on another device");
    if (mem == BARQ_MEM_DEVICE && !(aligned(k, 4) && aligned(v, 4)))
        return fail(BARQ_E_INVALID, "kv_cache_read: outputs must be 4-byte aligned");
    DeviceGuard g(h);
    const size_t hd = c->head_dim, row = n * hd * sizeof(float), bytes = c->n_head_kv * row;
    if (c->type == BARQ_TYPE_F32) {
        const size_t off = layer * c->layer_stride() + first * hd, pitch = c->head_stride() * sizeof(float);
        const hipMemcpyKind kind = mem == BARQ_MEM_DEVICE ? hipMemcpyDeviceToDevice : hipMemcpyDeviceToHost;
        if (k) BARQ_HIP(hipMemcpy2DAsync(k, row, c->k + off, pitch, row, c->n_head_kv, kind, h->stream));
        if (v) BARQ_HIP(hipMemcpy2DAsync(v, row, c->v + off, pitch, row, c->n_head_kv, kind, h->stream));
    } else {
        float *dk = k, *dv = v;
        if (mem == BARQ_MEM_HOST) {
            Arena a;
            const size_t ok_ = a.add(bytes), ov = a.add(bytes);
            BARQ_CHECK(ensure_ws(h, a.used));
            dk = k ? at<float>(h, ok_) : nullptr;
            dv = v ? at<float>(h, ov) : nullptr;
        }
        BARQ_CHECK(launched(barq::q4_read_launch(c->view(layer), c->n_head_kv, hd, first, n, dk, dv, h->stream),
                            "kv_cache_read"));
        if (mem == BARQ_MEM_HOST) {
            if (k) BARQ_HIP(hipMemcpyAsync(k, dk, bytes, hipMemcpyDeviceToHost, h->stream));
            if (v) BARQ_HIP(hipMemcpyAsync(v, dv, bytes, hipMemcpyDeviceToHost, h->stream));
        }
    }
    if (mem == BARQ_MEM_HOST) BARQ_HIP(hipStreamSynchronize(h->stream));
    return ok();
}

}  // extern "C"
