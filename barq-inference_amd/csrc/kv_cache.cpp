// C ABI of what a KV cache offers beyond the reference's (include/barq_rocm.h):
// reading its rows whatever it holds them as, and dropping positions.
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

int barq_rocm_kv_cache_evict(barq_rocm_handle* h, const barq_rocm_kv_cache* src, barq_rocm_kv_cache* dst, size_t layer,
                             const float* mass_in, float* mass_out, size_t mass_stride, size_t keep, size_t recent,
                             int32_t* kept, int mem) {
    const char* who = "kv_cache_evict";
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_handle(h));
    if (!src || !dst) return fail(BARQ_E_INVALID, "%s: null cache", who);
    if (layer >= src->n_layers || layer >= dst->n_layers)
        return fail(BARQ_E_INVALID, "%s: layer %zu of %zu and %zu", who, layer, src->n_layers, dst->n_layers);
    if (src->type != dst->type || src->n_head_kv != dst->n_head_kv || src->head_dim != dst->head_dim)
        return fail(BARQ_E_DIM, "%s: the caches' types, kv heads or head dims differ", who);
    if (recent > keep) return fail(BARQ_E_DIM, "%s: recent %zu above keep %zu", who, recent, keep);
    const size_t n = src->len[layer], m = keep < n ? keep : n, heads = src->n_head_kv, hd = src->head_dim;
    if (m > dst->max_size)
        return fail(BARQ_E_INVALID, "%s: %zu positions, the destination has room for %zu", who, m, dst->max_size);
    if (n && !mass_in) return fail(BARQ_E_INVALID, "%s: null mass", who);
    if (mass_stride < n) return fail(BARQ_E_DIM, "%s: mass_stride %zu, layer %zu holds %zu positions", who, mass_stride, layer, n);
    if (h->device != src->device || h->device != dst->device)
        return fail(BARQ_E_INVALID, "%s: cache is on another device", who);
    if (mem == BARQ_MEM_DEVICE && !(aligned(mass_in, 4) && aligned(mass_out, 4) && aligned(kept, 4)))
        return fail(BARQ_E_INVALID, "%s: buffers must be 4-byte aligned", who);
    // thread counts and head offsets of the kernels
    if (heads > 65535 || 2 * (double)heads * (double)m * (double)hd > 256.0 * 2147483647.0)
        return fail(BARQ_E_DIM, "%s: %zu kv heads x %zu positions x %zu dims", who, heads, m, hd);
    const auto done = [&]() {
        dst->len[layer] = m;
        if (layer == 0) dst->size = m;
        return ok();
    };
    if (n == 0) return done();
    DeviceGuard g(h);
    const bool q4 = src->type == BARQ_TYPE_Q4_0, move = m > 0 && !(src == dst && m == n), stage = move && src == dst;
    Arena a;
    const size_t oid = a.add(heads * m * sizeof(int32_t));
    const size_t omass = mem == BARQ_MEM_HOST ? a.add(heads * n * sizeof(float)) : 0;
    const size_t code = q4 ? barq::q4_code_bytes(m, hd) : m * hd * sizeof(float), scale = q4 ? barq::q4_scale_bytes(m, hd) : 0;
    const size_t ostage = stage ? a.add(2 * heads * (code + scale)) : 0;
    BARQ_CHECK(ensure_ws(h, a.used));
    int32_t* id = kept && mem == BARQ_MEM_DEVICE ? kept : at<int32_t>(h, oid);
    const float* mi = mass_in;
    float* mo = mass_out;
    size_t stride = mass_stride;
    const size_t row = n * sizeof(float);
    if (mem == BARQ_MEM_HOST) {
        float* w = at<float>(h, omass);
        BARQ_HIP(hipMemcpy2DAsync(w, row, mass_in, mass_stride * sizeof(float), row, heads, hipMemcpyHostToDevice, h->stream));
        mi = w;
        mo = mass_out ? w : nullptr;
        stride = n;
    }
    BARQ_CHECK(launched(barq::evict_select_launch(mi, mo, stride, heads, n, m, recent, id, h->stream), who));
    if (move) {
        uint8_t* st = at<uint8_t>(h, ostage);
        barq::CopyPlanes back{};
        if (q4) {
            const barq::Q4View from = src->view(layer), to = dst->view(layer);
            barq::Q4View mid = to;
            if (stage) {
                mid.code_head = code;
                mid.scale_head = scale;
                mid.kc = st;
                mid.vc = mid.kc + heads * code;
                mid.ks = mid.vc + heads * code;
                mid.vs = mid.ks + heads * scale;
            }
            BARQ_CHECK(launched(barq::gather_q4_launch(from, mid, heads, hd, m, id, h->stream), who));
            back = {4, {mid.kc, mid.vc, mid.ks, mid.vs}, {to.kc, to.vc, to.ks, to.vs}, {code, code, scale, scale},
                    {to.code_head, to.code_head, to.scale_head, to.scale_head}, {code, code, scale, scale}};
        } else {
            const size_t so = layer * src->layer_stride(), dof = layer * dst->layer_stride();
            float* k = stage ? reinterpret_cast<float*>(st) : dst->k + dof;
            float* v = stage ? k + heads * m * hd : dst->v + dof;
            BARQ_CHECK(launched(barq::gather_rows_launch(src->k + so, src->v + so, src->head_stride(), k, v,
                                                         stage ? m * hd : dst->head_stride(), heads, hd, m, id, h->stream),
                                who));
            const size_t pitch = dst->head_stride() * sizeof(float);
            back = {2, {reinterpret_cast<uint8_t*>(k), reinterpret_cast<uint8_t*>(v)},
                    {reinterpret_cast<uint8_t*>(dst->k + dof), reinterpret_cast<uint8_t*>(dst->v + dof)},
                    {code, code}, {pitch, pitch}, {code, code}};
        }
        if (stage) BARQ_CHECK(launched(barq::copy_planes_launch(back, heads, h->stream), who));
    }
    if (mem == BARQ_MEM_HOST) {
        if (mass_out)
            BARQ_HIP(hipMemcpy2DAsync(mass_out, mass_stride * sizeof(float), mo, row, row, heads, hipMemcpyDeviceToHost, h->stream));
        if (kept && m) BARQ_HIP(hipMemcpyAsync(kept, id, heads * m * sizeof(int32_t), hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return done();
}

}  // extern "C"
