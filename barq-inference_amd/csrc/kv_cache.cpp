// C ABI of what a KV cache offers beyond the reference's (include/barq_rocm.h):
// reading its rows whatever it holds them as, dropping positions, and
// the attention that gathers what the dropping goes by.
#include "../../include/barq_rocm.h"

#include <hip/hip_runtime.h>

#include "api_internal.hpp"
#include "kv_cache.hpp"
#include "kv_evict_plan.hpp"
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
    if (c->n_head_kv > 65535) return fail(BARQ_E_DIM, "kv_cache_read: %zu kv heads (at most 65535)", c->n_head_kv);
    DeviceGuard g(h);
    const size_t hd = c->head_dim, row = n * hd * sizeof(float), bytes = c->n_head_kv * row;
    if (c->type == BARQ_TYPE_F32) {
        const size_t off = layer * c->layer_stride() + first * hd, pitch = c->head_stride() * sizeof(float);
        if (mem == BARQ_MEM_DEVICE) {
            barq::CopyPlanes p{};
            for (int i = 0; i < 2; i++)
                if (float* to = i ? v : k) {
                    p.src[p.n] = reinterpret_cast<const uint8_t*>((i ? c->v : c->k) + off);
                    p.dst[p.n] = reinterpret_cast<uint8_t*>(to);
                    p.src_head[p.n] = pitch;
                    p.dst_head[p.n] = p.bytes[p.n] = row;
                    p.n++;
                }
            BARQ_CHECK(launched(barq::copy_planes_launch(p, c->n_head_kv, h->stream), "kv_cache_read"));
            return ok();
        }
        if (k) BARQ_HIP(hipMemcpy2DAsync(k, row, c->k + off, pitch, row, c->n_head_kv, hipMemcpyDeviceToHost, h->stream));
        if (v) BARQ_HIP(hipMemcpy2DAsync(v, row, c->v + off, pitch, row, c->n_head_kv, hipMemcpyDeviceToHost, h->stream));
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
    // positions (their count rounds up to 4096), heads and threads of the kernels
    if (n > 0x7ffff000u) return fail(BARQ_E_DIM, "%s: %zu positions (at most 2^31 - 4096)", who, n);
    const bool q4 = src->type == BARQ_TYPE_Q4_0, move = m > 0 && !(src == dst && m == n), stage = move && src == dst;
    if (heads > 65535 || (move && barq::evict_heads(q4, heads, m, hd) == 0))
        return fail(BARQ_E_DIM, "%s: %zu kv heads x %zu positions x %zu dims", who, heads, m, hd);
    const auto done = [&]() {
        dst->len[layer] = m;
        if (layer == 0) dst->size = m;
        return ok();
    };
    if (n == 0) return done();
    DeviceGuard g(h);
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

// Scores of one launch at most (half of the 256 MB last-level cache, from which
// they are read again): a longer prompt's rows are taken in chunks.
static constexpr size_t MASS_SCORES = (size_t)128 << 20;

int barq_rocm_attention_mass(barq_rocm_handle* h, const float* q, const barq_rocm_kv_cache* c, size_t layer, size_t n_head,
                             size_t n_head_kv, size_t head_dim, size_t q_len, size_t kv_len, size_t start_pos, int out_type,
                             void* out, const float* mass_in, float* mass_out, size_t mass_stride, int mem) {
    const char* who = "attention_mass";
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_handle(h));
    if (!c) return fail(BARQ_E_INVALID, "%s: null cache", who);
    if (out_type != BARQ_TYPE_F32 && out_type != BARQ_TYPE_Q8_K)
        return fail(BARQ_E_UNSUPPORTED, "%s: out_type %d (BARQ_TYPE_F32 or BARQ_TYPE_Q8_K)", who, out_type);
    if (q_len == 0 || n_head == 0)
        return fail(BARQ_E_DIM, "%s: no query rows or heads", who);
    if (!q || !out || !mass_out) return fail(BARQ_E_INVALID, "%s: null buffer", who);
    if (layer >= c->n_layers) return fail(BARQ_E_INVALID, "%s: layer %zu of %zu", who, layer, c->n_layers);
    if (n_head_kv != c->n_head_kv || head_dim != c->head_dim)
        return fail(BARQ_E_DIM, "%s: n_head_kv %zu / head_dim %zu, cache has %zu / %zu", who, n_head_kv, head_dim,
                    c->n_head_kv, c->head_dim);
    if (!barq::attention_supported(head_dim))
        return fail(BARQ_E_UNSUPPORTED, "%s: head_dim %zu (64, 128 or 256 supported)", who, head_dim);
    const bool q8 = out_type == BARQ_TYPE_Q8_K, q4 = c->type == BARQ_TYPE_Q4_0, host = mem == BARQ_MEM_HOST;
    if (n_head > 65535 || q_len > 65535 || start_pos > 0x7fffffff - q_len)
        return fail(BARQ_E_DIM, "%s: n_head %zu and q_len %zu must be at most 65535, start_pos %zu + q_len below 2^31", who,
                    n_head, q_len, start_pos);
    if (q8 && (n_head * head_dim) % 256 != 0)
        return fail(BARQ_E_DIM, "%s: n_head * head_dim = %zu is not a multiple of 256", who, n_head * head_dim);
    if (kv_len == 0 || kv_len > c->len[layer])
        return fail(BARQ_E_DIM, "%s: kv_len %zu, layer %zu holds %zu positions", who, kv_len, layer, c->len[layer]);
    if (kv_len > 0x7ffff000u) return fail(BARQ_E_DIM, "%s: kv_len %zu (at most 2^31 - 4096)", who, kv_len);
    if (mass_stride < kv_len) return fail(BARQ_E_DIM, "%s: mass_stride %zu below kv_len %zu", who, mass_stride, kv_len);
    if (h->device != c->device) return fail(BARQ_E_INVALID, "%s: cache is on another device", who);
    if (!host && (!aligned(q, 16) || !aligned(out, 4) || !aligned(mass_in, 4) || !aligned(mass_out, 4)))
        return fail(BARQ_E_INVALID, "%s: q must be 16-byte aligned, the other buffers 4-byte aligned", who);
    DeviceGuard g(h);
    const size_t stride = round_up(kv_len, 32), per_row = n_head * stride * sizeof(float);
    size_t rows = MASS_SCORES / per_row;
    rows = rows < 1 ? 1 : rows > q_len ? q_len : rows;
    const auto splits = [&](size_t n) {
        return (size_t)(q4 ? barq::attention_q4_scores_splits(n_head, n_head_kv, head_dim, n, kv_len)
                           : barq::attention_scores_splits(n_head, n_head_kv, n, kv_len));
    };
    const size_t last = q_len % rows;   // the last chunk's rows, if fewer
    const auto prompt = [&](size_t n) { return !q4 && barq::attn_prompt_scores_path(n_head, n_head_kv, head_dim, n, kv_len); };
    const auto states = [&](size_t n) {
        return prompt(n) ? barq::attn_prompt_scores_workspace(n_head, n_head_kv, head_dim, n, kv_len)
                         : splits(n) * n_head * n * (head_dim + 2) * sizeof(float);
    };
    size_t part = states(rows);
    if (last && states(last) > part) part = states(last);
    const size_t nq = n_head * q_len * head_dim, out_row = q8 ? n_head * head_dim / 256 * 292 : n_head * head_dim * 4;
    Arena a;
    const size_t os = a.add(rows * per_row), op = a.add(part), ost = a.add(n_head * rows * sizeof(float2));
    size_t sums = barq::attention_mass_sums(n_head, n_head_kv, rows, stride);
    if (last && barq::attention_mass_sums(n_head, n_head_kv, last, stride) > sums)   // (shorter runs may be more)
        sums = barq::attention_mass_sums(n_head, n_head_kv, last, stride);
    const size_t osum = a.add(sums);
    const size_t oq = host ? a.add(nq * 4) : 0, oo = host ? a.add(q_len * out_row) : 0;
    const size_t om = host ? a.add(n_head_kv * kv_len * sizeof(float)) : 0;
    BARQ_CHECK(ensure_ws(h, a.used));
    const size_t mrow = kv_len * sizeof(float);
    const float* mi = mass_in;
    float* mo = mass_out;
    size_t ms = mass_stride;
    uint8_t* ob = static_cast<uint8_t*>(out);
    if (host) {
        BARQ_HIP(hipMemcpyAsync(at<float>(h, oq), q, nq * 4, hipMemcpyHostToDevice, h->stream));
        q = at<float>(h, oq);
        mo = at<float>(h, om);
        if (mass_in) {
            BARQ_HIP(hipMemcpy2DAsync(mo, mrow, mass_in, mass_stride * sizeof(float), mrow, n_head_kv, hipMemcpyHostToDevice,
                                      h->stream));
            mi = mo;
        }
        ms = kv_len;
        ob = at<uint8_t>(h, oo);
    }
    for (size_t i = 0; i < q_len; i += rows) {
        const size_t n = rows < q_len - i ? rows : q_len - i;
        barq::AttnArgs args{};
        args.q = q + i * head_dim;
        args.k = c->k;   // (null in a 4-bit cache)
        args.v = c->v;
        args.layer_off = layer * c->layer_stride();
        args.head_stride = c->head_stride();
        args.n_head = n_head;
        args.n_head_kv = n_head_kv;
        args.head_dim = head_dim;
        args.q_len = n;
        args.kv_len = kv_len;
        args.start_pos = start_pos + i;
        args.part = at<float>(h, op);
        args.out = q8 ? nullptr : reinterpret_cast<float*>(ob + i * out_row);
        const barq::AttnScores sc{at<float>(h, os), stride, q_len};
        uint8_t* out_q8 = q8 ? ob + i * out_row : nullptr;
        float2* stat = at<float2>(h, ost);
        const bool merged = prompt(n), few = !merged && barq::attention_mass_few(n_head, n_head_kv, n);
        const int ns = merged ? 0 : (int)splits(n);
        if (merged) {
            args.out_q8 = out_q8;
            BARQ_CHECK(launched(barq::attn_prompt_scores_launch(args, sc, stat, h->stream), who));
        } else {
            BARQ_CHECK(launched(q4 ? barq::attention_q4_scores_launch(args, sc, c->view(layer), h->stream)
                                   : barq::attention_scores_launch(args, sc, h->stream), who));
            if (!few) BARQ_CHECK(launched(barq::attention_combine_launch(args, ns, out_q8, stat, h->stream), who));
        }
        barq::MassArgs m{};
        m.scores = sc.scores;
        m.score_stride = stride;
        m.part = args.part;
        m.ns = ns;
        m.head_dim = (int)head_dim;
        m.n_head = (int)n_head;
        m.n_head_kv = (int)n_head_kv;
        m.q_len = (int)n;
        m.kv_len = (int)kv_len;
        m.start_pos = (long long)(start_pos + i);
        m.stat = stat;
        m.sums = at<float>(h, osum);
        m.mass_in = i ? mo : mi;
        m.mass_out = mo;
        m.mass_stride = ms;
        BARQ_CHECK(launched(few ? barq::attention_mass_few_launch(m, args, out_q8, h->stream)
                                : barq::attention_mass_launch(m, h->stream), who));
    }
    if (host) {
        BARQ_HIP(hipMemcpyAsync(out, ob, q_len * out_row, hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipMemcpy2DAsync(mass_out, mass_stride * sizeof(float), mo, mrow, mrow, n_head_kv, hipMemcpyDeviceToHost,
                                  h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return ok();
}

}  // extern "C"
