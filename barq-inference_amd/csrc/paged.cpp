// C ABI of the paged KV cache (include/barq_rocm.h): the pool, a step's batch of
// sequences, append with norm and rotation, read, attention; norm_rope and the
// rotary frequencies for long contexts.
#include "../../include/barq_rocm.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <memory>
#include <vector>

#include "api_internal.hpp"
#include "launch.hpp"
#include "paged_plan.hpp"

using namespace barq_api;

namespace {

constexpr size_t INT_MOST = 0x7fffffff;
constexpr size_t GRID_MOST = (1u << 24) - 1;   // workgroups of 256: a launch has fewer than 2^32 threads

struct Pool {
    int device = 0, type = BARQ_TYPE_F16, log_page = 0;
    size_t n_pages = 0, page_size = 0, n_layers = 0, n_head_kv = 0, head_dim = 0;
    uint8_t *k = nullptr, *v = nullptr;
    bool f16() const { return type == BARQ_TYPE_F16; }
    size_t layer_bytes() const { return n_pages * n_head_kv * page_size * head_dim * (f16() ? 2 : 4); }
    ~Pool() {
        DeviceGuard g(device);
        (void)hipDeviceSynchronize();
        if (k) (void)hipFree(k);
        if (v) (void)hipFree(v);
    }
};

// A buffer of pinned host memory that a set() fills; the event is behind the kernel that reads it.
struct Stage {
    uint8_t* p = nullptr;
    size_t size = 0;
    hipEvent_t done = nullptr;
    bool used = false;
};

}  // namespace

struct barq_rocm_paged_cache {
    std::shared_ptr<Pool> pool;
};

struct barq_rocm_paged_batch {
    std::shared_ptr<Pool> pool;
    size_t n_head = 0, max_seqs = 0, max_tokens = 0, max_pages = 0, part_rows = 0;
    size_t window = 0, n_sink = 0;
    barq::PagedShape shape;
    // device, of a fixed size: graphs captured with this batch keep the addresses
    uint8_t* mem = nullptr;
    float* rows = nullptr;   // [max_tokens, n_head * head_dim], from the first call for Q8_K rows on
    size_t counts_at = 0, groups_at = 0, merges_at = 0, few_at = 0, many_at = 0, table_at = 0, stat_at = 0, part_at = 0;
    size_t items_most = 0, merges_most = 0;
    Stage stage[2];
    int next = 0;
    std::vector<uint32_t> stamp;   // pages that the latest set() writes, by its number
    uint32_t number = 0;
    barq::PagedPlan plan;          // of the latest set()
    barq::PagedCounts counts{};

    const barq::PagedCounts* dev_counts() const { return reinterpret_cast<const barq::PagedCounts*>(mem + counts_at); }
    ~barq_rocm_paged_batch() {
        DeviceGuard g(pool->device);
        (void)hipDeviceSynchronize();
        if (mem) (void)hipFree(mem);
        if (rows) (void)hipFree(rows);
        for (Stage& s : stage) {
            if (s.p) (void)hipHostFree(s.p);
            if (s.done) (void)hipEventDestroy(s.done);
        }
    }
};

namespace {

int check_rotary(const barq_rocm_rotary* r, size_t head_dim, const char* who) {
    if (!r || r->rot_dim == 0) return ok();
    if (r->rot_dim % 2 != 0 || r->rot_dim > head_dim)
        return fail(BARQ_E_DIM, "%s: rot_dim=%zu must be even and at most head_dim=%zu", who, r->rot_dim, head_dim);
    if (r->layout != BARQ_ROPE_INTERLEAVED && r->layout != BARQ_ROPE_SPLIT_HALF)
        return fail(BARQ_E_INVALID, "%s: layout must be BARQ_ROPE_INTERLEAVED or BARQ_ROPE_SPLIT_HALF", who);
    if (!r->inv_freq) return fail(BARQ_E_INVALID, "%s: null inv_freq", who);
    return ok();
}

barq::Rotary rotary_of(const barq_rocm_rotary* r, const float* inv_freq) {
    if (!r || r->rot_dim == 0) return {nullptr, 0, barq::ROPE_INTERLEAVED, 1.0f, 1.0f};
    return {inv_freq, (int)r->rot_dim, r->layout, r->freq_scale, r->magnitude};
}

int check_batch(barq_rocm_handle* h, const barq_rocm_paged_batch* b, size_t layer, const char* who) {
    BARQ_CHECK(check_handle(h));
    if (!b) return fail(BARQ_E_INVALID, "%s: null batch", who);
    if (h->device != b->pool->device) return fail(BARQ_E_INVALID, "%s: cache is on another device", who);
    if (layer >= b->pool->n_layers) return fail(BARQ_E_INVALID, "%s: layer %zu of %zu", who, layer, b->pool->n_layers);
    return ok();
}

// Whether the handle's stream is being captured: its replays then take the counts of later set() calls.
int capturing(barq_rocm_handle* h, bool& yes) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    BARQ_HIP(hipStreamIsCapturing(h->stream, &s));
    yes = s != hipStreamCaptureStatusNone;
    return ok();
}

// Copies of host buffers in the workspace.
struct Staged {
    barq_rocm_handle* h;
    Arena a;
    size_t add(const void* p, size_t bytes) { return p ? a.add(bytes) : 0; }
    template <class T>
    int in(const T*& p, size_t off, size_t bytes) {
        if (!p) return ok();
        T* d = at<T>(h, off);
        BARQ_HIP(hipMemcpyAsync(d, p, bytes, hipMemcpyHostToDevice, h->stream));
        p = d;
        return ok();
    }
};

barq::PagedAppend append_args(const barq_rocm_paged_batch* b, size_t layer, bool captured) {
    const Pool& p = *b->pool;
    barq::PagedAppend a{};
    a.k_pool = p.k + layer * p.layer_bytes();
    a.v_pool = p.v + layer * p.layer_bytes();
    a.groups = reinterpret_cast<const barq::PagedGroup*>(b->mem + b->groups_at);
    a.counts = b->dev_counts();
    a.n_tokens = captured ? -1 : b->counts.n_tokens;
    a.n_groups = captured ? -1 : b->counts.groups;
    a.n_kv = (int)p.n_head_kv;
    a.log_page = p.log_page;
    return a;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------------------
// rotary frequencies, norm_rope

int barq_rocm_rope_frequencies(int scaling, size_t rot_dim, double base, double factor, double trained, double fast,
                               double slow, float* inv_freq, float* magnitude) {
    const char* who = "rope_frequencies";
    if (!inv_freq || !magnitude) return fail(BARQ_E_INVALID, "%s: null output", who);
    if (rot_dim == 0 || rot_dim % 2 != 0) return fail(BARQ_E_DIM, "%s: rot_dim=%zu must be even", who, rot_dim);
    if (scaling < BARQ_ROPE_PLAIN || scaling > BARQ_ROPE_YARN)
        return fail(BARQ_E_UNSUPPORTED, "%s: scaling %d", who, scaling);
    if (!(base > 0) || !std::isfinite(base)) return fail(BARQ_E_INVALID, "%s: base %g must be positive", who, base);
    if (scaling != BARQ_ROPE_PLAIN && (!(factor >= 1) || !std::isfinite(factor)))
        return fail(BARQ_E_INVALID, "%s: factor %g must be at least 1", who, factor);
    if (scaling == BARQ_ROPE_NTK && rot_dim == 2) return fail(BARQ_E_DIM, "%s: rot_dim 2 has no second pair to stretch", who);
    if (scaling == BARQ_ROPE_YARN && (!(trained > 0) || !(slow >= 0) || !(fast > slow) || !std::isfinite(trained) || !std::isfinite(fast)))
        return fail(BARQ_E_INVALID, "%s: trained %g, fast %g and slow %g need trained > 0 and fast > slow >= 0", who, trained, fast, slow);
    const double n = (double)rot_dim;
    if (scaling == BARQ_ROPE_NTK) base *= std::pow(factor, n / (n - 2));
    for (size_t i = 0; i < rot_dim / 2; i++) {
        double f = std::pow(base, -2.0 * (double)i / n);
        if (scaling == BARQ_ROPE_LINEAR) f /= factor;
        if (scaling == BARQ_ROPE_YARN) {
            const double turns = trained * f / (2 * M_PI), keep = std::fmin(std::fmax((turns - slow) / (fast - slow), 0), 1);
            f = f * keep + f / factor * (1 - keep);
        }
        inv_freq[i] = (float)f;
    }
    *magnitude = scaling == BARQ_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1) : 1.0f;
    return ok();
}

int barq_rocm_norm_rope(barq_rocm_handle* h, const float* x, size_t seq_len, size_t n_heads, size_t head_dim,
                        size_t start_pos, const float* norm, float eps, const barq_rocm_rotary* rotary, float* out, int mem) {
    const char* who = "norm_rope";
    BARQ_CHECK(check_mem(mem));
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(BARQ_E_UNSUPPORTED, "%s: head_dim %zu (64, 128 or 256 supported)", who, head_dim);
    BARQ_CHECK(check_rotary(rotary, head_dim, who));
    if (seq_len == 0 || n_heads == 0) return ok();
    if (!x || !out) return fail(BARQ_E_INVALID, "%s: null buffer", who);
    if (seq_len > GRID_MOST || start_pos > INT_MOST - seq_len || n_heads > INT_MOST / head_dim || n_heads * head_dim > (SIZE_MAX / 16) / seq_len)
        return fail(BARQ_E_DIM, "%s: %zu rows from position %zu, %zu heads", who, seq_len, start_pos, n_heads);
    if (mem == BARQ_MEM_DEVICE && !(aligned(x, 16) && aligned(out, 16) && aligned(norm, 4) && (!rotary || aligned(rotary->inv_freq, 4))))
        return fail(BARQ_E_INVALID, "%s: x and out must be 16-byte aligned, norm and inv_freq 4-byte", who);
    BARQ_CHECK(check_handle(h));
    DeviceGuard g(h);
    const size_t bytes = seq_len * n_heads * head_dim * 4, fb = rotary ? rotary->rot_dim / 2 * 4 : 0;
    const float* freq = rotary && rotary->rot_dim ? rotary->inv_freq : nullptr;
    float* to = out;
    if (mem == BARQ_MEM_HOST) {
        Staged s{h, {}};
        const size_t ox = s.add(x, bytes), oo = s.add(out, bytes), on = s.add(norm, head_dim * 4), of = s.add(freq, fb);
        BARQ_CHECK(ensure_ws(h, s.a.used));
        BARQ_CHECK(s.in(x, ox, bytes));
        BARQ_CHECK(s.in(norm, on, head_dim * 4));
        BARQ_CHECK(s.in(freq, of, fb));
        to = at<float>(h, oo);
    }
    BARQ_CHECK(launched(barq::norm_rope_launch(x, to, seq_len, n_heads, head_dim, start_pos, norm, eps, rotary_of(rotary, freq),
                                               h->stream), who));
    if (mem == BARQ_MEM_HOST) {
        BARQ_HIP(hipMemcpyAsync(out, to, bytes, hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return ok();
}

// ---------------------------------------------------------------------------
// the pool

int barq_rocm_paged_cache_create(barq_rocm_handle* h, size_t n_pages, size_t page_size, size_t n_layers, size_t n_head_kv,
                                 size_t head_dim, int type, barq_rocm_paged_cache** out) {
    const char* who = "paged_cache_create";
    if (!out) return fail(BARQ_E_INVALID, "%s: null output pointer", who);
    *out = nullptr;
    if (type != BARQ_TYPE_F32 && type != BARQ_TYPE_F16)
        return fail(BARQ_E_UNSUPPORTED, "%s: type %d (BARQ_TYPE_F16 or BARQ_TYPE_F32)", who, type);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(BARQ_E_UNSUPPORTED, "%s: head_dim %zu (64, 128 or 256 supported)", who, head_dim);
    if (page_size < (size_t)barq::PAGE_BLOCK || page_size > barq::PAGE_MAX || (page_size & (page_size - 1)) != 0)
        return fail(BARQ_E_DIM, "%s: page_size %zu must be a power of two from %d to %zu", who, page_size, barq::PAGE_BLOCK, barq::PAGE_MAX);
    if (n_pages == 0 || n_layers == 0 || n_head_kv == 0)
        return fail(BARQ_E_DIM, "%s: n_pages, n_layers and n_head_kv must be positive", who);
    if (n_pages > INT_MOST / page_size || n_head_kv > 65535)
        return fail(BARQ_E_DIM, "%s: %zu pages of %zu positions (at most 2^31 - 1 in all), %zu kv heads", who, n_pages, page_size, n_head_kv);
    size_t bytes = n_pages;
    for (const size_t f : {page_size, n_layers, n_head_kv, head_dim, (size_t)8})
        if (__builtin_mul_overflow(bytes, f, &bytes)) return fail(BARQ_E_DIM, "%s: size overflow", who);
    BARQ_CHECK(check_handle(h));
    DeviceGuard g(h);
    std::unique_ptr<barq_rocm_paged_cache> c;
    try {
        c.reset(new barq_rocm_paged_cache());
        c->pool = std::make_shared<Pool>();
    } catch (const std::exception&) {
        return fail(BARQ_E_ALLOC, "%s: out of host memory", who);
    }
    Pool& p = *c->pool;
    p.device = h->device;
    p.type = type;
    p.n_pages = n_pages;
    p.page_size = page_size;
    p.n_layers = n_layers;
    p.n_head_kv = n_head_kv;
    p.head_dim = head_dim;
    while ((size_t)1 << p.log_page < page_size) p.log_page++;
    hipError_t e = hipMalloc(&p.k, n_layers * p.layer_bytes());
    if (e == hipSuccess) e = hipMalloc(&p.v, n_layers * p.layer_bytes());
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return fail(BARQ_E_ALLOC, "%s: %zu bytes: %s", who, 2 * n_layers * p.layer_bytes(), hipGetErrorString(e));
    }
    *out = c.release();
    return ok();
}

int barq_rocm_paged_cache_destroy(barq_rocm_paged_cache* c) {
    delete c;
    return ok();
}

// ---------------------------------------------------------------------------
// a step's sequences

int barq_rocm_paged_batch_create(barq_rocm_handle* h, barq_rocm_paged_cache* c, size_t n_head, size_t max_seqs,
                                 size_t max_tokens, size_t max_pages, size_t window, size_t n_sink,
                                 barq_rocm_paged_batch** out) {
    const char* who = "paged_batch_create";
    if (!out) return fail(BARQ_E_INVALID, "%s: null output pointer", who);
    *out = nullptr;
    if (!c) return fail(BARQ_E_INVALID, "%s: null cache", who);
    BARQ_CHECK(check_handle(h));
    const Pool& p = *c->pool;
    if (h->device != p.device) return fail(BARQ_E_INVALID, "%s: cache is on another device", who);
    if (n_head == 0 || n_head % p.n_head_kv != 0)
        return fail(BARQ_E_DIM, "%s: %zu query heads must be a multiple of the cache's %zu kv heads", who, n_head, p.n_head_kv);
    if (max_seqs == 0 || max_tokens == 0 || max_pages == 0)
        return fail(BARQ_E_DIM, "%s: max_seqs, max_tokens and max_pages must be positive", who);
    if (n_head > INT_MOST / p.head_dim || max_tokens > INT_MOST / n_head || max_seqs > INT_MOST / n_head ||
        max_seqs > INT_MOST / max_pages || window > INT_MOST || n_sink > INT_MOST ||
        max_tokens * n_head / 16 + 4 * max_seqs * p.n_head_kv > GRID_MOST)   // (tiles of rows; groups of new tokens, twice)
        return fail(BARQ_E_DIM, "%s: %zu sequences, %zu tokens, %zu pages, %zu heads, window %zu, %zu first tokens", who, max_seqs,
                    max_tokens, max_pages, n_head, window, n_sink);
    DeviceGuard g(h);
    std::unique_ptr<barq_rocm_paged_batch> b;
    try {
        b.reset(new barq_rocm_paged_batch());
        b->pool = c->pool;
        b->stamp.assign(p.n_pages, 0);
    } catch (const std::exception&) {
        if (b && !b->pool) b->pool = c->pool;
        return fail(BARQ_E_ALLOC, "%s: out of host memory", who);
    }
    const size_t G = n_head / p.n_head_kv;
    b->n_head = n_head;
    b->max_seqs = max_seqs;
    b->max_tokens = max_tokens;
    b->max_pages = max_pages;
    b->window = window;
    b->n_sink = window ? n_sink : 0;
    barq::PagedShape& sh = b->shape;
    sh.G = (int)G;
    sh.n_kv = (int)p.n_head_kv;
    sh.window = (int64_t)window;
    sh.n_sink = (int64_t)b->n_sink;
    barq::paged_shape_for(sh, p.f16(), p.head_dim);
    b->part_rows = sh.part_rows = barq::paged_part_rows(sh, max_tokens);
    b->items_most = barq::paged_max_tiles(max_seqs, max_tokens, G) + 2 * (size_t)(sh.few_target + sh.many_target) + 4;
    b->merges_most = barq::paged_max_tiles(max_seqs, max_tokens, G);
    Arena a;
    b->counts_at = a.add(sizeof(barq::PagedCounts));
    b->groups_at = a.add(barq::paged_max_groups(max_seqs, max_tokens) * sizeof(barq::PagedGroup));
    b->merges_at = a.add(b->merges_most * sizeof(barq::PagedMerge));
    b->few_at = a.add(b->items_most * sizeof(barq::PagedItem));
    b->many_at = a.add(b->items_most * sizeof(barq::PagedItem));
    b->table_at = a.add((max_seqs * max_pages + 4) * sizeof(int32_t));
    b->stat_at = a.add(p.n_head_kv * b->part_rows * sizeof(float2));
    b->part_at = a.add(p.n_head_kv * b->part_rows * p.head_dim * sizeof(float));
    hipError_t e = hipMalloc(&b->mem, a.used);
    // (no sequences yet)
    if (e == hipSuccess) e = hipMemset(b->mem + b->counts_at, 0, sizeof(barq::PagedCounts));
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);   // (before a set() on another stream)
    for (Stage& s : b->stage)
        if (e == hipSuccess) e = hipEventCreateWithFlags(&s.done, hipEventDisableTiming);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return fail(BARQ_E_ALLOC, "%s: %zu bytes: %s", who, a.used, hipGetErrorString(e));
    }
    *out = b.release();
    return ok();
}

int barq_rocm_paged_batch_destroy(barq_rocm_paged_batch* b) {
    delete b;
    return ok();
}

int barq_rocm_paged_batch_set(barq_rocm_handle* h, barq_rocm_paged_batch* b, size_t n_seqs, const int32_t* q_len,
                              const int32_t* kv_len, const int32_t* pages, size_t pages_stride) {
    const char* who = "paged_batch_set";
    BARQ_CHECK(check_batch(h, b, 0, who));
    const Pool& p = *b->pool;
    // (a number that wraps round would take an old set()'s pages for this one's)
    if (b->number == UINT32_MAX) {
        std::fill(b->stamp.begin(), b->stamp.end(), 0u);
        b->number = 0;
    }
    size_t tokens = 0, entries = 0;
    char msg[160];
    const barq::PagedFault fault = barq::paged_check({b->max_seqs, b->max_tokens, b->max_pages, p.n_pages, p.page_size}, n_seqs, q_len,
                                                     kv_len, pages, pages_stride, b->stamp.data(), ++b->number, tokens, entries, msg,
                                                     sizeof msg);
    if (fault != barq::PagedFault::none)
        return fail(fault == barq::PagedFault::dim ? BARQ_E_DIM : BARQ_E_INVALID, "%s: %s", who, msg);
    DeviceGuard g(h);
    bool captured = false;
    BARQ_CHECK(capturing(h, captured));
    if (captured) return fail(BARQ_E_UNSUPPORTED, "%s: the stream is being captured (set the batch before, and between replays)", who);
    barq::PagedPlan plan;
    barq::PagedCounts counts{};
    Stage& st = b->stage[b->next];
    barq::PagedPieces pieces{};
    size_t used = 0;
    try {
        std::vector<barq::PagedSeq> seqs(n_seqs);
        size_t at = 0;
        for (size_t s = 0; s < n_seqs; s++) {
            seqs[s] = {q_len[s], kv_len[s], (int64_t)at};
            at += ((size_t)kv_len[s] + p.page_size - 1) / p.page_size;
        }
        barq::paged_plan(b->shape, seqs, plan);
    } catch (const std::exception&) {
        return fail(BARQ_E_ALLOC, "%s: out of host memory", who);
    }
    if (plan.few.size() > b->items_most || plan.many.size() > b->items_most || plan.merges.size() > b->merges_most)
        return fail(BARQ_E_DIM, "%s: the plan does not fit the batch", who);   // (it does: paged_plan.hpp)
    counts.n_tokens = (int32_t)tokens;
    for (size_t s = 0; s < n_seqs; s++)
        if (q_len[s]) counts.groups += (kv_len[s] - 1) / barq::PAGE_BLOCK - (kv_len[s] - q_len[s]) / barq::PAGE_BLOCK + 1;
    counts.few = (int32_t)plan.n_few;
    counts.many = (int32_t)plan.many.size();
    counts.merges = (int32_t)plan.merges.size();
    const auto piece = [&](size_t to, size_t bytes) {
        if (!bytes) return (size_t)0;
        const size_t from = used;
        pieces.dst[pieces.n] = b->mem + to;
        pieces.from[pieces.n] = (uint32_t)from;
        pieces.bytes[pieces.n++] = (uint32_t)round_up(bytes, 16);
        used += round_up(bytes, 16);
        return from;
    };
    const size_t pc = piece(b->counts_at, sizeof counts), pt = piece(b->groups_at, (size_t)counts.groups * sizeof(barq::PagedGroup));
    const size_t pm = piece(b->merges_at, plan.merges.size() * sizeof(barq::PagedMerge));
    const size_t pf = piece(b->few_at, plan.few.size() * sizeof(barq::PagedItem));
    const size_t pn = piece(b->many_at, plan.many.size() * sizeof(barq::PagedItem));
    const size_t pp = piece(b->table_at, entries * sizeof(int32_t));
    if (used > UINT32_MAX) return fail(BARQ_E_DIM, "%s: %zu bytes of tables", who, used);
    if (st.used) BARQ_HIP(hipEventSynchronize(st.done));
    st.used = false;
    if (used > st.size) {
        if (st.p) (void)hipHostFree(st.p);
        st.p = nullptr;
        st.size = 0;
        const size_t want = round_up(used, 4096) * 2;
        void* m = nullptr;
        const hipError_t e = hipHostMalloc(&m, want, hipHostMallocDefault);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            return fail(BARQ_E_ALLOC, "%s: %zu bytes of host memory: %s", who, want, hipGetErrorString(e));
        }
        st.p = static_cast<uint8_t*>(m);
        st.size = want;
    }
    std::memcpy(st.p + pc, &counts, sizeof counts);
    auto* group = reinterpret_cast<barq::PagedGroup*>(st.p + pt);
    auto* table = reinterpret_cast<int32_t*>(st.p + pp);
    int32_t t0 = 0;
    for (size_t s = 0; s < n_seqs; s++) {
        const int32_t* ids = pages + s * pages_stride;
        group = barq::paged_groups(t0, q_len[s], kv_len[s], ids, p.log_page, group);
        t0 += q_len[s];
        const size_t n = ((size_t)kv_len[s] + p.page_size - 1) / p.page_size;
        if (n) std::memcpy(table, ids, n * sizeof(int32_t));
        table += n;
    }
    const auto put = [&](size_t to, const void* from, size_t bytes) {
        if (bytes) std::memcpy(st.p + to, from, bytes);
    };
    put(pm, plan.merges.data(), plan.merges.size() * sizeof(barq::PagedMerge));
    put(pf, plan.few.data(), plan.few.size() * sizeof(barq::PagedItem));
    put(pn, plan.many.data(), plan.many.size() * sizeof(barq::PagedItem));
    pieces.src = st.p;
    BARQ_CHECK(launched(barq::paged_upload_launch(pieces, h->stream), who));
    BARQ_HIP(hipEventRecord(st.done, h->stream));
    st.used = true;
    b->next ^= 1;
    b->plan = std::move(plan);
    b->counts = counts;
    return ok();
}

// ---------------------------------------------------------------------------
// append, read, attention

int barq_rocm_paged_append(barq_rocm_handle* h, barq_rocm_paged_batch* b, size_t layer, const float* q, float* q_out,
                           const float* k, const float* v, const float* q_norm, const float* k_norm, float eps,
                           const barq_rocm_rotary* rotary, int mem) {
    const char* who = "paged_append";
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_batch(h, b, layer, who));
    const Pool& p = *b->pool;
    BARQ_CHECK(check_rotary(rotary, p.head_dim, who));
    if ((q == nullptr) != (q_out == nullptr)) return fail(BARQ_E_INVALID, "%s: q and q_out go together", who);
    DeviceGuard g(h);
    bool captured = false;
    BARQ_CHECK(capturing(h, captured));
    const size_t t = (size_t)b->counts.n_tokens;
    if (t == 0 && !captured) return ok();
    if (!k || !v) return fail(BARQ_E_INVALID, "%s: null buffer", who);
    if (mem == BARQ_MEM_DEVICE &&
        !(aligned(q, 16) && aligned(q_out, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_norm, 4) && aligned(k_norm, 4) &&
          (!rotary || aligned(rotary->inv_freq, 4))))
        return fail(BARQ_E_INVALID, "%s: q, q_out, k and v must be 16-byte aligned, norms and inv_freq 4-byte", who);
    if (mem == BARQ_MEM_HOST && captured) return fail(BARQ_E_UNSUPPORTED, "%s: host buffers while the stream is being captured", who);
    const size_t nq = t * b->n_head * p.head_dim * 4, nk = t * p.n_head_kv * p.head_dim * 4, nw = p.head_dim * 4;
    const float* freq = rotary && rotary->rot_dim ? rotary->inv_freq : nullptr;
    float* to = q_out;
    if (mem == BARQ_MEM_HOST) {
        Staged s{h, {}};
        const size_t fb = freq ? rotary->rot_dim / 2 * 4 : 0;
        const size_t oq = s.add(q, nq), oo = s.add(q_out, nq), ok_ = s.add(k, nk), ov = s.add(v, nk), on = s.add(q_norm, nw),
                     om = s.add(k_norm, nw), of = s.add(freq, fb);
        BARQ_CHECK(ensure_ws(h, s.a.used));
        BARQ_CHECK(s.in(q, oq, nq));
        BARQ_CHECK(s.in(k, ok_, nk));
        BARQ_CHECK(s.in(v, ov, nk));
        BARQ_CHECK(s.in(q_norm, on, nw));
        BARQ_CHECK(s.in(k_norm, om, nw));
        BARQ_CHECK(s.in(freq, of, fb));
        if (q_out) to = at<float>(h, oo);
    }
    barq::PagedAppend a = append_args(b, layer, captured);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.q_out = to;
    a.n_q = q ? (int)b->n_head : 0;
    a.eps = eps;
    a.rotary = rotary_of(rotary, freq);
    BARQ_CHECK(launched(barq::paged_append_launch(a, p.f16(), p.head_dim, h->stream), who));
    if (mem == BARQ_MEM_HOST) {
        if (q_out) BARQ_HIP(hipMemcpyAsync(q_out, to, nq, hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return ok();
}

int barq_rocm_paged_read(barq_rocm_handle* h, const barq_rocm_paged_batch* b, size_t layer, void* k, void* v, int mem) {
    const char* who = "paged_read";
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_batch(h, b, layer, who));
    const Pool& p = *b->pool;
    DeviceGuard g(h);
    bool captured = false;
    BARQ_CHECK(capturing(h, captured));
    const size_t t = (size_t)b->counts.n_tokens, bytes = t * p.n_head_kv * p.head_dim * (p.f16() ? 2 : 4);
    if (t == 0 && !captured) return ok();
    if (!k && !v) return fail(BARQ_E_INVALID, "%s: null buffer", who);
    if (mem == BARQ_MEM_DEVICE && !(aligned(k, 4) && aligned(v, 4)))
        return fail(BARQ_E_INVALID, "%s: outputs must be 4-byte aligned", who);
    if (mem == BARQ_MEM_HOST && captured) return fail(BARQ_E_UNSUPPORTED, "%s: host buffers while the stream is being captured", who);
    void *dk = k, *dv = v;
    if (mem == BARQ_MEM_HOST) {
        Arena a;
        const size_t ok_ = a.add(bytes), ov = a.add(bytes);
        BARQ_CHECK(ensure_ws(h, a.used));
        dk = k ? at<uint8_t>(h, ok_) : nullptr;
        dv = v ? at<uint8_t>(h, ov) : nullptr;
    }
    BARQ_CHECK(launched(barq::paged_read_launch(append_args(b, layer, captured), p.f16(), p.head_dim, dk, dv, h->stream), who));
    if (mem == BARQ_MEM_HOST) {
        if (k) BARQ_HIP(hipMemcpyAsync(k, dk, bytes, hipMemcpyDeviceToHost, h->stream));
        if (v) BARQ_HIP(hipMemcpyAsync(v, dv, bytes, hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return ok();
}

int barq_rocm_paged_attention(barq_rocm_handle* h, barq_rocm_paged_batch* b, size_t layer, const float* q, int out_type,
                              void* out, int mem) {
    const char* who = "paged_attention";
    BARQ_CHECK(check_mem(mem));
    BARQ_CHECK(check_batch(h, b, layer, who));
    const Pool& p = *b->pool;
    if (out_type != BARQ_TYPE_F32 && out_type != BARQ_TYPE_Q8_K)
        return fail(BARQ_E_UNSUPPORTED, "%s: out_type %d (BARQ_TYPE_F32 or BARQ_TYPE_Q8_K)", who, out_type);
    const bool q8 = out_type == BARQ_TYPE_Q8_K;
    const size_t width = b->n_head * p.head_dim;
    if (q8 && width % 256 != 0) return fail(BARQ_E_DIM, "%s: n_head * head_dim = %zu is not a multiple of 256", who, width);
    DeviceGuard g(h);
    bool captured = false;
    BARQ_CHECK(capturing(h, captured));
    const size_t t = (size_t)b->counts.n_tokens, rows = t * width * 4, blocks = t * (width / 256) * 292;
    if (t == 0 && !captured) return ok();
    if (!q || !out) return fail(BARQ_E_INVALID, "%s: null buffer", who);
    if (mem == BARQ_MEM_DEVICE && !(aligned(q, 16) && aligned(out, 4)))
        return fail(BARQ_E_INVALID, "%s: q must be 16-byte aligned, the output 4-byte aligned", who);
    if (mem == BARQ_MEM_HOST && captured) return fail(BARQ_E_UNSUPPORTED, "%s: host buffers while the stream is being captured", who);
    Arena a;
    const size_t oo = mem == BARQ_MEM_HOST && !q8 ? a.add(rows) : 0;
    const size_t oq = mem == BARQ_MEM_HOST ? a.add(rows) : 0, ob = mem == BARQ_MEM_HOST && q8 ? a.add(blocks) : 0;
    BARQ_CHECK(ensure_ws(h, a.used));
    if (q8 && !b->rows) {   // f32 rows that are quantized afterwards, for any number of tokens (replays' among them)
        if (captured) return fail(BARQ_E_UNSUPPORTED, "%s: the first call for Q8_K rows allocates: make one before the capture", who);
        const hipError_t e = hipMalloc(&b->rows, b->max_tokens * width * 4);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            return fail(BARQ_E_ALLOC, "%s: %zu bytes: %s", who, b->max_tokens * width * 4, hipGetErrorString(e));
        }
    }
    barq::PagedAttn x{};
    x.q = q;
    if (mem == BARQ_MEM_HOST) {
        BARQ_HIP(hipMemcpyAsync(at<float>(h, oq), q, rows, hipMemcpyHostToDevice, h->stream));
        x.q = at<float>(h, oq);
    }
    x.out = q8 ? b->rows : mem == BARQ_MEM_HOST ? at<float>(h, oo) : static_cast<float*>(out);
    x.out_q8 = !q8 ? nullptr : mem == BARQ_MEM_HOST ? at<uint8_t>(h, ob) : static_cast<uint8_t*>(out);
    x.k = p.k + layer * p.layer_bytes();
    x.v = p.v + layer * p.layer_bytes();
    x.table = reinterpret_cast<const int32_t*>(b->mem + b->table_at);
    x.few = reinterpret_cast<const barq::PagedItem*>(b->mem + b->few_at);
    x.many = reinterpret_cast<const barq::PagedItem*>(b->mem + b->many_at);
    x.merges = reinterpret_cast<const barq::PagedMerge*>(b->mem + b->merges_at);
    x.counts = b->dev_counts();
    x.n_tokens = captured ? -1 : (int)t;
    x.n_few = (int)b->plan.n_few;
    x.once = b->plan.once;   // (a hint: a captured call keeps the one of its capture)
    x.n_many = (int)b->plan.many.size();
    x.n_merges = (int)b->plan.merges.size();
    x.merge_span = 128;
    if (!captured) {
        x.merge_span = 1;
        for (const barq::PagedMerge& m : b->plan.merges) {
            const int n = m.n_split > barq::PAGED_MERGE_WAVE ? m.rows : (m.rows + 3) / 4;
            x.merge_span = n > x.merge_span ? n : x.merge_span;
        }
    }
    x.n_head = (int)b->n_head;
    x.n_kv = (int)p.n_head_kv;
    x.G = b->shape.G;
    x.log_page = p.log_page;
    x.window = (int)std::min<size_t>(b->window, 0x7ffff000);   // (no position is beyond that)
    x.n_sink = (int)b->n_sink;
    x.scale = (float)(M_LOG2E / std::sqrt((double)p.head_dim));
    x.part = reinterpret_cast<float*>(b->mem + b->part_at);
    x.stat = reinterpret_cast<float2*>(b->mem + b->stat_at);
    x.part_rows = b->part_rows;
    BARQ_CHECK(launched(barq::paged_attention_launch(x, p.f16(), (int)p.head_dim, h->stream), who));
    if (mem == BARQ_MEM_HOST) {
        if (q8) BARQ_HIP(hipMemcpyAsync(out, x.out_q8, blocks, hipMemcpyDeviceToHost, h->stream));
        else BARQ_HIP(hipMemcpyAsync(out, x.out, rows, hipMemcpyDeviceToHost, h->stream));
        BARQ_HIP(hipStreamSynchronize(h->stream));
    }
    return ok();
}

}  // extern "C"
