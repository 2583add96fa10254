// Paged KV cache: the fl_pages_* entry points, and the launches of the kernels in
// pages_kernels.h.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <new>

#include "host_api.h"
#include "pages_kernels.h"

using namespace fl;

namespace {

// Pinned host memory that a copy to the device reads: written again only when that
// copy is done.
struct Stage {
    char *host = nullptr;
    size_t cap = 0;
    hipEvent_t done = nullptr;
    bool used = false;
};
constexpr int kStages = 4;
constexpr int kPageMaxQueries = 1 << 20;
constexpr int kMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads along x: a grid's threads are counted in 32 bits
constexpr int kPageMaxGroup = 32;  // query heads per kv head: the rows of the largest form of every cache

struct DevBuf {
    char *p = nullptr;
    size_t cap = 0;
};

}  // namespace

struct fl_pages {
    fl_ctx *ctx = nullptr;  // nullptr: bookkeeping alone
    int device = 0;
    hipStream_t stream = nullptr;
    fl_pages_config cfg{};
    PagePool pool{};
    PageTable t;
    // the last attention call's plan: built again when its arguments or the tables change
    PagePlan plan;
    std::vector<int32_t> plan_seqs, plan_seen;
    int plan_heads = 0;
    uint64_t plan_version = 0;
    size_t plan_order = 0, plan_pages = 0, plan_units = 0, plan_joins = 0, plan_join_of = 0, plan_arrived = 0;  // offsets
    DevBuf d_plan, d_runs, d_read, d_copies, ws;
    Stage stages[kStages];
    int stage = 0;
};

namespace {

int fail(fl_pages *p, int code, const char *fmt, ...) __attribute__((format(printf, 3, 4)));
int fail(fl_pages *p, int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return fl_host_fail(p ? p->ctx : nullptr, code, buf);
}

#define PGCHK(p, expr)                                                                                     \
    do {                                                                                                   \
        const hipError_t e_ = (expr);                                                                      \
        if (e_ != hipSuccess) return fail((p), FL_E_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));   \
    } while (0)
#define PGTRY(expr)           \
    do {                      \
        const int rc_ = (expr); \
        if (rc_) return rc_;  \
    } while (0)

// The pool's device for the length of a call, the caller's behind it.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const fl_pages *p) {
        int now = 0;
        if (p->ctx && hipGetDevice(&now) == hipSuccess && now != p->device && hipSetDevice(p->device) == hipSuccess)
            before = now;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

size_t elem_bytes(int fmt) { return fmt == FL_KV_F32 ? 4 : fmt == FL_KV_F16 ? 2 : 1; }

int check_config(const fl_pages_config *c) {
    if (!c) return fail(nullptr, FL_E_INVALID, "null config");
    if (c->kv_format != FL_KV_F32 && c->kv_format != FL_KV_F16 && c->kv_format != FL_KV_Q8)
        return fail(nullptr, FL_E_UNSUPPORTED, "paged cache of format %d", c->kv_format);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(nullptr, FL_E_UNSUPPORTED, "head_dim %d (64 or 128)", c->head_dim);
    if (c->page_size < 32 || c->page_size > 4096 || c->page_size % 32)
        return fail(nullptr, FL_E_INVALID, "page size %d (a multiple of 32 up to 4096)", c->page_size);
    if (c->num_layers < 1 || c->num_kv_heads < 1 || (long long)c->num_layers * c->num_kv_heads > 65535)
        return fail(nullptr, FL_E_INVALID, "%d layers of %d kv heads", c->num_layers, c->num_kv_heads);
    if (c->num_pages < 1 || c->num_pages > kMaxGrid || (long long)c->num_pages * c->page_size > 0x7FFFFFFFll)
        return fail(nullptr, FL_E_INVALID, "%d pages of %d tokens", c->num_pages, c->page_size);
    if (c->max_seqs < 1 || c->max_seq_len < 1 || c->max_seq_len > (1 << 24) ||
        (long long)c->max_seqs * ((c->max_seq_len + c->page_size - 1) / c->page_size) > (1ll << 28))
        return fail(nullptr, FL_E_INVALID, "%d sequences of up to %d tokens", c->max_seqs, c->max_seq_len);
    return 0;
}

// No call may be recorded into a graph: its replays would not move the bookkeeping.
int check_stream(fl_pages *p) {
    if (!p->ctx) return fail(p, FL_E_STATE, "the pages have no device memory");
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    PGCHK(p, hipStreamIsCapturing(p->stream, &st));
    if (st != hipStreamCaptureStatusNone) return fail(p, FL_E_STATE, "a paged cache's calls cannot be captured into a graph");
    return 0;
}

// What was in a grown buffer is lost; work that reads it is done when hipFree returns.
int ensure(fl_pages *p, DevBuf &b, size_t bytes) {
    if (b.cap >= bytes) return 0;
    const size_t cap = std::max(bytes, std::max<size_t>(4096, 2 * b.cap));
    char *n = nullptr;
    hipError_t e = hipMalloc((void **)&n, cap);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return fail(p, FL_E_OOM, "hipMalloc(%zu) failed: %s", cap, hipGetErrorString(e));
    }
    if (b.p) {
        (void)hipStreamSynchronize(p->stream);
        (void)hipFree(b.p);
    }
    b.p = n;
    b.cap = cap;
    return 0;
}

// Room for `bytes` in the stage of the next send() but `ahead`.
int stage_room(fl_pages *p, int ahead, size_t bytes) {
    Stage &s = p->stages[(p->stage + ahead) % kStages];
    if (s.used) PGCHK(p, hipEventSynchronize(s.done));
    s.used = false;
    if (s.cap < bytes) {
        const size_t cap = std::max<size_t>(4096, 2 * bytes);
        char *n = nullptr;
        if (hipHostMalloc((void **)&n, cap, hipHostMallocDefault) != hipSuccess) {
            (void)hipGetLastError();
            return fail(p, FL_E_OOM, "hipHostMalloc(%zu) failed", cap);
        }
        if (s.host) (void)hipHostFree(s.host);
        s.host = n;
        s.cap = cap;
    }
    if (!s.done) PGCHK(p, hipEventCreateWithFlags(&s.done, hipEventDisableTiming));
    return 0;
}

// Pinned memory for `bytes` that go to the device with send().
int stage_for(fl_pages *p, size_t bytes, char **host) {
    PGTRY(stage_room(p, 0, bytes));
    *host = p->stages[p->stage].host;
    return 0;
}

int send(fl_pages *p, void *dev, size_t bytes) {
    Stage &s = p->stages[p->stage];
    PGCHK(p, hipMemcpyAsync(dev, s.host, bytes, hipMemcpyHostToDevice, p->stream));
    PGCHK(p, hipEventRecord(s.done, p->stream));
    s.used = true;
    p->stage = (p->stage + 1) % kStages;
    return 0;
}

int upload(fl_pages *p, DevBuf &b, const void *data, size_t bytes) {
    char *h;
    PGTRY(ensure(p, b, bytes));
    PGTRY(stage_for(p, bytes, &h));
    memcpy(h, data, bytes);
    return send(p, b.p, bytes);
}

// Room for a list of up to n copies, before the bookkeeping that makes it.
int copies_room(fl_pages *p, int ahead, long long n) {
    return n > kInlineCopies ? stage_room(p, ahead, (size_t)n * sizeof(PageCopy)) : 0;
}

int run_copies(fl_pages *p) {
    const auto &c = p->t.copies;
    if (c.empty()) return 0;
    PageCopies list;
    list.list = nullptr;
    if (c.size() <= kInlineCopies) {
        memcpy(list.some, c.data(), c.size() * sizeof(PageCopy));
    } else {
        PGTRY(upload(p, p->d_copies, c.data(), c.size() * sizeof(PageCopy)));
        list.list = (const PageCopy *)p->d_copies.p;
    }
    const int D = p->cfg.head_dim, unit = 32 * D * (int)elem_bytes(p->cfg.kv_format);
    const int sunit = p->cfg.kv_format == FL_KV_Q8 ? 2 * D : 0;
    hipLaunchKernelGGL(k_pages_copy, dim3((unsigned)c.size(), p->pool.layers * p->pool.nkv), dim3(256), 0, p->stream,
                       p->pool, list, unit, sunit);
    PGCHK(p, hipGetLastError());
    return 0;
}

// Runs `op` on the bookkeeping, with its error as the context's.
template <typename F>
int on_table(fl_pages *p, F op) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    try {
        const int rc = op(p->t);
        return rc ? fail(p, rc, "%s", p->t.error.c_str()) : 0;
    } catch (const std::bad_alloc &) {
        return fail(p, FL_E_OOM, "out of host memory");
    } catch (...) {
        return fail(p, FL_E_INVALID, "unexpected host error");
    }
}

template <typename F>
int with_form(int fmt, int D, F f) {
    if (D == 64) return fmt == FL_KV_F32 ? f.template operator()<FL_KV_F32, 64>() :
                        fmt == FL_KV_F16 ? f.template operator()<FL_KV_F16, 64>() : f.template operator()<FL_KV_Q8, 64>();
    return fmt == FL_KV_F32 ? f.template operator()<FL_KV_F32, 128>() :
           fmt == FL_KV_F16 ? f.template operator()<FL_KV_F16, 128>() : f.template operator()<FL_KV_Q8, 128>();
}

struct LaunchAttn {
    hipStream_t st;
    const PageAttnArgs &a;
    int items;
    bool wide;
    template <int FMT, int D>
    int operator()() const { return a.arrived ? launch<FMT, D, true>() : launch<FMT, D, false>(); }
    template <int FMT, int D, bool HERE>
    int launch() const {
        const dim3 grid((unsigned)(items * a.pool.nkv));
        if (!wide) {
            hipLaunchKernelGGL((k_pages_attn<FMT, D, 1, HERE>), grid, dim3(256), 0, st, a);
        } else if constexpr (FMT == FL_KV_F16) {
            // two steps of K and V, or one and the queries, or the waves' results
            constexpr size_t row = (D + 4) * 4, kv = 8 * 32 * D * 2;
            constexpr size_t lds = std::max({2 * kv, kv + 128 * row, 8 * 32 * row});
            hipLaunchKernelGGL((k_pages_attn_wide<D, HERE>), grid, dim3(512), lds, st, a);
        } else {
            hipLaunchKernelGGL((k_pages_attn<FMT, D, 2, HERE>), grid, dim3(256), 0, st, a);
        }
        return (int)hipGetLastError();
    }
};

struct LaunchWrite {
    hipStream_t st;
    const PageWriteArgs &a;
    const PageRuns &runs;
    int n, layers;
    template <int FMT, int D>
    int operator()() const {
        hipLaunchKernelGGL((k_pages_write<FMT, D>), dim3(n, a.pool.nkv, layers), dim3(256), 0, st, a, runs);
        return (int)hipGetLastError();
    }
};

struct LaunchRead {
    hipStream_t st;
    const PageReadArgs &a;
    const PageRuns &runs;
    int n;
    template <int FMT, int D>
    int operator()() const {
        hipLaunchKernelGGL((k_pages_read<FMT, D>), dim3(n, a.pool.nkv), dim3(256), 0, st, a, runs);
        return (int)hipGetLastError();
    }
};

// Runs as an argument of a launch; `dev` holds those of a long list already.
PageRuns runs_of(const std::vector<PageRun> &v, const DevBuf &dev) {
    PageRuns r;
    r.list = nullptr;
    if (v.size() > kInlineRuns) r.list = (const PageRun *)dev.p;
    else memcpy(r.some, v.data(), v.size() * sizeof(PageRun));
    return r;
}

// Costs fitted to measured calls (a block of 32 tokens of D = 128: 0.7 us where the memory
// bounds it, 1.1 for 128 rows).
PageForms forms_of(const fl_pages *p) {
    const int fmt = p->cfg.kv_format, D = p->cfg.head_dim, cus = 256;
    const int fill = 2 * cus;  // (4 a CU, which D = 64 has the registers for, 22 us against 19 for 32768 tokens of 8 x 64, binary16)
    if (fmt == FL_KV_F16) return {3, {16, 64, 128}, fill, {1, 1, 1.6f}, 6, 8, cus};
    return {2, {16, 32}, fill, {2, 3}, 6, 4, cus * page_waves(fmt, D, 2)};
}

// Whether the workgroups of the plan's items join its partial results: where the last to
// arrive reads 8 at most per thread (4 channels of a query and head), in flight together, and
// they are few (8 answers behind 785 tokens 14.8 us against 17.3 with a launch for them, drafts
// of 5 sequences 14.4 against 17.0, 21 sequences behind 595 tokens, two times 4 a thread, 15.4
// against 17.7).  With more it goes over them again and again, past the caches: two times 8 of
// 4 sequences behind 1774 tokens 19.2 against 17.6, 16 sequences of up to 8000 45.4 against 41.7,
// 32 in a tree 44 against 24.  (Calls one after another, which the host's launches bound; the
// GPU alone takes 11.6 us for the 8 answers against 9.4 with the second launch: the stores past the
// caches, the count and the loads behind it are a chain of 4 us.)  And stores past the caches cost more than those that
// stay: 644 queries, 10 MB, 62.2 against 58.5.  (One workgroup a kv head clears the rows of
// queries that see nothing: few.)
bool joins_here(const fl_pages *p, int heads) {
    const PagePlan &l = p->plan;
    const int threads = l.wide && p->cfg.kv_format == FL_KV_F16 ? 512 : 256;
    const int rows = l.most_queries * (heads / p->cfg.num_kv_heads);
    const long long rounds = (rows * (p->cfg.head_dim / 4) + threads - 1) / threads;
    return !l.items.empty() && l.empty <= 64 && rounds * l.most_parts <= 8 &&
           (long long)l.num_units * heads * p->cfg.head_dim <= (1 << 18);
}

// The plan of these queries, on the device.
int make_plan(fl_pages *p, const int32_t *seqs, const int32_t *seen, int n, int heads) {
    const int group = heads / p->cfg.num_kv_heads;
    if (p->plan_version == p->t.version && p->plan_heads == heads && (int)p->plan_seqs.size() == n &&
        !memcmp(p->plan_seqs.data(), seqs, n * sizeof *seqs) && !memcmp(p->plan_seen.data(), seen, n * sizeof *seen))
        return 0;
    p->plan_version = 0;
    PGTRY(on_table(p, [&](PageTable &t) {
        const int rc = page_plan(t, seqs, seen, n, group, p->cfg.num_kv_heads, p->cfg.head_dim, forms_of(p), p->plan);
        if (rc) return rc;
        p->plan_seqs.assign(seqs, seqs + n);
        p->plan_seen.assign(seen, seen + n);
        return 0;
    }));
    const PagePlan &l = p->plan;
    size_t bytes = 0;
    auto place = [&](size_t b) {
        const size_t at = bytes;
        bytes = (bytes + b + 63) / 64 * 64;
        return at;
    };
    place(l.items.size() * sizeof(PageItem));
    p->plan_order = place(l.order.size() * sizeof(PageQuery));
    p->plan_pages = place(l.page_ids.size() * sizeof(int));
    p->plan_units = place(l.units.size() * sizeof(int));
    p->plan_joins = place(l.joins.size() * sizeof(PageJoin));
    p->plan_join_of = place(l.join_of.size() * sizeof(int));
    p->plan_arrived = bytes;
    const size_t counts = joins_here(p, heads) ? l.joins.size() * p->cfg.num_kv_heads * sizeof(int) : 0;
    bytes += counts;
    char *h;
    PGTRY(ensure(p, p->d_plan, bytes));
    PGTRY(ensure(p, p->ws, (size_t)l.num_units * heads * (p->cfg.head_dim + 2) * sizeof(float)));
    PGTRY(stage_for(p, bytes, &h));
    auto put = [&](size_t at, const auto &v) {
        if (!v.empty()) memcpy(h + at, v.data(), v.size() * sizeof v[0]);
    };
    put(0, l.items);
    put(p->plan_order, l.order);
    put(p->plan_pages, l.page_ids);
    put(p->plan_units, l.units);
    put(p->plan_joins, l.joins);
    put(p->plan_join_of, l.join_of);
    memset(h + p->plan_arrived, 0, counts);
    PGTRY(send(p, p->d_plan.p, bytes));
    p->plan_heads = heads;
    p->plan_version = p->t.version;
    return 0;
}

int check_layers(fl_pages *p, int layer, int layers) {
    if (layer < 0 || layers < 1 || layer > p->cfg.num_layers - layers)
        return fail(p, FL_E_INVALID, "layers %d..%d of %d", layer, layer + layers - 1, p->cfg.num_layers);
    return 0;
}

}  // namespace

int fl_pages_bytes(const fl_pages_config *cfg, size_t *kv_bytes, size_t *scale_bytes) {
    PGTRY(check_config(cfg));
    const size_t values = (size_t)cfg->num_layers * cfg->num_pages * cfg->num_kv_heads * cfg->page_size * cfg->head_dim;
    if (kv_bytes) *kv_bytes = values * elem_bytes(cfg->kv_format);
    if (scale_bytes) *scale_bytes = cfg->kv_format == FL_KV_Q8 ? values / 32 * 2 : 0;
    return 0;
}

int fl_pages_create(fl_ctx *ctx, const fl_pages_config *cfg, void *k, void *v, void *k_scale, void *v_scale,
                    fl_pages **out) {
    if (!out) return fail(nullptr, FL_E_INVALID, "out is null");
    *out = nullptr;
    PGTRY(check_config(cfg));
    const bool q8 = cfg->kv_format == FL_KV_Q8;
    if (ctx) {
        if (!k || !v || (q8 && (!k_scale || !v_scale))) return fl_host_fail(ctx, FL_E_INVALID, "null pool memory");
        for (const void *p : {k, v, q8 ? k_scale : nullptr, q8 ? v_scale : nullptr})
            if ((uintptr_t)p % 16) return fl_host_fail(ctx, FL_E_INVALID, "pool memory is not aligned to 16 bytes");
    }
    fl_pages *p = new (std::nothrow) fl_pages();
    if (!p) return fl_host_fail(ctx, FL_E_OOM, "out of host memory");
    p->ctx = ctx;
    p->cfg = *cfg;
    p->pool = PagePool{k, v, (uint16_t *)k_scale, (uint16_t *)v_scale, cfg->num_layers, cfg->num_pages, cfg->page_size,
                       cfg->num_kv_heads, cfg->page_size / kPageBlock, 0};
    // exact for x < 2^19 blocks: the error x / 2^32 is below 1 / per (per <= 128; per = 1 has no 32-bit inverse)
    p->pool.per_inv = p->pool.per > 1 ? (uint32_t)(((1ull << 32) + p->pool.per - 1) / p->pool.per) : 0;
    if (ctx) {
        p->device = fl_ctx_device(ctx);
        p->stream = (hipStream_t)fl_ctx_stream(ctx);
    }
    int rc = on_table(p, [&](PageTable &t) { return t.init(*cfg); });
    if (!rc && ctx && cfg->num_pages > kInlineCopies) {
        OnDevice on(p);
        // (a call's copies go to as many pages at most, so this never fails later)
        rc = ensure(p, p->d_copies, (size_t)cfg->num_pages * sizeof(PageCopy));
    }
    if (rc) {
        fl_pages_destroy(p);
        return rc;
    }
    *out = p;
    return 0;
}

void fl_pages_destroy(fl_pages *p) {
    if (!p) return;
    if (p->ctx) {
        OnDevice on(p);
        // (hipFree waits for the device, so the context may be gone already)
        for (DevBuf *b : {&p->d_plan, &p->d_runs, &p->d_read, &p->d_copies, &p->ws})
            if (b->p) (void)hipFree(b->p);
        for (Stage &s : p->stages) {
            if (s.done) (void)hipEventDestroy(s.done);
            if (s.host) (void)hipHostFree(s.host);
        }
    }
    delete p;
}

int fl_pages_fork(fl_pages *p, const int32_t *src, const int32_t *dst, const int32_t *lens, int n) {
    return on_table(p, [&](PageTable &t) { return t.fork(src, dst, lens, n); });
}

int fl_pages_free(fl_pages *p, const int32_t *seqs, int n) {
    return on_table(p, [&](PageTable &t) { return t.release(seqs, n); });
}

int fl_pages_truncate(fl_pages *p, const int32_t *seqs, const int32_t *lens, int n) {
    return on_table(p, [&](PageTable &t) { return t.truncate(seqs, lens, n); });
}

int fl_pages_copy(fl_pages *p, const int32_t *src, const int32_t *dst, int n) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    if (!p->ctx) return on_table(p, [&](PageTable &t) { return t.copy(src, dst, n); });
    PGTRY(check_stream(p));
    OnDevice on(p);
    PGTRY(copies_room(p, 0, std::min((long long)std::max(n, 0) * p->t.max_pages, (long long)p->t.free_pages)));
    PGTRY(on_table(p, [&](PageTable &t) { return t.copy(src, dst, n); }));
    return run_copies(p);
}

int fl_pages_compact(fl_pages *p, int *moved) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    OnDevice on(p);
    if (p->ctx) {
        PGTRY(check_stream(p));
        PGTRY(copies_room(p, 0, std::min(p->t.free_pages, p->cfg.num_pages - p->t.free_pages)));
    }
    PGTRY(on_table(p, [&](PageTable &t) { return t.compact(); }));
    if (moved) *moved = (int)p->t.copies.size();
    return p->ctx ? run_copies(p) : 0;
}

int fl_pages_extend(fl_pages *p, const int32_t *seqs, const int32_t *counts, int n) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    if (!p->ctx) return on_table(p, [&](PageTable &t) { return t.extend(seqs, counts, n); });
    PGTRY(check_stream(p));
    OnDevice on(p);
    // Room for the lists first: no allocation fails behind the bookkeeping.  A call that fails
    // in it leaves the runs of the one before, and these may still be written.
    long long most = 0;
    for (int i = 0; i < n && counts; i++) most += std::min(std::max(counts[i], 0), p->cfg.max_seq_len) / kPageBlock + 2;
    most = std::min(most, (long long)p->cfg.num_pages * p->pool.per + n);
    if (most > kMaxGrid) return fail(p, FL_E_INVALID, "too many tokens at once");
    DevBuf more;
    const size_t bytes = most > kInlineRuns ? (size_t)most * sizeof(PageRun) : 0;
    int rc = copies_room(p, 0, n);  // (the first to be sent, or behind the runs)
    if (!rc && bytes) rc = copies_room(p, 1, n);
    if (!rc && bytes) rc = stage_room(p, 0, bytes);
    if (!rc && bytes > p->d_runs.cap) rc = ensure(p, more, std::max(bytes, 2 * p->d_runs.cap));
    if (!rc) rc = on_table(p, [&](PageTable &t) { return t.extend(seqs, counts, n); });
    if (!rc && more.p) std::swap(more, p->d_runs);
    if (more.p) (void)hipFree(more.p);  // (waits for what reads it)
    if (rc) return rc;
    const auto &r = p->t.runs;
    if (r.size() > kInlineRuns) PGTRY(upload(p, p->d_runs, r.data(), r.size() * sizeof(PageRun)));
    return run_copies(p);
}

int fl_pages_write(fl_pages *p, int layer, int layers, const float *k, const float *v, size_t row_stride) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    PGTRY(check_layers(p, layer, layers));
    PGTRY(check_stream(p));
    const size_t row = (size_t)p->cfg.num_kv_heads * p->cfg.head_dim;
    if (!k || !v) return fail(p, FL_E_INVALID, "null keys or values");
    if (((uintptr_t)k | (uintptr_t)v) % 4) return fail(p, FL_E_INVALID, "keys or values are not aligned");
    if (row_stride < row) return fail(p, FL_E_INVALID, "rows of %zu values %zu apart", row, row_stride);
    if (!p->t.runs_valid) return fail(p, FL_E_STATE, "fl_pages_write follows fl_pages_extend, with no other change between");
    if (!p->t.tokens) return 0;
    OnDevice on(p);
    PageWriteArgs a{};
    a.pool = p->pool;
    a.k = k;
    a.v = v;
    a.stride = (long long)row_stride;
    a.layer0 = layer;
    a.n = p->t.tokens;
    const int n = (int)p->t.runs.size();
    PGCHK(p, (hipError_t)with_form(p->cfg.kv_format, p->cfg.head_dim,
                                   LaunchWrite{p->stream, a, runs_of(p->t.runs, p->d_runs), n, layers}));
    return 0;
}

int fl_pages_read(fl_pages *p, int layer, const int32_t *seqs, const int32_t *starts, const int32_t *counts, int n,
                  float *k, float *v) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    PGTRY(check_layers(p, layer, 1));
    PGTRY(check_stream(p));
    if (n < 0 || (n > 0 && (!seqs || !starts || !counts))) return fail(p, FL_E_INVALID, "bad sequence list");
    std::vector<PageRun> runs;
    PGTRY(on_table(p, [&](PageTable &t) {
        long long total = 0;
        for (int i = 0; i < n; i++) {
            if (seqs[i] < 0 || seqs[i] >= t.seqs || starts[i] < 0 || counts[i] < 0 ||
                (long long)starts[i] + counts[i] > t.len[seqs[i]]) {
                t.error = "tokens that are not there";
                return FL_E_INVALID;
            }
            total += counts[i];
        }
        if (total > 0x7FFFFFFFll) {
            t.error = "too many tokens";
            return FL_E_INVALID;
        }
        int token = 0;
        for (int i = 0; i < n; i++) {
            t.add_runs(seqs[i], starts[i], starts[i] + counts[i], token, runs);
            token += counts[i];
        }
        return 0;
    }));
    if (runs.empty()) return 0;
    if (!k && !v) return fail(p, FL_E_INVALID, "null keys and values");
    if (((uintptr_t)k | (uintptr_t)v) % 4) return fail(p, FL_E_INVALID, "keys or values are not aligned");
    if (runs.size() > kMaxGrid) return fail(p, FL_E_INVALID, "too many tokens at once");
    OnDevice on(p);
    if (runs.size() > kInlineRuns) PGTRY(upload(p, p->d_read, runs.data(), runs.size() * sizeof(PageRun)));
    PageReadArgs a{p->pool, k, v, layer};
    PGCHK(p, (hipError_t)with_form(p->cfg.kv_format, p->cfg.head_dim,
                                   LaunchRead{p->stream, a, runs_of(runs, p->d_read), (int)runs.size()}));
    return 0;
}

int fl_pages_attention(fl_pages *p, int layer, const float *q, size_t q_stride, const int32_t *seqs,
                       const int32_t *seen, int n, int num_heads, float *out) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    PGTRY(check_layers(p, layer, 1));
    const int D = p->cfg.head_dim, nkv = p->cfg.num_kv_heads;
    if (num_heads < 1 || num_heads % nkv) return fail(p, FL_E_INVALID, "%d heads over %d kv heads", num_heads, nkv);
    if (num_heads / nkv > kPageMaxGroup || num_heads > 65535)
        return fail(p, FL_E_UNSUPPORTED, "%d query heads, %d per kv head", num_heads, num_heads / nkv);
    if (n < 0 || n > kPageMaxQueries) return fail(p, FL_E_INVALID, "%d queries (up to %d)", n, kPageMaxQueries);
    if (n == 0) return 0;
    if (!q || !out || !seqs || !seen) return fail(p, FL_E_INVALID, "null argument");
    if ((uintptr_t)q % 4 || (uintptr_t)out % 16) return fail(p, FL_E_INVALID, "queries or result are not aligned");
    if (q_stride < (size_t)num_heads * D) return fail(p, FL_E_INVALID, "queries of %d values %zu apart", num_heads * D, q_stride);
    PGTRY(check_stream(p));
    const uintptr_t q0 = (uintptr_t)q, o0 = (uintptr_t)out;
    if (q0 < o0 + (size_t)n * num_heads * D * 4 && o0 < q0 + ((n - 1) * q_stride + (size_t)num_heads * D) * 4)
        return fail(p, FL_E_INVALID, "queries and result overlap");
    OnDevice on(p);
    PGTRY(make_plan(p, seqs, seen, n, num_heads));
    const PagePlan &l = p->plan;
    const char *d = p->d_plan.p;
    PageAttnArgs a{};
    a.pool = p->pool;
    a.layer = layer;
    a.group = num_heads / nkv;
    a.scale = (float)(1.4426950408889634 / std::sqrt((double)D));
    a.q = q;
    a.q_stride = (long long)q_stride;
    a.order = (const PageQuery *)(d + p->plan_order);
    a.page_ids = (const int *)(d + p->plan_pages);
    a.part = (float *)p->ws.p;
    a.ml = a.part + (size_t)l.num_units * num_heads * D;
    a.out = out;
    a.items = (const PageItem *)d;
    const bool here = joins_here(p, num_heads);
    if (here && !l.joins.empty()) {
        a.arrived = (int *)(d + p->plan_arrived);
        a.joins = (const PageJoin *)(d + p->plan_joins);
        a.units = (const int *)(d + p->plan_units);
        a.join_of = (const int *)(d + p->plan_join_of);
        a.njoins = (int)l.joins.size();
        a.nempty = l.empty;
    }
    if ((long long)l.items.size() * nkv > (l.wide && p->cfg.kv_format == FL_KV_F16 ? kMaxGrid / 2 : kMaxGrid)) return fail(p, FL_E_INVALID, "too many queries at once");
    if (!l.items.empty())
        PGCHK(p, (hipError_t)with_form(p->cfg.kv_format, D, LaunchAttn{p->stream, a, (int)l.items.size(), l.wide}));
    if (!here && !l.joins.empty()) {
        PageJoinArgs j{(const PageJoin *)(d + p->plan_joins), (const int *)(d + p->plan_units), a.part, a.ml, out, num_heads};
        const dim3 grid((unsigned)l.joins.size(), (unsigned)((num_heads * D + 127) / 128));
        if (D == 64) hipLaunchKernelGGL(k_pages_join<64>, grid, dim3(256), 0, p->stream, j);
        else hipLaunchKernelGGL(k_pages_join<128>, grid, dim3(256), 0, p->stream, j);
        PGCHK(p, hipGetLastError());
    }
    return 0;
}

int fl_pages_len(const fl_pages *p, int seq) { return p && seq >= 0 && seq < p->t.seqs ? p->t.len[seq] : -1; }

int fl_pages_pending(const fl_pages *p) { return p && p->t.runs_valid ? p->t.tokens : -1; }

int fl_pages_free_count(const fl_pages *p) { return p ? p->t.free_pages : -1; }

int fl_pages_tables(const fl_pages *p, int32_t *tables, int32_t *lens) {
    if (!p) return fl_host_fail(nullptr, FL_E_INVALID, "null pages");
    if (tables) memcpy(tables, p->t.table.data(), p->t.table.size() * sizeof(int));
    if (lens) memcpy(lens, p->t.len.data(), p->t.len.size() * sizeof(int));
    return 0;
}

int fl_pages_copies(const fl_pages *p, int32_t *copies, int cap) {
    if (!p) return -1;
    const auto &c = p->t.copies;
    for (int i = 0; copies && i < cap && i < (int)c.size(); i++) {
        copies[3 * i] = c[i].src;
        copies[3 * i + 1] = c[i].dst;
        copies[3 * i + 2] = c[i].blocks;
    }
    return (int)c.size();
}

int fl_pages_plan(fl_pages *p, const int32_t *seqs, const int32_t *seen, int n, int num_heads, int32_t *items, int cap) {
    if (!p) return fail(p, FL_E_INVALID, "null pages");
    const int nkv = p->cfg.num_kv_heads;
    if (num_heads < 1 || num_heads % nkv || num_heads / nkv > kPageMaxGroup)
        return fail(p, FL_E_INVALID, "%d heads over %d kv heads", num_heads, nkv);
    int made = 0;
    PGTRY(on_table(p, [&](PageTable &t) {
        PagePlan l;
        const int rc = page_plan(t, seqs, seen, n, num_heads / nkv, nkv, p->cfg.head_dim, forms_of(p), l);
        if (rc) return rc;
        for (const PageItem &it : l.items)
            for (int i = 0; i < it.nq; i++, made++) {
                if (!items || made >= cap) continue;
                const int row[6] = {l.order[it.q0 + i].query, it.slot0, it.slot1, l.page_ids[it.page0], it.form,
                                    it.unit < 0 ? -1 : it.unit + i};
                memcpy(items + 6 * made, row, sizeof row);
            }
        return 0;
    }));
    return made;
}
