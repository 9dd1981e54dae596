// paged.cuh -- what the paged-cache operators share: the argument checks (pure host code: they run without a device) and the device view of a paged cache.
#pragma once
#include "api_internal.h"
#include <atomic>
#include <initializer_list>

#define OP_CHECK(cond, ...) do { if (!(cond)) return cdna4_set_err(CDNA4_E_UNSUPPORTED, __VA_ARGS__); } while (0)
#define ARG_CHECK(cond, ...) do { if (!(cond)) return cdna4_set_err(CDNA4_E_INVALID, __VA_ARGS__); } while (0)

constexpr long PAGED_MAX_SEQ = 8192, PAGED_MAX_SLOTS = 1l << 30;

// the device of the context for the duration of a call: the caller's current device is put back afterwards (tensors may live on another device than the current one)
struct DeviceScope {
    int prev = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != device) err = hipSetDevice(device); else prev = -1;
    }
    ~DeviceScope() { if (prev >= 0) (void)hipSetDevice(prev); }
};
// opt a kernel in to `bytes` of dynamic LDS beside its static LDS, once per device (function attributes belong to a device).  K: the kernel; a failed attempt is made again by the next call
template <auto K> static inline hipError_t pg_opt_in_lds(int device, int bytes) {
    static std::atomic<unsigned long long> done{0};
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute((const void *)K, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
    return e;
}
#define DEVICE_SCOPE(ctx) DeviceScope device_scope_((ctx)->device); HIP_TRY(device_scope_.err)

// device view of the cache: rows are addressed as 64-bit page base + 32-bit offset inside the page
struct PagedCache {
    char *k, *v; const int *table, *n_kv;
    long k_page, v_page, k_head, v_head;        // bytes between pages / KV heads
    int k_row, v_row;                           // bytes between the slots of a page (page * row < 2^31)
    int page_shift, W, n_pages, n_seq, n_head_kv, D;
    long table_row;                             // ints between table rows
};
static __device__ __forceinline__ int paged_len(const PagedCache &c, int s) { const long cap = (long)c.W << c.page_shift; return (int)min((long)max(c.n_kv[s], 0), cap); }
// page id of slot j of sequence s, -1 if it is not mapped
static __device__ __forceinline__ int paged_page(const PagedCache &c, int s, int j) {
    const int id = c.table[(long)s * c.table_row + (j >> c.page_shift)];
    return (unsigned)id < (unsigned)c.n_pages ? id : -1;
}

static inline long pg_extent(const cdna4_tensor *t, int esz) {          // bytes from the first to behind the last element
    long e = esz; for (int i = 0; i < 4; ++i) e += (t->ne[i] - 1) * t->nb[i]; return e;
}
static inline bool pg_empty(const cdna4_tensor *t) { for (int i = 0; i < 4; ++i) if (t->ne[i] <= 0) return true; return false; }
// no two elements at one address (written tensors): every dimension steps over the extent of the smaller ones
static inline bool pg_disjoint_elems(const cdna4_tensor *t, int esz) {
    int o[4] = {0, 1, 2, 3};
    for (int i = 0; i < 4; ++i) for (int j = i + 1; j < 4; ++j) if (t->nb[o[j]] < t->nb[o[i]]) { const int x = o[i]; o[i] = o[j]; o[j] = x; }
    long need = esz;
    for (int i = 0; i < 4; ++i) { const int d = o[i]; if (t->ne[d] <= 1) continue; if (t->nb[d] < need) return false; need = t->nb[d] * (t->ne[d] - 1) + need; }
    return true;
}
static inline bool pg_overlap(const void *a, long na, const void *b, long nb) { const char *x = (const char *)a, *y = (const char *)b; return x && y && x < y + nb && y < x + na; }
static inline bool pg_overlap(const cdna4_tensor *a, int ea, const cdna4_tensor *b, int eb) { return pg_overlap(a->data, pg_extent(a, ea), b->data, pg_extent(b, eb)); }
// memory of an argument: nothing that a call writes may share bytes with anything else that it reads or writes (the workgroups that write run beside those that read)
struct PgRange { const char *name; const void *p; long n; bool written; };
static inline PgRange pg_range(const char *name, const cdna4_tensor *t, int esz, bool written) { return PgRange{name, t && !pg_empty(t) ? t->data : nullptr, t && !pg_empty(t) ? pg_extent(t, esz) : 0, written}; }
static inline PgRange pg_range(const char *name, const void *p, long n, bool written) { return PgRange{name, n > 0 ? p : nullptr, n, written}; }
// pairs: i * 16 + j, i < j, of arguments that have a check of their own
template <int N> static inline int pg_apart(const char *op, const PgRange (&r)[N], std::initializer_list<int> pairs = {}) {
    for (int i = 0; i < N; ++i) for (int j = i + 1; j < N; ++j) {
        if (!r[i].written && !r[j].written) continue;
        bool own = false; for (const int x : pairs) own |= x == i * 16 + j;
        ARG_CHECK(own || !pg_overlap(r[i].p, r[i].n, r[j].p, r[j].n), "%s: %s and %s share memory and one of them is written", op, r[i].name, r[j].name);
    }
    return CDNA4_OK;
}
static inline bool pg_same(const cdna4_tensor *a, const cdna4_tensor *b) {
    if (a->data != b->data) return false;
    for (int i = 0; i < 4; ++i) if (a->ne[i] != b->ne[i] || (a->ne[i] > 1 && a->nb[i] != b->nb[i])) return false;
    return true;
}
static inline bool pg_sizes_ok(const cdna4_tensor *t) {                 // (no product of sizes and strides below leaves 64 bits)
    for (int i = 0; i < 4; ++i) if (t->ne[i] < 0 || t->ne[i] > (1l << 40) || t->nb[i] < 0 || (t->ne[i] > 1 && t->nb[i] > (1l << 48) / (t->ne[i] - 1))) return false;
    return true;
}

// K and V caches that a call writes are apart: memory of their own, or views of one pool that take turns (pages of K beside pages of V, or rows inside a page)
static inline bool pg_kv_apart(const cdna4_tensor *k, const cdna4_tensor *v) {
    if (pg_empty(k) || !pg_overlap(k, 2, v, 2)) return true;
    if (k->ne[3] > 1 && k->nb[3] == v->nb[3]) {          // in-page extents that both fit beside each other into the distance of two pages
        cdna4_tensor kp = *k, vp = *v; kp.ne[3] = vp.ne[3] = 1;
        const long step = k->nb[3], ek = pg_extent(&kp, 2), ev = pg_extent(&vp, 2), d = (((const char *)v->data - (const char *)k->data) % step + step) % step;
        if (ek <= d && d + ev <= step) return true;
    }
    for (int i = 0; i < 4; ++i) if (k->ne[i] > 1 && k->nb[i] != v->nb[i]) return false;
    // one tensor with a dimension of two for K and V: every stride steps over the extent of the smaller ones
    const char *kd = (const char *)k->data, *vd = (const char *)v->data;
    long ne[5] = {k->ne[0], k->ne[1], k->ne[2], k->ne[3], 2}, nb[5] = {k->nb[0], k->nb[1], k->nb[2], k->nb[3], vd > kd ? vd - kd : kd - vd}, need = 2;
    for (int n = 0; n < 5; ++n) {
        int least = -1; for (int i = 0; i < 5; ++i) if (ne[i] > 1 && (least < 0 || nb[i] < nb[least])) least = i;
        if (least < 0) break;
        if (nb[least] < need) return false;
        need += nb[least] * (ne[least] - 1); ne[least] = 1;
    }
    return true;
}

// a descriptor whose dimensions of one element (or none) have the strides of a dense tensor: the caller's say nothing
static inline cdna4_tensor pg_norm(const cdna4_tensor *t, int esz) {
    cdna4_tensor n = *t;
    for (int i = 0; i < 4; ++i) if (n.ne[i] == 1) n.nb[i] = i ? n.nb[i - 1] * n.ne[i - 1] : esz;
    return n;
}
#define PG_NORM(t, esz) cdna4_tensor t##_n; if (t) { t##_n = pg_norm(t, esz); t = &t##_n; }
// cache + table of an operator; `written`: the operator stores into the cache.  Fills c (data pointers of an empty call may be NULL: the caller returns before it launches).
static inline int pg_cache_check(const char *op, const cdna4_tensor *k, const cdna4_tensor *v, const cdna4_tensor *table, bool written, PagedCache *c) {
    ARG_CHECK(k && v && table, "%s: null argument", op);
    ARG_CHECK(pg_sizes_ok(k) && pg_sizes_ok(v) && pg_sizes_ok(table), "%s: sizes and strides", op);
    PG_NORM(k, 2) PG_NORM(v, 2) PG_NORM(table, 4)
    OP_CHECK((k->type == CDNA4_TYPE_F16 || k->type == CDNA4_TYPE_BF16) && v->type == k->type, "%s: f16 or bf16 K and V caches", op);
    for (int i = 0; i < 4; ++i) ARG_CHECK(k->ne[i] == v->ne[i], "%s: K and V caches of one shape [D, page, n_head_kv, n_pages]", op);
    const long D = k->ne[0], page = k->ne[1];
    OP_CHECK(D == 64 || D == 128 || D == 256, "%s: head size 64, 128 or 256 (got %ld)", op, D);
    OP_CHECK(page >= 16 && page <= 4096 && (page & (page - 1)) == 0, "%s: pages of a power of two of slots, 16 to 4096 (got %ld)", op, page);
    OP_CHECK(k->ne[2] >= 1 && k->ne[2] <= 1024 && k->ne[3] >= 1 && k->ne[3] <= 0x7fffffffl, "%s: 1 to 1024 KV heads, 1 to 2^31 - 1 pages", op);
    for (const cdna4_tensor *t : {k, v}) {
        OP_CHECK(t->nb[0] == 2 && (uintptr_t)t->data % 16 == 0 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && t->nb[3] % 16 == 0, "%s: cache rows dense and 16-byte aligned", op);
        OP_CHECK(t->nb[1] <= (1l << 31) / page - 1, "%s: a page's rows within 2^31 bytes", op);
        ARG_CHECK(!written || pg_disjoint_elems(t, 2), "%s: the cache is written: its rows may not overlap", op);
        ARG_CHECK(t->data, "%s: null cache", op);
    }
    ARG_CHECK(table->type == CDNA4_TYPE_I32 && table->nb[0] == 4 && table->nb[1] % 4 == 0 && table->ne[2] == 1 && table->ne[3] == 1 && (uintptr_t)table->data % 4 == 0, "%s: table i32 [W, n_seq]", op);
    OP_CHECK(table->ne[1] <= PAGED_MAX_SEQ && table->ne[0] <= PAGED_MAX_SLOTS / page, "%s: at most %ld sequences of %ld slots", op, PAGED_MAX_SEQ, PAGED_MAX_SLOTS);
    int shift = 0; while ((1l << shift) < page) ++shift;
    c->k = (char *)k->data; c->v = (char *)v->data; c->table = (const int *)table->data; c->n_kv = nullptr;
    c->k_page = k->nb[3]; c->v_page = v->nb[3]; c->k_head = k->nb[2]; c->v_head = v->nb[2]; c->k_row = (int)k->nb[1]; c->v_row = (int)v->nb[1];
    c->page_shift = shift; c->W = (int)table->ne[0]; c->n_pages = (int)k->ne[3]; c->n_seq = (int)table->ne[1]; c->n_head_kv = (int)k->ne[2]; c->D = (int)D;
    c->table_row = table->nb[1] / 4;
    return CDNA4_OK;
}
// [>= W * page, n_head_kv, n_seq] of f32 (weight) or i32 (pos)
static inline int pg_slots_check(const char *op, const char *name, const cdna4_tensor *t, int type, const PagedCache &c, bool written) {
    ARG_CHECK(pg_sizes_ok(t) && t->type == type && t->nb[0] == 4 && (uintptr_t)t->data % 4 == 0 && t->nb[1] % 4 == 0 && t->nb[2] % 4 == 0, "%s: %s f32 (pos: i32) with dense rows", op, name);
    ARG_CHECK(t->ne[0] >= ((long)c.W << c.page_shift) && t->ne[1] == c.n_head_kv && t->ne[2] == c.n_seq && t->ne[3] == 1, "%s: %s [>= W * page, n_head_kv, n_seq]", op, name);
    ARG_CHECK(!written || pg_disjoint_elems(t, 4), "%s: %s is written: its elements may not overlap", op, name);
    return CDNA4_OK;
}
