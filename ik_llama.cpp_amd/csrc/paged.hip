// paged.hip -- storing into, evicting from and forking a paged key / value cache (the attention that reads it: paged_attn.hip).
#include "paged.cuh"
#include "fa_decode.cuh"
#include <algorithm>

struct SlotView { char *p; long head, seq; };           // weight / pos: bytes between KV heads and sequences
static SlotView slot_view(const cdna4_tensor *t) { SlotView s = {nullptr, 0, 0}; if (t) { s.p = (char *)t->data; s.head = t->nb[1]; s.seq = t->nb[2]; } return s; }
template <typename X> static __device__ __forceinline__ X *slot_row(const SlotView &v, int s, int h) { return reinterpret_cast<X *>(v.p + (long)s * v.seq + (long)h * v.head); }

// ------------------------------------------------------------------------------------------------ store
struct StoreArgs {
    PagedCache c; const char *k, *v; long k_head, v_head, k_tok, v_tok;
    const int *start, *n_past; SlotView weight, pos; int *n_kv_out; int n_tok, pack, blocks;          // pack: tokens of a workgroup; blocks: workgroups of tokens
};
// two f32 -> two 16-bit values of the cache type, rounded to nearest even (the one rounding of K and V)
template <bool BF16> static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) return float_to_bf16_bits(a) | (float_to_bf16_bits(b) << 16);
    else { typedef _Float16 h2 __attribute__((ext_vector_type(2))); const h2 h = {(_Float16)a, (_Float16)b}; return __builtin_bit_cast(uint32_t, h); }
}
// the sequence of token i (the same for all lanes): the last s with start[s] <= i, -1 if there is none (a wave reads the whole vector at once: one memory latency instead of a binary
// search's chain of them)
static __device__ __forceinline__ int token_seq(const int *start, int n_seq, int i) {
    int n = 0;
    for (int b = 0; b < n_seq; b += 64) {
        const int s = b + (int)(threadIdx.x & 63);
        n += __popcll(__ballot(s < n_seq && start[min(s, n_seq - 1)] <= i));
    }
    return n - 1;
}
// One workgroup per token, or per 256 / units tokens where a token's rows are half a workgroup's or less (one to a workgroup / packed: 16000 tokens of one head of 64: 18.5 / 5.5 us, of four:
// 13.4 / 8.5).  A thread moves 8 values of K or V at a time (32 bytes in, 16 out).  Bound by memory for prompts (16866 tokens of 8 x 128 in six ragged sequences, bf16: 208 MB in 42 us,
// 5.0 TB/s, what a large copy reaches), by the chain of lookups for single tokens (64 sequences: 3 us).  The f32 rows do not depend on where they go: the first load of every thread runs
// under the lookups of sequence, length and page (unconditional, on a clamped unit: loaded under a branch and carried into the loop, this compiler reuses three of the four registers before
// they are read).
template <bool BF16> __global__ void __launch_bounds__(256) paged_store_kernel(StoreArgs a) {
    if ((int)blockIdx.x >= a.blocks) {          // the workgroups behind the tokens: the new lengths
        const int s = ((int)blockIdx.x - a.blocks) * 256 + (int)threadIdx.x;
        if (s < a.c.n_seq) {
            const int n = a.c.n_kv[s], add = a.start ? max(a.start[s + 1] - a.start[s], 0) : 1;
            a.n_kv_out[s] = n < 0 ? n : (int)min((long)n + add, (long)a.c.W << a.c.page_shift);
        }
        return;
    }
    const int lg = a.c.D == 64 ? 3 : a.c.D == 128 ? 4 : 5, half = a.c.n_head_kv << lg, units = 2 * half;        // units of 8 values: all of K, then all of V
    int tok = blockIdx.x, u = threadIdx.x, step = 256;
    if (a.pack > 1) { const int nth = (int)threadIdx.x / units; tok = tok * a.pack + nth; u -= nth * units; step = units; if (nth >= a.pack) tok = a.n_tok; }
    const int row = min(tok, a.n_tok - 1);
    auto source = [&](int u) {
        const int w = u >= half ? u - half : u, h = w >> lg, d = (w - (h << lg)) * 8;
        return reinterpret_cast<const float4 *>((u >= half ? a.v + (long)row * a.v_tok + (long)h * a.v_head : a.k + (long)row * a.k_tok + (long)h * a.k_head) + d * 4);
    };
    const float4 *src = source(min(u, units - 1));
    const float4 f0 = src[0], f1 = src[1];
    int s = tok;
    if (a.start) {
        s = token_seq(a.start, a.c.n_seq, __builtin_amdgcn_readfirstlane(tok));                                     // of the wave's first token;
        if (a.pack > 1) while (s + 1 < a.c.n_seq && a.start[s + 1] <= tok) ++s;                                     // its others lie in the same or a later one
    }
    if (tok >= a.n_tok || s < 0 || s >= a.c.n_seq || (a.start && tok >= a.start[a.c.n_seq])) return;
    const int n = a.c.n_kv[s], nth = a.start ? tok - a.start[s] : 0;
    const long slot = (long)n + nth;
    if (n < 0 || nth < 0 || slot >= ((long)a.c.W << a.c.page_shift)) return;
    const int page = paged_page(a.c, s, (int)slot);
    if (page < 0) return;
    const int in = (int)slot & ((1 << a.c.page_shift) - 1);
    char *kp = a.c.k + (long)page * a.c.k_page + (long)in * a.c.k_row, *vp = a.c.v + (long)page * a.c.v_page + (long)in * a.c.v_row;
    auto store = [&](int unit, const float4 &x, const float4 &y) {
        const int w = unit >= half ? unit - half : unit, h = w >> lg, d = (w - (h << lg)) * 8;
        char *p = unit >= half ? vp + (long)h * a.c.v_head : kp + (long)h * a.c.k_head;
        *reinterpret_cast<uint4 *>(p + d * 2) = make_uint4(pack2<BF16>(x.x, x.y), pack2<BF16>(x.z, x.w), pack2<BF16>(y.x, y.y), pack2<BF16>(y.z, y.w));
    };
    const int first = u;
    if (u < units) store(u, f0, f1);
    for (u += step; u < units; u += step) { const float4 *p = source(u); const float4 x = p[0], y = p[1]; store(u, x, y); }
    for (int h = first; h < a.c.n_head_kv; h += step) {
        if (a.weight.p) slot_row<float>(a.weight, s, h)[slot] = 0.0f;
        if (a.pos.p) slot_row<int>(a.pos, s, h)[slot] = a.n_past[s] + nth;
    }
}
static int new_rows_check(const char *name, const cdna4_tensor *t, const PagedCache &c) {
    ARG_CHECK(pg_sizes_ok(t) && t->type == CDNA4_TYPE_F32 && t->ne[0] == c.D && t->ne[1] == c.n_head_kv && t->ne[3] == 1, "paged_store: %s f32 [D, n_head_kv, n_tok]", name);
    OP_CHECK(t->nb[0] == 4 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && (uintptr_t)t->data % 16 == 0, "paged_store: %s rows dense and 16-byte aligned", name);
    return CDNA4_OK;
}
int cdna4_op_paged_store(cdna4_context *ctx, const cdna4_tensor *k, const cdna4_tensor *v, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table,
                         const int32_t *n_kv, const int32_t *start, const int32_t *n_past, const cdna4_tensor *weight, const cdna4_tensor *pos, int32_t *n_kv_out, void *stream) {
    ARG_CHECK(ctx && k && v, "paged_store: null argument");
    PG_NORM(k, 4) PG_NORM(v, 4) PG_NORM(weight, 4) PG_NORM(pos, 4)
    StoreArgs a; int rc = pg_cache_check("paged_store", k_cache, v_cache, table, true, &a.c); if (rc) return rc;
    if ((rc = new_rows_check("k", k, a.c)) || (rc = new_rows_check("v", v, a.c))) return rc;
    ARG_CHECK(k->ne[2] == v->ne[2], "paged_store: as many rows of k as of v");
    const long n_tok = k->ne[2], n_seq = a.c.n_seq;
    OP_CHECK(n_tok <= (1l << 23), "paged_store: at most 2^23 tokens");
    ARG_CHECK(start || n_tok == n_seq, "paged_store: without start, one token per sequence");
    if (weight && (rc = pg_slots_check("paged_store", "weight", weight, CDNA4_TYPE_F32, a.c, true))) return rc;
    if (pos && (rc = pg_slots_check("paged_store", "pos", pos, CDNA4_TYPE_I32, a.c, true))) return rc;
    if (n_seq == 0) return CDNA4_OK;
    ARG_CHECK(n_kv && (a.c.table || a.c.W == 0) && (n_tok == 0 || (k->data && v->data)) && (!pos || n_past), "paged_store: null data");
    ARG_CHECK((!weight || weight->data || a.c.W == 0) && (!pos || pos->data || a.c.W == 0), "paged_store: null data");
    const PgRange args[] = {pg_range("k_cache", k_cache, 2, true), pg_range("v_cache", v_cache, 2, true), pg_range("weight", weight, 4, true), pg_range("pos", pos, 4, true),
                            pg_range("n_kv_out", n_kv_out, n_seq * 4, true), pg_range("k", k, 4, false), pg_range("v", v, 4, false), pg_range("table", table, 4, false),
                            pg_range("n_kv", n_kv, n_seq * 4, false), pg_range("start", start, (n_seq + 1) * 4, false), pg_range("n_past", n_past, n_seq * 4, false)};
    if ((rc = pg_apart("paged_store", args, {0 * 16 + 1}))) return rc;
    ARG_CHECK(pg_kv_apart(k_cache, v_cache), "paged_store: K and V share rows");
    a.k = (const char *)k->data; a.v = (const char *)v->data; a.k_head = k->nb[1]; a.v_head = v->nb[1]; a.k_tok = k->nb[2]; a.v_tok = v->nb[2];
    a.c.n_kv = n_kv; a.start = start; a.n_past = n_past; a.weight = slot_view(weight); a.pos = slot_view(pos); a.n_kv_out = n_kv_out; a.n_tok = (int)n_tok;
    const int units = 2 * a.c.n_head_kv * (a.c.D / 8);
    a.pack = std::max(1, 256 / units); a.blocks = (int)((n_tok + a.pack - 1) / a.pack);
    const long blocks = a.blocks + (n_kv_out ? (n_seq + 255) / 256 : 0);
    if (blocks == 0) return CDNA4_OK;
    DEVICE_SCOPE(ctx);
    if (k_cache->type == CDNA4_TYPE_BF16) hipLaunchKernelGGL(paged_store_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(paged_store_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}

// ------------------------------------------------------------------------------------------------ fork
struct ForkArgs { PagedCache c; const int *parent, *fresh; int *table_out, *n_kv_out; long out_row; };
// grid (KV heads, rows): a workgroup copies one share in n_head_kv of the cut page's used slots, K and V; the first one also writes the row of the table.  Bound by memory: 256 rows with
// tables of 8192 slots and on average half a page of 256 slots each (8 heads of 128): 278 MB in 53 us, 5.2 TB/s; 4 rows: 3 us, the chain parent -> length -> page -> copy.
__global__ void __launch_bounds__(256) paged_fork_kernel(ForkArgs a) {
    const int h = blockIdx.x, i = blockIdx.y, p = a.parent[i];
    const bool live = (unsigned)p < (unsigned)a.c.n_seq && a.c.n_kv[(unsigned)p < (unsigned)a.c.n_seq ? p : 0] >= 0;
    const int n = live ? paged_len(a.c, p) : -1;
    const int full = live ? n >> a.c.page_shift : 0, used = live ? n & ((1 << a.c.page_shift) - 1) : 0;
    const int fresh = a.fresh[i], to = (unsigned)fresh < (unsigned)a.c.n_pages ? fresh : -1;
    if (h == 0) {
        int *row = a.table_out + (long)i * a.out_row;
        for (int w = threadIdx.x; w < a.c.W; w += 256) row[w] = w < full ? a.c.table[(long)p * a.c.table_row + w] : w == full && used ? to : -1;
        if (threadIdx.x == 0) a.n_kv_out[i] = n;
    }
    if (!used || to < 0) return;
    const int from = paged_page(a.c, p, full << a.c.page_shift);
    if (from < 0) return;
    // the workgroup's share of the page in the order of memory: K and V of a head's slots where those are neighbours, of a slot's heads where these are (token-major pages)
    const unsigned per_row = a.c.D / 8, share = used * per_row, first = h * share, heads = a.c.n_head_kv;
    const bool by_slot = a.c.k_head < a.c.k_row;
    const char *ks = a.c.k + (long)from * a.c.k_page, *vs = a.c.v + (long)from * a.c.v_page;
    char *kd = a.c.k + (long)to * a.c.k_page, *vd = a.c.v + (long)to * a.c.v_page;
    const int lg = a.c.D == 64 ? 3 : a.c.D == 128 ? 4 : 5;
#pragma unroll 4
    for (unsigned u = threadIdx.x; u < share; u += 256) {
        const unsigned at = (by_slot ? first + u : u) >> lg, d = (u & (per_row - 1)) * 16;          // (share is whole rows)
        const unsigned r = by_slot ? at / heads : at, hh = by_slot ? at - r * heads : (unsigned)h;
        const long ko = (long)hh * a.c.k_head + (long)r * a.c.k_row + d, vo = (long)hh * a.c.v_head + (long)r * a.c.v_row + d;
        const uint4 x = *reinterpret_cast<const uint4 *>(ks + ko), y = *reinterpret_cast<const uint4 *>(vs + vo);
        *reinterpret_cast<uint4 *>(kd + ko) = x; *reinterpret_cast<uint4 *>(vd + vo) = y;
    }
}
int cdna4_op_paged_fork(cdna4_context *ctx, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const int32_t *n_kv, const int32_t *parent,
                        const int32_t *fresh, const cdna4_tensor *table_out, int32_t *n_kv_out, void *stream) {
    ARG_CHECK(ctx && table_out, "paged_fork: null argument");
    PG_NORM(table_out, 4)
    ForkArgs a; int rc = pg_cache_check("paged_fork", k_cache, v_cache, table, true, &a.c); if (rc) return rc;
    ARG_CHECK(pg_sizes_ok(table_out) && table_out->type == CDNA4_TYPE_I32 && table_out->nb[0] == 4 && table_out->nb[1] % 4 == 0 && table_out->ne[0] == a.c.W && table_out->ne[2] == 1 &&
              table_out->ne[3] == 1 && pg_disjoint_elems(table_out, 4), "paged_fork: table_out i32 [W, n_out]");
    const long n_out = table_out->ne[1], n_seq = a.c.n_seq;
    OP_CHECK(n_out <= PAGED_MAX_SEQ, "paged_fork: at most %ld rows", PAGED_MAX_SEQ);
    if (n_out == 0) return CDNA4_OK;
    ARG_CHECK(n_seq > 0 && n_kv && parent && fresh && n_kv_out && ((a.c.table && table_out->data) || a.c.W == 0), "paged_fork: null data");
    const PgRange args[] = {pg_range("k_cache", k_cache, 2, true), pg_range("v_cache", v_cache, 2, true), pg_range("table_out", table_out, 4, true), pg_range("n_kv_out", n_kv_out, n_out * 4, true),
                            pg_range("table", table, 4, false), pg_range("n_kv", n_kv, n_seq * 4, false), pg_range("parent", parent, n_out * 4, false), pg_range("fresh", fresh, n_out * 4, false)};
    if ((rc = pg_apart("paged_fork", args, {0 * 16 + 1}))) return rc;
    ARG_CHECK(pg_kv_apart(k_cache, v_cache), "paged_fork: K and V share rows");
    a.c.n_kv = n_kv; a.parent = parent; a.fresh = fresh; a.table_out = (int *)table_out->data; a.n_kv_out = n_kv_out; a.out_row = table_out->nb[1] / 4;
    DEVICE_SCOPE(ctx);
    hipLaunchKernelGGL(paged_fork_kernel, dim3((unsigned)a.c.n_head_kv, (unsigned)n_out), dim3(256), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}

// ------------------------------------------------------------------------------------------------ evict
struct EvictArgs {
    PagedCache c; SlotView weight, pos, weight_out, pos_out; const int *n_past; int *n_kv_out; int budget, sink, recent, in_place, list;        // list: ints per (sequence, head) in `moves`
    int *moves;                                                                                                                           // [count, from[max], to[max]]
};
// sort key of a slot: larger = kept first.  Held slots above everything, then the order of the floats (-0 as 0, NaN as -inf)
static __device__ __forceinline__ uint32_t evict_key(float w, int p, int sink, int recent_from) {
    const uint32_t b = __float_as_uint(fmaxf(w + 0.0f, -INFINITY)), key = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return p < sink || p >= recent_from ? 0xffffffffu : key;
}
// One workgroup per (sequence, KV head): a chain of dependent steps over n slots, so what counts is that weight and pos are read from memory once, that many of their bytes are under way at
// a time and that the steps are few and short.
// * The first pass (16 bytes a lane) turns weight and pos into keys in LDS (up to 32768; a longer row computes them again in every pass: 130000 slots cut to 100: 80 us) and copies what lies before the budget to
//   weight_out / pos_out: of those slots the freed ones are written again by the moves.
// * The budget-th largest key by digits of 11, 11 and 10 bits, the first counted while the keys are made.  Two copies of the histogram by lane parity: weights share few leading digits and
//   adds to one address follow one another.  As soon as all keys of the bin in question are kept the search is over: with weights that differ, after the second digit.
// * Slots in order: every wave owns a contiguous range, counts its holes (freed, before the budget) and movers (kept, behind it), and lists them behind those of the waves before it.  Ranks
//   among equals are taken only if not all keys that equal the last kept one are kept.
// * Few moves (`here`: at most EVICT_HERE a row, as when a cache is cut back after every few tokens) are made in the same launch from lists in LDS; otherwise the lists go to memory and a
//   second launch moves the rows with the whole chip.
// Measured: 128 rows of up to 4160 slots cut to 4096: one launch of 10.2 us (reading 3, digits 2.4, lists 2, moves 2).  32 rows of up to 32768 slots cut to 4096: 23 us (reading 6, digits 5,
// lists 7: the vector instructions of 32 of the 256 CUs, some 20 for every slot in each) and 26 - 27 us for the moves (108 MB, 4.1 TB/s).
constexpr int EVICT_THREADS = 1024, EVICT_WAVES = 16, EVICT_KEYS = 32768, EVICT_HERE = 128, EVICT_BINS = 2048, EVICT_COPIES = 2;
static __device__ __forceinline__ void evict_move(const EvictArgs &a, int s, int h, int from, int to, int sub) {          // 16 lanes to a row: K, V, weight and pos
    if (sub == 0) {
        slot_row<float>(a.weight_out, s, h)[to] = slot_row<const float>(a.weight, s, h)[from];
        slot_row<int>(a.pos_out, s, h)[to] = slot_row<const int>(a.pos, s, h)[from];
    }
    const int pf = paged_page(a.c, s, from), pt = paged_page(a.c, s, to);
    if (pf < 0 || pt < 0) return;
    const int mask = (1 << a.c.page_shift) - 1;
    const char *ks = a.c.k + (long)pf * a.c.k_page + (long)h * a.c.k_head + (long)(from & mask) * a.c.k_row, *vs = a.c.v + (long)pf * a.c.v_page + (long)h * a.c.v_head + (long)(from & mask) * a.c.v_row;
    char *kd = a.c.k + (long)pt * a.c.k_page + (long)h * a.c.k_head + (long)(to & mask) * a.c.k_row, *vd = a.c.v + (long)pt * a.c.v_page + (long)h * a.c.v_head + (long)(to & mask) * a.c.v_row;
    for (int d = sub * 16; d < a.c.D * 2; d += 256) {
        const uint4 x = *reinterpret_cast<const uint4 *>(ks + d), y = *reinterpret_cast<const uint4 *>(vs + d);
        *reinterpret_cast<uint4 *>(kd + d) = x; *reinterpret_cast<uint4 *>(vd + d) = y;
    }
}
struct __attribute__((packed, aligned(4))) F4u { float v[4]; };          // rows of weight / pos begin at any multiple of 4 bytes
struct __attribute__((packed, aligned(4))) I4u { int v[4]; };
// inclusive sum over the lanes of a wave (DPP: shifts inside rows of 16, then the rows' last lanes broadcast)
static __device__ __forceinline__ unsigned wave_scan(unsigned v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true); v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true); v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false); v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
// sum of the totals of the waves before this one
static __device__ __forceinline__ unsigned waves_before(const unsigned (&tot)[EVICT_WAVES], int wave) {
    unsigned b = 0;
#pragma unroll
    for (int i = 0; i < EVICT_WAVES - 1; ++i) b += i < wave ? tot[i] : 0u;
    return b;
}
template <bool HERE> __global__ void __launch_bounds__(EVICT_THREADS) paged_evict_select_kernel(EvictArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t s_key[];
    __shared__ unsigned hist[EVICT_BINS * EVICT_COPIES], tot[3][EVICT_WAVES], s_digit, s_rest, s_equal; __shared__ int s_moves[HERE ? 2 * EVICT_HERE : 1];
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int raw = a.c.n_kv[s], n = paged_len(a.c, s), most = (a.list - 1) / 2;
    const int recent_from = (int)max((long)a.n_past[s] - a.recent, -(1l << 31));
    int *moves = HERE ? nullptr : a.moves + ((long)s * a.c.n_head_kv + h) * a.list;
    const float *w = slot_row<const float>(a.weight, s, h); const int *p = slot_row<const int>(a.pos, s, h);
    float *wo = slot_row<float>(a.weight_out, s, h); int *po = slot_row<int>(a.pos_out, s, h);
    if (h == 0 && tid == 0) a.n_kv_out[s] = raw < 0 ? raw : min(n, a.budget);
    const bool over = n > a.budget, in_lds = n <= EVICT_KEYS;
    if (!over && (a.in_place || n == 0)) { if (!HERE && tid == 0) moves[0] = 0; return; }
    auto zero = [&]() {
        for (int i = tid * 4; i < EVICT_BINS * EVICT_COPIES; i += EVICT_THREADS * 4) *reinterpret_cast<uint4 *>(hist + i) = make_uint4(0u, 0u, 0u, 0u);
    };
    auto count_digit = [&](uint32_t digit) { atomicAdd(&hist[digit * EVICT_COPIES + (lane & (EVICT_COPIES - 1))], 1u); };
    zero();
    __syncthreads();
    auto take = [&](float x, int y) { const uint32_t k = evict_key(x, y, a.sink, recent_from); count_digit(k >> 21); return k; };
#pragma unroll 4
    for (int j = 4 * tid; j < n - 3; j += 4 * EVICT_THREADS) {
        const F4u x = *reinterpret_cast<const F4u *>(w + j); const I4u y = *reinterpret_cast<const I4u *>(p + j);
        if (over) {
            uint4 k; k.x = take(x.v[0], y.v[0]); k.y = take(x.v[1], y.v[1]); k.z = take(x.v[2], y.v[2]); k.w = take(x.v[3], y.v[3]);
            if (in_lds) *reinterpret_cast<uint4 *>(s_key + j) = k;
        }
        if (!a.in_place) {
            if (j + 4 <= a.budget) { *reinterpret_cast<F4u *>(wo + j) = x; *reinterpret_cast<I4u *>(po + j) = y; }
            else for (int i = 0; i < 4; ++i) if (j + i < a.budget) { wo[j + i] = x.v[i]; po[j + i] = y.v[i]; }
        }
    }
    if (tid < (n & 3)) {
        const int j = (n & ~3) + tid; const float x = w[j]; const int y = p[j];
        if (over) { const uint32_t k = take(x, y); if (in_lds) s_key[j] = k; }
        if (!a.in_place && j < a.budget) { wo[j] = x; po[j] = y; }
    }
    if (!over) { if (!HERE && tid == 0) moves[0] = 0; return; }
    __syncthreads();
    // the keys of slots j ... j + 3 (j a multiple of 4; what lies behind the row's end is anything)
    auto keys4 = [&](int j) {
        if (in_lds) return *reinterpret_cast<const uint4 *>(s_key + j);
        const int at = min(j, n - 4), off = j - at;          // (a row that is not in LDS has more than 4 slots; at its end the last four are read and shifted down)
        F4u x = *reinterpret_cast<const F4u *>(w + at); I4u y = *reinterpret_cast<const I4u *>(p + at);
        if (off & 1) { x.v[0] = x.v[1]; x.v[1] = x.v[2]; x.v[2] = x.v[3]; y.v[0] = y.v[1]; y.v[1] = y.v[2]; y.v[2] = y.v[3]; }
        if (off & 2) { x.v[0] = x.v[2]; x.v[1] = x.v[3]; y.v[0] = y.v[2]; y.v[1] = y.v[3]; }
        auto one = [&](int i) { return evict_key(x.v[i], y.v[i], a.sink, recent_from); };
        return make_uint4(one(0), one(1), one(2), one(3));
    };
    uint32_t prefix = 0, rest = (uint32_t)a.budget; bool all_equal = false;         // the budget-th largest key lies among those that equal `prefix` so far; `rest` of them are kept
    for (int shift = 21; ; shift = max(shift - 11, 0)) {                            // bits [21, 32), [10, 21), [0, 10)
        const int width = shift ? 11 : 10;
        if (shift < 21) {
            const int high = shift + width; const uint32_t want = prefix >> high, mask = (1u << width) - 1;
#pragma unroll 4
            for (int j = 4 * tid; j < n; j += 4 * EVICT_THREADS) {
                const uint4 k = keys4(j); const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) if ((x[i] >> high) == want && j + i < n) count_digit((x[i] >> shift) & mask);
            }
            __syncthreads();
        }
        // two bins a thread, from the top bin down
        const int bin = EVICT_BINS - 2 - 2 * tid; const uint4 c4 = *reinterpret_cast<const uint4 *>(hist + bin * EVICT_COPIES);
        const unsigned hi = c4.z + c4.w, lo = c4.x + c4.y;
        unsigned above = wave_scan(hi + lo);
        if (lane == 63) tot[0][wave] = above;
        __syncthreads();
        above += waves_before(tot[0], wave) - (hi + lo);
        if (above < rest && above + hi >= rest) { s_digit = bin + 1; s_rest = rest - above; s_equal = hi; }
        else if (above + hi < rest && above + hi + lo >= rest) { s_digit = bin; s_rest = rest - above - hi; s_equal = lo; }
        zero();
        __syncthreads();
        prefix |= s_digit << shift; rest = s_rest; all_equal = s_equal == rest;
        if (all_equal || shift == 0) break;
    }
    // kept: every key >= prefix if all of the last bin are kept, otherwise (the whole key is in prefix) the larger ones and the first `rest` of the equal ones
    const int span = ((n + EVICT_WAVES - 1) / EVICT_WAVES + 255) & ~255, j0 = min(wave * span, n), j1 = min(j0 + span, n);
    unsigned tie0 = 0;
    if (!all_equal) {                                       // (uniform)
        unsigned ties = 0;
        for (int j = j0 + 4 * lane; j < j1; j += 256) {
            const uint4 k = keys4(j); const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) ties += x[i] == prefix && j + i < j1;
        }
        ties = wave_scan(ties);
        if (lane == 63) tot[1][wave] = ties;
        __syncthreads();
        tie0 = waves_before(tot[1], wave);
        __syncthreads();
    }
    // four slots to a lane, 256 to a step; holes and movers counted in the halves of one number.  First round: how many has the wave; second: where they go
    unsigned holes = 0, movers = 0;
    for (int round = 0; round < 2; ++round) {
        unsigned t = tie0, found = 0, lane_holes = 0, lane_movers = 0;
        for (int b = j0; b < j1; b += 256) {
            const int j = b + 4 * lane; const uint4 k = keys4(min(j, (n - 1) & ~3)); const uint32_t x[4] = {k.x, k.y, k.z, k.w};
            unsigned keep = 0, in = 15u;
#pragma unroll
            for (int i = 3; i >= 0; --i) keep = 2 * keep + (x[i] >= prefix);
            if (b + 256 > j1) in = j1 >= j + 4 ? 15u : j1 <= j ? 0u : (1u << (j1 - j)) - 1;
            if (!all_equal) {
                unsigned tie = 0;
#pragma unroll
                for (int i = 3; i >= 0; --i) tie = 2 * tie + (x[i] == prefix);
                tie &= in;
                const unsigned mine = __popc(tie), upto = wave_scan(mine);
                unsigned r = t + upto - mine;
#pragma unroll
                for (int i = 0; i < 4; ++i) if ((tie >> i) & 1) { if (r >= rest) keep &= ~(1u << i); ++r; }
                t += (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
            }
            const unsigned before = b + 256 <= a.budget ? 15u : b >= a.budget ? 0u : a.budget >= j + 4 ? 15u : a.budget <= j ? 0u : (1u << (a.budget - j)) - 1;      // the lane's slots before the budget
            const unsigned hole = in & ~keep & before, mover = in & keep & ~before, c = __popc(hole) | (__popc(mover) << 16);
            if (!round) { lane_holes += c & 0xffffu; lane_movers += c >> 16; continue; }
            const unsigned upto = wave_scan(c), at = found + upto - c;
            if (c) {
                int *list = HERE ? s_moves : moves + 1; const int half = HERE ? EVICT_HERE : most;
                unsigned nh = half + holes + (at & 0xffffu), nm = movers + (at >> 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) { if ((hole >> i) & 1) list[nh++] = j + i; if ((mover >> i) & 1) list[nm++] = j + i; }
            }
            found += (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
            if (!in_lds) { holes += found & 0xffffu; movers += found >> 16; found = 0; }          // (a long row's wave may have more than 2^16 of either)
        }
        if (!round) {
            const unsigned nh = wave_scan(lane_holes), nm = wave_scan(lane_movers);
            if (lane == 63) { tot[1][wave] = nh; tot[2][wave] = nm; }
            __syncthreads();
            holes = waves_before(tot[1], wave); movers = waves_before(tot[2], wave);
        }
    }
    if constexpr (HERE) {
        __syncthreads();
        int count = 0;
#pragma unroll
        for (int i = 0; i < EVICT_WAVES; ++i) count += (int)tot[2][i];
        for (int m = tid >> 4; m < count; m += EVICT_THREADS / 16) evict_move(a, s, h, s_moves[m], s_moves[EVICT_HERE + m], tid & 15);
    } else if (tid == EVICT_THREADS - 1) moves[0] = (int)(waves_before(tot[2], EVICT_WAVES - 1) + tot[2][EVICT_WAVES - 1]);
}
// grid (chunks of moves, KV heads, sequences): bound by memory
__global__ void __launch_bounds__(256) paged_evict_move_kernel(EvictArgs a) {
    const int h = blockIdx.y, s = blockIdx.z;
    const int *moves = a.moves + ((long)s * a.c.n_head_kv + h) * a.list; const int count = moves[0], most = (a.list - 1) / 2;
    for (int m = blockIdx.x * 16 + (threadIdx.x >> 4); m < count; m += gridDim.x * 16) evict_move(a, s, h, moves[1 + m], moves[1 + most + m], threadIdx.x & 15);
}
// at most this many rows of a (sequence, head) move: a mover lies behind the budget, a hole before it
static long evict_most(const PagedCache &c, int budget) { return std::min<long>(budget, std::max<long>(((long)c.W << c.page_shift) - budget, 0)); }
static int64_t evict_check(const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *pos, int budget, int n_sink,
                           int n_recent, const cdna4_tensor *weight_out, const cdna4_tensor *pos_out, EvictArgs *a) {
    ARG_CHECK(weight && pos && weight_out && pos_out, "paged_evict: null argument");
    int rc = pg_cache_check("paged_evict", k_cache, v_cache, table, true, &a->c); if (rc) return rc;
    if ((rc = pg_slots_check("paged_evict", "weight", weight, CDNA4_TYPE_F32, a->c, false)) || (rc = pg_slots_check("paged_evict", "pos", pos, CDNA4_TYPE_I32, a->c, false)) ||
        (rc = pg_slots_check("paged_evict", "weight_out", weight_out, CDNA4_TYPE_F32, a->c, true)) || (rc = pg_slots_check("paged_evict", "pos_out", pos_out, CDNA4_TYPE_I32, a->c, true))) return rc;
    ARG_CHECK(budget >= 1 && n_sink >= 0 && n_recent >= 0 && (long)n_sink + n_recent <= budget, "paged_evict: 1 <= budget, 0 <= n_sink + n_recent <= budget");
    const bool ws = pg_same(weight, weight_out), ps = pg_same(pos, pos_out);
    ARG_CHECK(pg_empty(weight) || (ws == ps && (ws || (!pg_overlap(weight, 4, weight_out, 4) && !pg_overlap(pos, 4, pos_out, 4))) && !pg_overlap(weight_out, 4, pos, 4) &&
              !pg_overlap(pos_out, 4, weight, 4) && !pg_overlap(weight_out, 4, pos_out, 4)), "paged_evict: weight_out and pos_out are weight and pos themselves, or memory apart from both");
    a->in_place = ws; a->budget = budget; a->sink = n_sink; a->recent = n_recent; a->list = (int)(1 + 2 * evict_most(a->c, budget));
    return (int64_t)a->c.n_seq * a->c.n_head_kv * a->list * 4;
}
int64_t cdna4_paged_evict_workspace(const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *pos, int budget, int n_sink,
                                    int n_recent, const cdna4_tensor *weight_out, const cdna4_tensor *pos_out) {
    PG_NORM(weight, 4) PG_NORM(pos, 4) PG_NORM(weight_out, 4) PG_NORM(pos_out, 4)
    EvictArgs a; return evict_check(k_cache, v_cache, table, weight, pos, budget, n_sink, n_recent, weight_out, pos_out, &a);
}
int cdna4_op_paged_evict(cdna4_context *ctx, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const int32_t *n_kv, const cdna4_tensor *weight,
                         const cdna4_tensor *pos, const int32_t *n_past, int budget, int n_sink, int n_recent, const cdna4_tensor *weight_out, const cdna4_tensor *pos_out, int32_t *n_kv_out, void *stream) {
    ARG_CHECK(ctx, "paged_evict: null argument");
    PG_NORM(weight, 4) PG_NORM(pos, 4) PG_NORM(weight_out, 4) PG_NORM(pos_out, 4)
    EvictArgs a; const int64_t bytes = evict_check(k_cache, v_cache, table, weight, pos, budget, n_sink, n_recent, weight_out, pos_out, &a); if (bytes < 0) return (int)bytes;
    if (a.c.n_seq == 0) return CDNA4_OK;
    const long n = a.c.n_seq;
    ARG_CHECK(n_kv && n_past && n_kv_out && (a.c.W == 0 || (a.c.table && weight->data && pos->data && weight_out->data && pos_out->data)), "paged_evict: null data");
    const PgRange args[] = {pg_range("k_cache", k_cache, 2, true), pg_range("v_cache", v_cache, 2, true), pg_range("weight_out", weight_out, 4, true), pg_range("pos_out", pos_out, 4, true),
                            pg_range("n_kv_out", n_kv_out, n * 4, true), pg_range("weight", weight, 4, false), pg_range("pos", pos, 4, false), pg_range("table", table, 4, false),
                            pg_range("n_kv", n_kv, n * 4, false), pg_range("n_past", n_past, n * 4, false)};
    int rc = pg_apart("paged_evict", args, {0 * 16 + 1, 2 * 16 + 5, 3 * 16 + 6});          // (in place or apart: evict_check)
    if (rc) return rc;
    ARG_CHECK(pg_kv_apart(k_cache, v_cache), "paged_evict: K and V share rows");
    a.c.n_kv = n_kv; a.n_past = n_past; a.n_kv_out = n_kv_out;
    a.weight = slot_view(weight); a.pos = slot_view(pos); a.weight_out = slot_view(weight_out); a.pos_out = slot_view(pos_out);
    DEVICE_SCOPE(ctx);
    if ((rc = cdna4_ensure_ws(ctx, (size_t)bytes, (hipStream_t)stream))) return rc;
    a.moves = (int *)ctx->ws;
    const long most = evict_most(a.c, budget);
    const dim3 grid((unsigned)a.c.n_head_kv, (unsigned)n); hipStream_t st = (hipStream_t)stream;
    const size_t lds = (size_t)std::min<long>((long)a.c.W << a.c.page_shift, EVICT_KEYS) * 4;
    if (most <= EVICT_HERE) {
        HIP_TRY(pg_opt_in_lds<paged_evict_select_kernel<true>>(ctx->device, EVICT_KEYS * 4));
        hipLaunchKernelGGL(paged_evict_select_kernel<true>, grid, dim3(EVICT_THREADS), lds, st, a);
        HIP_TRY(hipGetLastError()); return CDNA4_OK;
    }
    HIP_TRY(pg_opt_in_lds<paged_evict_select_kernel<false>>(ctx->device, EVICT_KEYS * 4));
    hipLaunchKernelGGL(paged_evict_select_kernel<false>, grid, dim3(EVICT_THREADS), lds, st, a);
    HIP_TRY(hipGetLastError());
    const unsigned gx = (unsigned)std::min<long>((most + 15) / 16, 64);
    hipLaunchKernelGGL(paged_evict_move_kernel, dim3(gx, (unsigned)a.c.n_head_kv, (unsigned)n), dim3(256), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}
