// beam.hip -- one step of a beam search: the best continuations over beams and vocabulary.
//
// The logits are read once (4 bytes a candidate against a handful of operations: bound by that read).  A workgroup takes 8192 (2048) neighbouring logits of a row into registers and leaves
// their maximum, the sum of their exponentials and their n_out best, sorted; a second launch joins a group's chunks: log sum exp of every beam, then the best of the sorted lists.
//
// Choosing the k best of many without sorting them: in a total order without ties, the k-th best of the threads' (or lanes' quads') own best elements is a bound that at least k elements
// reach, and every element that reaches it belongs to one of the k owners whose best does -- so the collected list is never longer than k shares, whatever the values, and in random order
// it is hardly longer than k.
#include "paged.cuh"
#include "fa_decode.cuh"
#include <algorithm>

typedef unsigned long long u64;
constexpr int BEAM_MAX_OUT = 64, BEAM_MAX_BEAMS = 256, BEAM_CHUNK = 8192; constexpr long BEAM_MAX_CANDS = 1l << 26;
constexpr int BEAM_MAX_LISTS = (int)(BEAM_MAX_CANDS / BEAM_CHUNK) + BEAM_MAX_BEAMS;

struct BeamArgs {
    const char *logits; long row; const float *score; const int *done; int n_beam, n_out, pad, n_vocab, chunk, chunks;          // chunk: logits of a workgroup
    float *score_out; int *parent, *token;
    float2 *stat; u64 *best;            // [rows][chunks] maximum and sum of exponentials; [rows][chunks][n_out] sorted keys (0: none)
};
// (logit descending, token ascending) as one number; NaN counts as -inf, both zeros are one
static __device__ __forceinline__ u64 logit_key(float x, int t) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return ((u64)(b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u)) << 32) | (uint32_t)~t;
}
static __device__ __forceinline__ float key_logit(u64 k) { const uint32_t b = (uint32_t)(k >> 32); return __uint_as_float(b ^ ((b & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }
static __device__ __forceinline__ int key_token(u64 k) { return (int)~(uint32_t)k; }
static __device__ __forceinline__ u64 shfl_max(u64 k, int d) {
    const u64 o = ((u64)(uint32_t)__shfl_xor((int)(k >> 32), d, 64) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)k, d, 64);
    return o > k ? o : k;
}
struct __attribute__((packed, aligned(4))) F4a4 { float x, y, z, w; };          // rows begin at any multiple of 4 bytes

// EPT logits a thread.  Owners of the bound: quads of lanes (64) for n_out <= 16, single threads above; the list holds n_out shares of either.
template <int EPT> __global__ void __launch_bounds__(256) beam_scan_kernel(BeamArgs a) {
    __shared__ u64 s_own[256], s_list[BEAM_MAX_OUT * EPT]; __shared__ float s_red[8]; __shared__ u64 s_bound; __shared__ int s_n;
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, base = blockIdx.x * 256 * EPT;
    const float *x = reinterpret_cast<const float *>(a.logits + (long)r * a.row) + base;
    const int n = min(256 * EPT, a.n_vocab - base);
    float v[EPT];
    if (n == 256 * EPT) {
#pragma unroll
        for (int e = 0; e < EPT / 4; ++e) { const F4a4 f = reinterpret_cast<const F4a4 *>(x)[e * 256 + tid]; v[4 * e] = f.x; v[4 * e + 1] = f.y; v[4 * e + 2] = f.z; v[4 * e + 3] = f.w; }
    } else {
#pragma unroll
        for (int e = 0; e < EPT; ++e) v[e] = x[min((e / 4 * 256 + tid) * 4 + e % 4, n - 1)];
    }
    auto index = [&](int e) { return (e / 4 * 256 + tid) * 4 + e % 4; };
    // the thread's best (the lowest index of equals: strictly larger ones replace it) and the chunk's maximum
    float top = -INFINITY; u64 own = 0;
    int at = -1;
#pragma unroll
    for (int e = 0; e < EPT; ++e) { const bool in = index(e) < n; if (in && (v[e] > top || at < 0)) { at = e; } top = in ? fmaxf(top, v[e]) : top; }
    // (a NaN first element does not hold its place against numbers: v > top then compares with -inf or with what followed)
#pragma unroll
    for (int e = 0; e < EPT; ++e) if (e == at) own = logit_key(v[e], base + index(e));
    const float wm = wave_max(top);
    if (lane == 0) s_red[wave] = wm;
    if (tid == 0) { s_bound = 0; s_n = 0; }
    const bool quads = a.n_out <= 16;
    if (quads) { own = shfl_max(shfl_max(own, 1), 2); if ((lane & 3) == 0) s_own[tid >> 2] = own; } else s_own[tid] = own;
    __syncthreads();
    const float m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    if (!quads || tid < 64) {          // the owner with n_out - 1 better ones before it
        const u64 mine = s_own[tid]; int rank = 0; const int owners = quads ? 64 : 256;
#pragma unroll 8
        for (int i = 0; i < owners; ++i) rank += s_own[i] > mine;
        if (rank == a.n_out - 1 && mine) s_bound = mine;          // (fewer owners than n_out: the bound stays 0, everything is listed)
    }
    float l = 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) if (index(e) < n) l += m != -INFINITY ? __builtin_amdgcn_exp2f((v[e] - m) * 1.44269504088896341f) : v[e] != v[e] ? v[e] : 0.f;       // (NaN stays in the sum)
    l = wave_sum_dpp(l);
    if (lane == 0) s_red[4 + wave] = l;
    __syncthreads();
    const u64 bound = s_bound;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
        const u64 k = logit_key(v[e], base + index(e));
        if (index(e) < n && k >= bound) s_list[atomicAdd(&s_n, 1)] = k;
    }
    __syncthreads();
    const int count = s_n; const long row = (long)r * a.chunks + blockIdx.x;
    if (tid == 0) a.stat[row] = make_float2(m, (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]));
    for (int i = tid; i < count; i += 256) {
        const u64 mine = s_list[i]; int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) rank += s_list[j] > mine;
        if (rank < a.n_out) a.best[row * a.n_out + rank] = mine;
    }
    for (int i = count + tid; i < a.n_out; i += 256) a.best[row * a.n_out + i] = 0;
}

// a candidate of a group: value descending, then beam, logit descending, token (within a beam the value grows with the logit, in 64 bits not always visibly).  b < 0: none
struct Cand { double c; u64 key; int b; };
static __device__ __forceinline__ bool before(const Cand &p, const Cand &q) {
    if ((p.b < 0) != (q.b < 0)) return q.b < 0;
    if (p.c != q.c) return p.c > q.c;
    if (p.b != q.b) return p.b < q.b;
    return p.key > q.key;
}
struct Cands { double c[BEAM_MAX_OUT * ((BEAM_MAX_LISTS + 255) / 256)]; u64 key[BEAM_MAX_OUT * ((BEAM_MAX_LISTS + 255) / 256)]; int b[BEAM_MAX_OUT * ((BEAM_MAX_LISTS + 255) / 256)]; };
// how many of c[0 .. n) come before `p`: one comparison of doubles each, the rest of the order only where two are equal
template <typename C> static __device__ __forceinline__ int rank_among(const C &s, int n, const Cand &p) {
    int above = 0, same = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) { const double c = s.c[i]; above += c > p.c; same += c == p.c; }
    if (same > 1) {
        above = 0;
        for (int i = 0; i < n; ++i) { const Cand q = {s.c[i], s.key[i], s.b[i]}; above += before(q, p); }
    }
    return above;
}
struct Own { double c[256]; u64 key[256]; int b[256]; };
// the k best of get(0 .. n), sorted, into out (LDS); returns how many there are.  n <= 256 * the share that Cands is made for.
template <typename F> static __device__ __forceinline__ int choose(int n, int k, F get, Cand *out, Own &own, Cands &list, int *s_n, Cand *s_bound) {
    const int tid = threadIdx.x;
    Cand best = {-INFINITY, 0, -1};
    for (int i = tid; i < n; i += 256) { const Cand q = get(i); if (before(q, best)) best = q; }
    __syncthreads();
    own.c[tid] = best.c; own.key[tid] = best.key; own.b[tid] = best.b;
    if (tid == 0) { *s_n = 0; *s_bound = {-INFINITY, 0, 0x7fffffff}; }
    __syncthreads();
    if (best.b >= 0 && rank_among(own, 256, best) == k - 1) *s_bound = best;
    __syncthreads();
    const Cand bound = *s_bound;
    for (int i = tid; i < n; i += 256) {
        const Cand q = get(i);
        if (q.b >= 0 && !before(bound, q)) { const int p = atomicAdd(s_n, 1); list.c[p] = q.c; list.key[p] = q.key; list.b[p] = q.b; }
    }
    __syncthreads();
    const int count = *s_n;
    for (int i = tid; i < count; i += 256) { const Cand q = {list.c[i], list.key[i], list.b[i]}; const int rank = rank_among(list, count, q); if (rank < k) out[rank] = q; }
    __syncthreads();
    return min(count, k);
}
// One workgroup per group.  Only the n_out lists with the best heads can hold any of the n_out best, and of the list with rank r among them only its first n_out - r entries.
__global__ void __launch_bounds__(256) beam_join_kernel(BeamArgs a) {
    __shared__ double s_top[BEAM_MAX_BEAMS], s_lse[BEAM_MAX_BEAMS]; __shared__ float s_score[BEAM_MAX_BEAMS]; __shared__ int s_kind[BEAM_MAX_BEAMS];       // 0: logits, 1: finished, 2: nothing but -inf
    __shared__ Own own; __shared__ Cands list; __shared__ Cand s_heads[BEAM_MAX_OUT], s_best[BEAM_MAX_OUT], s_bound; __shared__ int s_n;
    const int g = blockIdx.x, tid = threadIdx.x, k = a.n_out;
    // 16 lanes to a beam
    for (int b0 = 0; b0 < a.n_beam; b0 += 16) {
        const int b = b0 + (tid >> 4), r = g * a.n_beam + min(b, a.n_beam - 1);
        float m = -INFINITY, l = 0.f;
        for (int c = tid & 15; c < a.chunks; c += 16) m = fmaxf(m, a.stat[(long)r * a.chunks + c].x);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        for (int c = tid & 15; c < a.chunks; c += 16) { const float2 s = a.stat[(long)r * a.chunks + c]; l += s.x == m ? s.y : s.y * __builtin_amdgcn_exp2f((s.x - m) * 1.44269504088896341f); }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) l += __shfl_xor(l, d, 64);
        if ((tid & 15) == 0 && b < a.n_beam) {
            const float score = a.score[r]; const bool done = a.done && a.done[r];
            s_top[b] = m; s_lse[b] = log((double)l); s_score[b] = score;
            const bool none = score != score || score == -INFINITY || (!done && (l != l || m == INFINITY || m == -INFINITY));
            s_kind[b] = none ? 2 : done ? 1 : 0;
        }
    }
    __syncthreads();
    const int per_row = min(k, a.n_vocab);
    // entry e of list (beam, chunk); finished beams and those of nothing have one list, made here: pad first if it counts, then tokens of -inf by their index
    auto entry = [&](int l, int e) {
        Cand q = {-INFINITY, 0, -1};
        const int b = l / a.chunks, c = l - b * a.chunks, kind = s_kind[b];
        if (kind == 0) {
            q.key = a.best[((long)(g * a.n_beam + b) * a.chunks + c) * k + e];
            if (q.key) {
                q.b = b;
                const float x = key_logit(q.key);
                q.c = (double)s_score[b] + (((double)x - s_top[b]) - s_lse[b]);
                if (x == -INFINITY || q.c != q.c) q.c = -INFINITY;
            }
        } else if (c == 0 && e < per_row) {
            const int t = kind == 2 ? e : e == 0 ? a.pad : e - 1 < a.pad ? e - 1 : e;
            q.b = b; q.key = logit_key(-INFINITY, t); q.c = kind == 1 && e == 0 ? (double)s_score[b] : -INFINITY;
        }
        return q;
    };
    const int lists = a.n_beam * a.chunks;
    const int heads = choose(lists, k, [&](int i) { return entry(i, 0); }, s_heads, own, list, &s_n, &s_bound);
    auto list_of = [&](const Cand &q) {          // the chunk of a head is where its token lies
        return q.b * a.chunks + (s_kind[q.b] ? 0 : key_token(q.key) / a.chunk);
    };
    const int total = k * (k + 1) / 2;
    const int found = choose(total, k, [&](int i) {
        int r = (int)((sqrtf(8.0f * i + 1.0f) - 1.0f) * 0.5f);          // i = r (r + 1) / 2 + e: entry e of the list with rank k - 1 - r has e <= r
        while (r * (r + 1) / 2 > i) --r;
        while ((r + 1) * (r + 2) / 2 <= i) ++r;
        const int e = i - r * (r + 1) / 2, h = k - 1 - r;
        return h < heads ? entry(list_of(s_heads[h]), e) : Cand{-INFINITY, 0, -1};
    }, s_best, own, list, &s_n, &s_bound);
    for (int i = tid; i < found; i += 256) {
        const Cand q = s_best[i]; const long o = (long)g * k + i;
        a.score_out[o] = (float)q.c; a.parent[o] = g * a.n_beam + q.b; a.token[o] = key_token(q.key);
    }
}
static int64_t beam_check(const cdna4_tensor *x, int n_beam, int n_out, int pad, BeamArgs *a) {
    ARG_CHECK(x, "beam_select: null argument");
    ARG_CHECK(pg_sizes_ok(x) && x->type == CDNA4_TYPE_F32 && x->ne[0] >= 1 && x->ne[2] == 1 && x->ne[3] == 1, "beam_select: logits f32 [n_vocab, n_group * n_beam]");
    OP_CHECK(x->nb[0] == 4 && x->nb[1] % 4 == 0 && (uintptr_t)x->data % 4 == 0, "beam_select: dense rows");
    OP_CHECK(n_beam >= 1 && n_beam <= BEAM_MAX_BEAMS && x->ne[0] * n_beam <= BEAM_MAX_CANDS && x->ne[1] <= 65535, "beam_select: 1 to 256 beams, n_beam * n_vocab <= 2^26, at most 65535 rows");
    ARG_CHECK(x->ne[1] % n_beam == 0, "beam_select: rows are groups of n_beam");
    OP_CHECK(n_out >= 1 && n_out <= BEAM_MAX_OUT && n_out <= x->ne[0] * n_beam, "beam_select: 1 <= n_out <= min(64, n_beam * n_vocab)");
    ARG_CHECK(pad >= 0 && pad < x->ne[0], "beam_select: pad is a token");
    a->logits = (const char *)x->data; a->row = x->nb[1]; a->n_vocab = (int)x->ne[0]; a->n_beam = n_beam; a->n_out = n_out; a->pad = pad;
    // 2048 logits to a workgroup where 8192 would leave most of the chip idle (fewer than 256 workgroups)
    a->chunk = x->ne[1] * ((x->ne[0] + BEAM_CHUNK - 1) / BEAM_CHUNK) < 256 ? BEAM_CHUNK / 4 : BEAM_CHUNK;
    a->chunks = (a->n_vocab + a->chunk - 1) / a->chunk;
    return x->ne[1] * a->chunks * (8 + 8 * (int64_t)n_out);
}
int64_t cdna4_beam_select_workspace(const cdna4_tensor *logits, int n_beam, int n_out, int pad) { BeamArgs a; return beam_check(logits, n_beam, n_out, pad, &a); }
int cdna4_op_beam_select(cdna4_context *ctx, const cdna4_tensor *logits, const float *score, const int32_t *done, int n_beam, int n_out, int pad, float *score_out, int32_t *parent, int32_t *token,
                         void *stream) {
    ARG_CHECK(ctx, "beam_select: null argument");
    BeamArgs a; const int64_t bytes = beam_check(logits, n_beam, n_out, pad, &a); if (bytes < 0) return (int)bytes;
    const long rows = logits->ne[1], out = rows / n_beam * n_out * 4;
    if (rows == 0) return CDNA4_OK;
    ARG_CHECK(logits->data && score && score_out && parent && token, "beam_select: null data");
    const void *outs[3] = {score_out, parent, token}; const void *ins[3] = {logits->data, score, done}; const long in_bytes[3] = {pg_extent(logits, 4), rows * 4, rows * 4};
    for (int i = 0; i < 3; ++i) for (int j = 0; j < 3; ++j)
        ARG_CHECK(!pg_overlap(outs[i], out, ins[j], in_bytes[j]) && (i == j || !pg_overlap(outs[i], out, outs[j], out)), "beam_select: an output overlaps another argument");
    a.score = score; a.done = done; a.score_out = score_out; a.parent = parent; a.token = token;
    DEVICE_SCOPE(ctx);
    const int rc = cdna4_ensure_ws(ctx, (size_t)bytes, (hipStream_t)stream); if (rc) return rc;
    a.stat = (float2 *)ctx->ws; a.best = (u64 *)(a.stat + rows * a.chunks);
    hipStream_t st = (hipStream_t)stream; const dim3 grid((unsigned)a.chunks, (unsigned)rows);
    if (a.chunk == BEAM_CHUNK) hipLaunchKernelGGL(beam_scan_kernel<32>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(beam_scan_kernel<8>, grid, dim3(256), 0, st, a);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)(rows / n_beam)), dim3(256), 0, st, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}
