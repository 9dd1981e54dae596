// beam.hip -- one step of a beam search: the best continuations over beams and vocabulary.
//
// The logits are read once (4 bytes a candidate against a handful of operations: bound by that read).  A workgroup takes 8192 (2048) neighbouring logits of a row into registers and leaves
// their maximum, the sum of their exponentials and their n_out best, sorted; a second launch joins a group's chunks: log sum exp of every beam, then the best of the sorted lists.
// The exponentials and their sums are 64 bits wide: candidates of different beams are ordered by values in which those sums stand, and 32 bits mixed up what differs by less than 10^-6
// (32 bits took 35.3 us for 256 rows of 128256, 131 MB, 32 groups of 8, 16 results; so it takes 47.8).  Medians of the launches: 39 us for the chunks, which are bound by 12 64-bit instructions
// a logit, and 9 us for the join; 4 rows of 32000: 4.5 and 5.3 us.
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

struct BeamStat { double sum; float top; };
struct BeamArgs {
    const char *logits; long row; const float *score; const int *done; int n_beam, n_out, pad, n_vocab, chunk, chunks;          // chunk: logits of a workgroup
    float *score_out; int *parent, *token;
    struct BeamStat *stat; u64 *best;   // [rows][chunks] maximum and sum of exponentials; [rows][chunks][n_out] sorted keys (0: none)
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
// e^x of a difference of two f32 values, x <= 0, in 64 bits: 2^(k / 16) from a table of 16 in LDS (one bank pair each) with k >> 4 added to the exponent, times the Taylor polynomial of
// 2^(r / 16), |r| <= 1/2, up to the fifth power (remainder (ln 2 / 32)^6 / 720 = 1.4 * 10^-13).  x below -700 counts as -700 (10^-304); NaN too, so the caller looks for those.
static __device__ __forceinline__ double exp_below(double x, const double *pow16) {
    constexpr double SCALE = 23.083120654223414, WHOLE = 6755399441055744.0, C = 0.043321698784996585;          // 16 / ln 2; 1.5 * 2^52 (adding it rounds to whole numbers, into the low bits); ln 2 / 16
    x = __builtin_fmax(x, -700.0);
    const double y = fma(x, SCALE, WHOLE), r = fma(x, SCALE, WHOLE - y);
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, y);
    const double p = fma(r, fma(r, fma(r, fma(r, fma(r, C * C * C * C * C / 120, C * C * C * C / 24), C * C * C / 6), C * C / 2), C), 1.0);
    return p * __builtin_bit_cast(double, __builtin_bit_cast(u64, pow16[k & 15]) + ((u64)(uint32_t)(k >> 4) << 52));
}
struct __attribute__((packed, aligned(4))) F4a4 { float x, y, z, w; };          // rows begin at any multiple of 4 bytes

// EPT logits a thread.  Owners of the bound: quads of lanes (64) for n_out <= 16, single threads above; the list holds n_out shares of either.
// The bound is first taken on values alone, which costs a maximum and a comparison per logit (with keys of value and index all through, the launch was bound by its vector instructions:
// 45 us for 256 rows of 128256, 131 MB), and from every wave a quarter of n_out (one bound of the workgroup for 64 results took as long as the rest: 480 rows of 70000: 48 us, so 38).  Ties at
// the bound can make that list too long, and a bound of -inf says nothing: then the keys decide.  A row's last chunk takes its logits one at a time, coalesced (as quads of which the last were
// cut lane by lane, those chunks ended last: 29 us in all for the 131 MB, so 24).  (These figures: with sums of 32 bits.)
template <int EPT> __global__ void __launch_bounds__(256) beam_scan_kernel(BeamArgs a) {
    constexpr int CAP = BEAM_MAX_OUT * EPT;
    __shared__ u64 s_own[256], s_list[CAP]; __shared__ float s_red[8]; __shared__ double s_sum[4], s_pow[16]; __shared__ u64 s_bound; __shared__ int s_n;
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, base = blockIdx.x * 256 * EPT;
    const float *x = reinterpret_cast<const float *>(a.logits + (long)r * a.row) + base;
    const int n = min(256 * EPT, a.n_vocab - base);
    const bool whole = n == 256 * EPT;          // (a cut chunk goes to the lanes one logit at a time, so that every wave has some)
    auto index = [&](int e) { return whole ? (e / 4 * 256 + tid) * 4 + e % 4 : e * 256 + tid; };
    float v[EPT];
    if (whole) {
#pragma unroll
        for (int e = 0; e < EPT / 4; ++e) { const F4a4 f = reinterpret_cast<const F4a4 *>(x)[e * 256 + tid]; v[4 * e] = f.x; v[4 * e + 1] = f.y; v[4 * e + 2] = f.z; v[4 * e + 3] = f.w; }
    } else {
#pragma unroll
        for (int e = 0; e < EPT; ++e) { const float f = x[min(index(e), n - 1)]; v[e] = index(e) < n ? f : -INFINITY; }
    }
    float top = v[0];
#pragma unroll
    for (int e = 1; e < EPT; ++e) top = fmaxf(top, v[e]);
    const bool quads = a.n_out <= 16; const int owners = quads ? 64 : 256;
    // a quarter of n_out from every wave: the smallest of the waves' bounds is one that n_out elements reach (no barrier and a fourth of the comparisons of a bound over the workgroup)
    float ot = top == top ? top : -INFINITY; int above = 0;
    if (quads) {
        ot = fmaxf(ot, fa_dpp<0xb1>(ot)); ot = fmaxf(ot, fa_dpp<0x4e>(ot));
#pragma unroll
        for (int i = 0; i < 64; i += 4) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ot), i)) > ot;
    } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ot), i)) > ot;
    }
    const float wm = wave_max(top), wb = -wave_max(4 * above < a.n_out ? -ot : -INFINITY);          // (4 above < n_out: fewer than n_out / 4, rounded up, are before it)
    if (lane == 0) { s_red[wave] = wm; s_red[4 + wave] = wb; }
    if (tid < 16) s_pow[tid] = exp2(tid * 0.0625);
    if (tid == 0) s_n = 0;
    __syncthreads();
    const float m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])), least = fminf(fminf(s_red[4], s_red[5]), fminf(s_red[6], s_red[7]));
    bool by_keys = least == -INFINITY;
    if (!by_keys) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) if (v[e] >= least) { const int p = atomicAdd(&s_n, 1); if (p < CAP) s_list[p] = logit_key(v[e], base + index(e)); }
    }
    double l = 0.0; bool nan = false;
#pragma unroll
    for (int e = 0; e < EPT; ++e) nan |= v[e] != v[e];
    if (m != -INFINITY) {          // (nothing but -inf: 0)
#pragma unroll
        for (int e = 0; e < EPT; ++e) l += exp_below((double)v[e] - (double)m, s_pow);
    }
    if (nan) l = __builtin_nan("");
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    if (lane == 0) s_sum[wave] = l;
    __syncthreads();
    if (!by_keys) by_keys = s_n > CAP;
    if (by_keys) {          // (uniform)
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < EPT; ++e) { const u64 k = index(e) < n ? logit_key(v[e], base + index(e)) : 0; own = k > own ? k : own; }
        if (quads) own = shfl_max(shfl_max(own, 1), 2);
        __syncthreads();
        if (!quads || (lane & 3) == 0) s_own[quads ? tid >> 2 : tid] = own;
        if (tid == 0) { s_n = 0; s_bound = 0; }
        __syncthreads();
        if (tid < owners) {
            const u64 mine = s_own[tid]; int rank = 0;
            for (int i = 0; i < owners; ++i) rank += s_own[i] > mine;
            if (rank == a.n_out - 1 && mine) s_bound = mine;          // (fewer owners than n_out have logits: the bound stays 0 and everything is listed)
        }
        __syncthreads();
        const u64 bound = s_bound;
#pragma unroll
        for (int e = 0; e < EPT; ++e) if (index(e) < n) { const u64 k = logit_key(v[e], base + index(e)); if (k >= bound) s_list[atomicAdd(&s_n, 1)] = k; }
        __syncthreads();
    }
    const int count = s_n; const long row = (long)r * a.chunks + blockIdx.x;
    if (tid == 0) a.stat[row] = BeamStat{(s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]), m};
    for (int i = tid; i < count; i += 256) {
        const u64 mine = s_list[i]; int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) rank += s_list[j] > mine;
        if (rank < a.n_out) a.best[row * a.n_out + rank] = mine;
    }
    for (int i = count + tid; i < a.n_out; i += 256) a.best[row * a.n_out + i] = 0;
}

// A candidate of a group in the order (value descending, beam, logit descending, token): the value's bits, ordered like the value, and the rest packed into one number (n_beam * n_vocab
// is at most 2^26, so beam and token take 28 bits beside the logit's 32).  rest 0: none.  Within a beam the value grows with the logit, in 64 bits not always visibly.
struct Cand { u64 value, rest; };
static __device__ __forceinline__ u64 ordered(double c) { const u64 b = __builtin_bit_cast(u64, c); return b ^ ((b >> 63) ? ~0ull : 1ull << 63); }
static __device__ __forceinline__ double unordered(u64 k) { return __builtin_bit_cast(double, k ^ ((k >> 63) ? 1ull << 63 : ~0ull)); }
static __device__ __forceinline__ bool before(const Cand &p, const Cand &q) { return p.value != q.value ? p.value > q.value : p.rest > q.rest; }
static __device__ __forceinline__ u64 quad_xor(u64 k, int d) {          // the value of lane ^ d, d = 1 or 2
    const int lo = (int)(uint32_t)k, hi = (int)(k >> 32);
    return d == 1 ? ((u64)(uint32_t)fa_dpp_i<0xb1>(hi) << 32) | (uint32_t)fa_dpp_i<0xb1>(lo) : ((u64)(uint32_t)fa_dpp_i<0x4e>(hi) << 32) | (uint32_t)fa_dpp_i<0x4e>(lo);
}
// how many of s[0 .. n) come before `p`, by the four lanes of a quad (all with the same p): values first, the rest of the order only where some are equal
static __device__ __forceinline__ int rank_among(const Cand *s, int n, const Cand &p) {
    int above = 0, same = 0;
#pragma unroll 8
    for (int i = threadIdx.x & 3; i < n; i += 4) { const u64 v = s[i].value; above += v > p.value; same += v == p.value; }
    same += fa_dpp_i<0xb1>(same); same += fa_dpp_i<0x4e>(same);
    if (same > 1) {
#pragma unroll 8
        for (int i = threadIdx.x & 3; i < n; i += 4) { const Cand q = s[i]; above += q.value == p.value && q.rest > p.rest; }
    }
    above += fa_dpp_i<0xb1>(above); above += fa_dpp_i<0x4e>(above);
    return above;
}
constexpr int BEAM_LIST = BEAM_MAX_OUT * ((BEAM_MAX_LISTS + 255) / 256);
struct JoinMem { Cand own[256], list[BEAM_LIST], bound; int n; };
// The k best of get(0 .. n), sorted, into out (LDS); returns how many there are.  1024 threads: a quad of lanes to a candidate (ranking is the longest part: 128 + 136 comparisons of
// 64 bits for a group of 8 beams and 16 results; with one lane to a candidate the launch took 18 us).  `mine` are the lane's first OWN candidates, made by the caller so that their loads are
// under way together; get(i) makes those behind them.  n is at most 256 times the share that JoinMem is made for.
static __device__ __forceinline__ int first_of_lane() { return (int)(threadIdx.x >> 2) + 256 * (int)(threadIdx.x & 3); }
template <int OWN, typename F> static __device__ __forceinline__ int choose(int n, int k, const Cand (&mine)[OWN], F get, Cand *out, JoinMem &mem) {
    const int quad = threadIdx.x >> 2; const bool lead = (threadIdx.x & 3) == 0;
    Cand best = mine[0];
#pragma unroll
    for (int p = 1; p < OWN; ++p) if (before(mine[p], best)) best = mine[p];
    for (int i = first_of_lane() + OWN * 1024; i < n; i += 1024) { const Cand q = get(i); if (before(q, best)) best = q; }
#pragma unroll
    for (int d = 1; d <= 2; ++d) { const Cand q = {quad_xor(best.value, d), quad_xor(best.rest, d)}; if (before(q, best)) best = q; }
    if (lead) mem.own[quad] = best;
    if (threadIdx.x == 0) { mem.n = 0; mem.bound = {0, 0}; }
    __syncthreads();
    const int rank = best.rest ? rank_among(mem.own, min(n, 256), best) : 256;
    if (n <= 256) {          // one candidate a quad: its rank is its place
        if (lead && rank < k) { out[rank] = best; atomicAdd(&mem.n, 1); }
        __syncthreads();
        return mem.n;
    }
    if (lead && rank == k - 1) mem.bound = best;
    __syncthreads();
    const Cand bound = mem.bound;
    auto take = [&](const Cand &q) { if (q.rest && !before(bound, q)) mem.list[atomicAdd(&mem.n, 1)] = q; };
#pragma unroll
    for (int p = 0; p < OWN; ++p) take(mine[p]);
    for (int i = first_of_lane() + OWN * 1024; i < n; i += 1024) take(get(i));
    __syncthreads();
    const int count = mem.n;
    for (int i = quad; i < count; i += 256) { const Cand q = mem.list[i]; const int r = rank_among(mem.list, count, q); if (lead && r < k) out[r] = q; }
    __syncthreads();
    return min(count, k);
}
// One workgroup per group.  Only the n_out lists with the best heads can hold any of the n_out best, and of the list with rank r among them only its first n_out - r entries.
// Bound by its chain of memory latencies (statistics, then the lists' entries): the heads are requested before the statistics.
// OWN: candidates of a group are at most that many times 1024 (1: up to 44 results; with 3 for all the small ones take 0.5 us more, the largest 1.2 us less).
template <int OWN> __global__ void __launch_bounds__(1024) beam_join_kernel(BeamArgs a) {
    __shared__ float s_top[BEAM_MAX_BEAMS], s_score[BEAM_MAX_BEAMS]; __shared__ double s_lse[BEAM_MAX_BEAMS]; __shared__ int s_kind[BEAM_MAX_BEAMS];       // 0: logits, 1: finished, 2: nothing but -inf
    __shared__ JoinMem mem; __shared__ Cand s_heads[BEAM_MAX_OUT], s_best[BEAM_MAX_OUT];
    const int g = blockIdx.x, tid = threadIdx.x, k = a.n_out, lists = a.n_beam * a.chunks;
    const u64 *best = a.best + (long)g * lists * k;
    u64 head[OWN];
#pragma unroll
    for (int p = 0; p < OWN; ++p) if (p * 1024 < lists) head[p] = best[(long)min(first_of_lane() + p * 1024, lists - 1) * k];
    for (int b0 = 0; b0 < a.n_beam; b0 += 64) {          // 16 lanes to a beam
        const int b = b0 + (tid >> 4), r = g * a.n_beam + min(b, a.n_beam - 1);
        const BeamStat *stat = a.stat + (long)r * a.chunks;
        const float score = a.score[r]; const bool done = a.done && a.done[r];
        float m = -INFINITY; double l = 0.0;          // the lane's chunks, on the row's maximum
        for (int c = tid & 15; c < a.chunks; c += 16) m = fmaxf(m, stat[c].top);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        for (int c = tid & 15; c < a.chunks; c += 16) { const BeamStat s = stat[c]; l += m == -INFINITY ? s.sum : s.sum * exp((double)s.top - (double)m); }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) l += __shfl_xor(l, d, 64);
        if ((tid & 15) == 0 && b < a.n_beam) {
            s_top[b] = m; s_lse[b] = log(l); s_score[b] = score;
            const bool none = score != score || score == -INFINITY || (!done && (l != l || m == INFINITY || m == -INFINITY));
            s_kind[b] = none ? 2 : done ? 1 : 0;
        }
    }
    __syncthreads();
    const int per_row = min(k, a.n_vocab), t_bits = 32 - __builtin_clz(a.n_vocab), shift = __builtin_ctz(a.chunk);
    const u64 t_mask = (1ull << t_bits) - 1;
    auto made = [&](double c, int b, u64 key) {          // (the beam's field starts at 1, so that no candidate's rest is 0)
        if (c != c || c == -INFINITY) { c = -INFINITY; key = logit_key(-INFINITY, key_token(key)); }
        return Cand{ordered(c), ((u64)(a.n_beam - b) << (32 + t_bits)) | ((key >> 32) << t_bits) | (~(u64)key_token(key) & t_mask)};
    };
    auto beam_of = [&](const Cand &q) { return a.n_beam - (int)(q.rest >> (32 + t_bits)); };
    auto token_of = [&](const Cand &q) { return (int)(~q.rest & t_mask); };
    // entry e of list c of beam b, which is `key`; finished beams and those of nothing have one list, made here: pad first if it counts, then tokens of -inf by their index
    auto entry = [&](int b, int c, int e, u64 key) {
        const int kind = s_kind[b];
        if (kind == 0) return key ? made((double)s_score[b] + (((double)key_logit(key) - (double)s_top[b]) - s_lse[b]), b, key) : Cand{0, 0};
        if (c || e >= per_row) return Cand{0, 0};
        const int t = kind == 2 ? e : e == 0 ? a.pad : e - 1 < a.pad ? e - 1 : e;
        return made(kind == 1 && e == 0 ? (double)s_score[b] : -INFINITY, b, logit_key(-INFINITY, t));
    };
    Cand mine[OWN];
#pragma unroll
    for (int p = 0; p < OWN; ++p) {
        mine[p] = {0, 0}; const int i = first_of_lane() + p * 1024;
        if (p * 1024 < lists && i < lists) { const int b = i / a.chunks; mine[p] = entry(b, i - b * a.chunks, 0, head[p]); }
    }
    const int heads = choose(lists, k, mine, [&](int i) { const int b = i / a.chunks; return entry(b, i - b * a.chunks, 0, best[(long)i * k]); }, s_heads, mem);
    // candidate i = r (r + 1) / 2 + e: entry e <= r of the list with rank h = k - 1 - r, which is entry e of chunk c of beam b; h -1: there is none
    struct Place { int h, e, b, c; };
    auto place = [&](int i) {
        int r = (int)((sqrtf(8.0f * i + 1.0f) - 1.0f) * 0.5f);
        while (r * (r + 1) / 2 > i) --r;
        while ((r + 1) * (r + 2) / 2 <= i) ++r;
        Place p = {k - 1 - r, i - r * (r + 1) / 2, 0, 0};
        if (p.h < 0 || p.h >= heads) p.h = -1;
        else { const Cand q = s_heads[p.h]; p.b = beam_of(q); p.c = s_kind[p.b] ? 0 : token_of(q) >> shift; }          // (the chunk of a head is where its token lies)
        return p;
    };
    const int total = k * (k + 1) / 2;          // (at most OWN * 1024)
    Place at[OWN]; u64 key[OWN];
#pragma unroll
    for (int p = 0; p < OWN; ++p) if (p * 1024 < total) { at[p] = place(first_of_lane() + p * 1024); key[p] = at[p].h >= 0 && at[p].e ? best[(long)(at[p].b * a.chunks + at[p].c) * k + at[p].e] : 0; }
#pragma unroll
    for (int p = 0; p < OWN; ++p) {
        mine[p] = {0, 0};
        if (p * 1024 < total && at[p].h >= 0) mine[p] = at[p].e == 0 ? s_heads[at[p].h] : entry(at[p].b, at[p].c, at[p].e, key[p]);
    }
    __syncthreads();          // (mem is free)
    const int found = choose(total, k, mine, [](int) { return Cand{0, 0}; }, s_best, mem);
    for (int i = tid; i < found; i += 1024) {
        const Cand q = s_best[i]; const long o = (long)g * k + i;
        a.score_out[o] = (float)unordered(q.value); a.parent[o] = g * a.n_beam + beam_of(q); a.token[o] = token_of(q);
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
    // 2048 logits to a workgroup where 8192 would leave most of the chip idle (fewer than 256 workgroups) or more than a fifth of its lanes (1000 rows of 4000: 20.2 -> 17.4 us)
    const long whole = (x->ne[0] + BEAM_CHUNK - 1) / BEAM_CHUNK;
    a->chunk = x->ne[1] * whole < 256 || whole * BEAM_CHUNK * 4 > x->ne[0] * 5 ? BEAM_CHUNK / 4 : BEAM_CHUNK;
    a->chunks = (a->n_vocab + a->chunk - 1) / a->chunk;
    return x->ne[1] * a->chunks * ((int64_t)sizeof(BeamStat) + 8 * (int64_t)n_out);
}
int64_t cdna4_beam_select_workspace(const cdna4_tensor *logits, int n_beam, int n_out, int pad) { PG_NORM(logits, 4) BeamArgs a; return beam_check(logits, n_beam, n_out, pad, &a); }
int cdna4_op_beam_select(cdna4_context *ctx, const cdna4_tensor *logits, const float *score, const int32_t *done, int n_beam, int n_out, int pad, float *score_out, int32_t *parent, int32_t *token,
                         void *stream) {
    ARG_CHECK(ctx, "beam_select: null argument");
    PG_NORM(logits, 4)
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
    a.stat = (BeamStat *)ctx->ws; a.best = (u64 *)(a.stat + rows * a.chunks);
    hipStream_t st = (hipStream_t)stream; const dim3 grid((unsigned)a.chunks, (unsigned)rows);
    if (a.chunk == BEAM_CHUNK) hipLaunchKernelGGL(beam_scan_kernel<32>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(beam_scan_kernel<8>, grid, dim3(256), 0, st, a);
    HIP_TRY(hipGetLastError());
    static_assert(BEAM_MAX_OUT * (BEAM_MAX_OUT + 1) / 2 <= 3 * 1024, "the candidates of a group are its lanes' own");
    if (n_out * (n_out + 1) / 2 <= 1024) hipLaunchKernelGGL(beam_join_kernel<1>, dim3((unsigned)(rows / n_beam)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(beam_join_kernel<3>, dim3((unsigned)(rows / n_beam)), dim3(1024), 0, st, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}
