// paged_attn.hip -- attention of one new token per sequence over a paged key / value cache.
//
// z[h][j] = scale q[h].k[j] (soft-capped), o[h] = sum_j softmax(z[h])[j] v[j]; the query heads of a KV head read the same rows, so the cache is read once per group of 16 heads and the
// operator is bound by that read (4 D bytes a slot and KV head against 4 D flops a query head).  Three things follow:
//
// * Matrix instructions, for any group size: 32 slots are one step of v_mfma_f32_16x16x32.  S^T = K Q^T puts a query head into every lane column and four slots into every lane, which is
//   the operand layout that O^T = V^T P^T wants for P: the probabilities never leave their registers, and the running reference and sum of a head are scalars of a lane.  V arrives as rows
//   (16 bytes a lane, a row per 16 lanes) and becomes the other operand by v_perm, so the loop touches no LDS at all.
// * f32 results from 16-bit operands: q and p are split into two f16 terms or three bf16 ones, K and V are what the cache holds; products and sums are f32.  bf16: exactly 24 bits.  f16: 22
//   bits, rounded to nearest, down to 2^-28 of a row's largest element or a step's largest probability, the products of the second terms summed apart and scaled (a third term would change
//   no result: the scores' own rounding is larger.  Root mean square error beside elementary 32-bit torch, scores of about 6, heads of 128: 2.3e-7 / 5.3e-7).  Without the scale the second
//   terms ended at 2^-32 of the row's maximum: 8192 slots behind one that takes all but 10^-3 of the weight were off by 10^-5.  The extra matrix instructions stay far below the load time
//   (32 or 48 of 16 clk per 16 KB and SIMD).
// * Sums that finite values cannot take out of range: every step of 32 slots is summed on its own maximum and added to accumulators whose weights sum to at most 1, and partial rows are
//   divided by their own sums before they are joined (bf16 values go up to the largest f32).
// * Equal shares: all tiles of 128 slots of all (sequence, KV head) pairs are numbered through, and every workgroup takes an equal contiguous range of the numbers, from the lengths as
//   they are on the device.  Groups of more than 16 query heads: 32 to a wave, or blocks of 16 with workgroups of their own and the same ranges.  A long sequence in a batch of short ones spreads over the chip by itself; a workgroup that covers a unit alone writes its result, the others
//   leave (reference, sum, row divided by it) for the join.
//
// Measured (8 KV heads of 128, medians): 64 sequences of up to 8192 slots, f16, 32 query heads: 1.12 GB in 199 us + 7 us for the join, 5.4 TB/s; one of 131071, bf16, 64 query heads: 537 MB in
// 106 us + 5 us; one of 301 slots: 7.4 us.  The first form, a wave per slot and a workgroup per KV head, took 10.7 ms, 336 ms and 192 us.
#include "paged.cuh"
#include "fa_decode.cuh"
#include <algorithm>
#include <cmath>
#include <type_traits>

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int TILE = 128, WAVES = 4, QH = 16;         // slots of a workgroup's tile (32 a wave), waves, query heads of a matrix instruction
constexpr int ONE_LDS = 104 * 1024;                   // most dynamic LDS of a workgroup that has a unit to itself (and more than the others take)
constexpr int ATTN_MAX_WG = 1024;                     // most workgroups of a launch; the size function, which knows no device, counts with it

struct AttnArgs {
    PagedCache c; const char *q; long q_head, q_seq; char *dst; long d_head, d_seq; char *weight; long w_head, w_seq;
    int group, n_head, lg, blocks, n_wg; float scale, softcap, inv_softcap;      // blocks: of 2^lg query heads in a group; n_wg: workgroups that share the tiles of one block of every group
    int *prefix;                // [n_seq + 1] tiles of a unit before sequence s
    float *part;                // [blocks][n_wg][2][2^lg][D + 2]: what a workgroup leaves of its first / last unit (reference, sum, row divided by the sum of every head)
    float2 *stat;               // [n_seq][n_head] reference and sum of a row (weight only)
    float *score; long score_row;   // [n_seq][n_head][score_row] scores in units of log 2 (weight only)
};

template <bool BF16> static __device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the slots of one query head)
template <typename F> static __device__ __forceinline__ float over_rows(float v, F f) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// the two / three 16-bit terms of a pair of f32 values, packed (first value in the low half)
template <bool BF16> struct Split;
template <> struct Split<false> {
    static constexpr int N = 2;
    static constexpr float UP = 4096.0f;          // the second term is the rounding error of the first times 2^12, in products of its own: for values up to 2^15 it is as far from overflow as
                                                  // they are and keeps its 11 bits where the first keeps them (both down to 2^-14)
    static __device__ __forceinline__ void of(float a, float b, uint32_t (&t)[2]) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 first = {(_Float16)a, (_Float16)b}, rest = {(_Float16)((a - (float)first[0]) * UP), (_Float16)((b - (float)first[1]) * UP)};
        t[0] = __builtin_bit_cast(uint32_t, first); t[1] = __builtin_bit_cast(uint32_t, rest);
    }
};
template <> struct Split<true> {
    static constexpr int N = 3;
    static __device__ __forceinline__ void of(float a, float b, uint32_t (&t)[3]) {      // 24 significant bits = three times 8: exact
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
            t[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            a -= __uint_as_float(x & 0xffff0000u); b -= __uint_as_float(y & 0xffff0000u);
        }
    }
};

// tanh in a dozen instructions: 1 - 2 / (e^2x + 1), whose absolute error is that of 1 (10^-7), and below 0.3 in magnitude, where the difference would lose digits, its Taylor series up to
// x^11 (remainder 2 * 10^-9 of x).  NaN stays NaN; the library's tanhf took 960 of the 1700 cycles of a step of 32 slots of 64 elements.
static __device__ __forceinline__ float tanh_of(float x) {
    const float s = x * x;
    const float small = x * fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, -1382.0f / 155925.0f, 62.0f / 2835.0f), -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float large = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * 2.88539008177792681f) + 1.0f);
    return fabsf(x) < 0.3f ? small : large;
}

// prefix sums of the sequences' tiles into LDS (pre[0] = 0 ... pre[n_seq]); 256 threads
static __device__ __forceinline__ void scan_tiles(const AttnArgs &a, int *pre, int *tot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int run = 0;
    if (threadIdx.x == 0) pre[0] = 0;
    for (int b = 0; b < a.c.n_seq; b += 256) {
        const int s = b + (int)threadIdx.x;
        int v = s < a.c.n_seq ? (paged_len(a.c, s) + TILE - 1) / TILE : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(v, o, 64); if (lane >= o) v += y; }
        if (lane == 63) tot[wave] = v;
        __syncthreads();
        int before = run;
        for (int w = 0; w < wave; ++w) before += tot[w];
        if (s < a.c.n_seq) pre[s + 1] = before + v;
        run += tot[0] + tot[1] + tot[2] + tot[3];
        __syncthreads();
    }
}
// the tiles of all units in n_wg contiguous ranges that differ by one at most: the first `more` workgroups take one tile more
struct Shares {
    int base, more;
    __device__ Shares(int total, int n_wg) { base = total / n_wg; more = total - base * n_wg; }
    __device__ int first(int w) const { return w * base + min(w, more); }
    __device__ int owner(int x) const { const int cut = more * (base + 1); return x < cut ? x / (base + 1) : more + (x - cut) / base; }
};

// ONE: a workgroup per unit (grid: units, sequences), for tables of few slots: no shares, nothing to join, and the weights are added from scores in LDS by the same launch.
// QB: blocks of 16 query heads that a wave takes.
// (Two waves a SIMD, 256 registers, wherever that is enough: with more the compiler puts a step's products into accumulation registers and moves every one of them out: 80 of 1300 instructions.)
template <int D, bool BF16, bool CAP, bool ONE, int QB> __global__ void __launch_bounds__(256, (D * QB <= 128 ? 2 : 1)) paged_attn_kernel(AttnArgs a) {
    constexpr int HEADS = QB * QH, KC = D / 32, VW = D == 64 ? 4 : 8, VH = D == 256 ? 2 : 1, NS = Split<BF16>::N;      // K chunks of 32 elements; V elements of a lane and half; halves of 128
    constexpr float P_SCALE = BF16 ? 1.0f / 32.0f : 32768.0f;          // of a step's probabilities: 32 of 2^-5 sum to 1 in bf16; f16 keeps the bits of those down to 2^-29 of the largest
    extern __shared__ __attribute__((aligned(16))) int s_mem[];
    __shared__ int s_tot[4]; __shared__ float s_m[WAVES][HEADS], s_l[WAVES][HEADS], s_row[2][HEADS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    int *pre = s_mem;                                                              // prefix sums (not ONE)
    float *s_o = reinterpret_cast<float *>(s_mem + (ONE ? 0 : (a.c.n_seq + 4) & ~3));       // [WAVES][heads][D + 4]
    int x = 0, x_end = 1, s = 0, blk = 0;
    if constexpr (!ONE) {
        scan_tiles(a, pre, s_tot);
        blk = blockIdx.x / a.n_wg;
        const Shares shares(pre[a.c.n_seq] * a.c.n_head_kv, a.n_wg);         // (the host has checked that tiles * KV heads < 2^31)
        if (blockIdx.x == 0) for (int i = threadIdx.x; i <= a.c.n_seq; i += 256) a.prefix[i] = pre[i];
        const int wg = blockIdx.x - blk * a.n_wg; x = __builtin_amdgcn_readfirstlane(shares.first(wg)); x_end = __builtin_amdgcn_readfirstlane(shares.first(wg + 1));
        if (x >= x_end) return;
        for (int b = 0; b < a.c.n_seq; b += 64) { const int i = b + lane; s += __popcll(__ballot(i < a.c.n_seq && pre[min(i, a.c.n_seq - 1) + 1] * a.c.n_head_kv <= x)); }
    }
    for (bool first = true; x < x_end; first = false) {
        int n, tiles, hk, tile0 = 0, ntile;
        if constexpr (ONE) {
            s = blockIdx.y; hk = blockIdx.x / a.blocks; blk = blockIdx.x - hk * a.blocks; n = paged_len(a.c, s); tiles = ntile = (n + TILE - 1) / TILE; x = x_end;
        } else {
            while (pre[s + 1] * a.c.n_head_kv <= x) ++s;
            s = __builtin_amdgcn_readfirstlane(s);
            tiles = __builtin_amdgcn_readfirstlane(pre[s + 1] - pre[s]); n = __builtin_amdgcn_readfirstlane(paged_len(a.c, s));
            const int rem = __builtin_amdgcn_readfirstlane(x - pre[s] * a.c.n_head_kv); hk = rem / tiles; tile0 = rem - hk * tiles;
            ntile = min(tiles - tile0, x_end - x);
            x += ntile;
        }
        const int h0 = hk * a.group + blk * HEADS, heads = min(HEADS, (hk + 1) * a.group - h0);
        // the queries: chunk c holds elements 32 c + 8 g ... + 7 of head 16 b + col; requested before the cache rows, split under their way
        float4 x0[QB][KC], x1[QB][KC];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const float *qr = reinterpret_cast<const float *>(a.q + (long)s * a.q_seq + (long)(h0 + min(QH * b + col, heads - 1)) * a.q_head) + 8 * g;
#pragma unroll
            for (int c = 0; c < KC; ++c) { x0[b][c] = reinterpret_cast<const float4 *>(qr + 32 * c)[0]; x1[b][c] = reinterpret_cast<const float4 *>(qr + 32 * c)[1]; }
        }
        const char *kb = a.c.k + (long)hk * a.c.k_head, *vb = a.c.v + (long)hk * a.c.v_head;
        const int *table = a.c.table + (long)s * a.c.table_row; const int in_page = (1 << a.c.page_shift) - 1;
        // 16 slots from j on lie in one page (pages are powers of two >= 16).  Its entry in the table (requested without a branch: the last one stands for those past the end), and the id that
        // this entry is: -1 past the end or unmapped
        auto entry = [&](int j) { return table[min(j, max(n - 1, 0)) >> a.c.page_shift]; };
        auto id_of = [&](int e, int j) { return j < n && (unsigned)e < (unsigned)a.c.n_pages ? e : -1; };
        const uint32_t k_lane = (uint32_t)col * (uint32_t)a.c.k_row + 16u * g, v_lane = 4u * g * (uint32_t)a.c.v_row + 2u * VW * col;
        u4 kr[2][KC]; uint32_t vr[8][VH][VW / 2];
        // (a half that is past the end or unmapped loads page 0: in bounds, and masked below)
        auto load_k = [&](int j, int id0, int id1) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int id = t ? id1 : id0, off = id < 0 ? 0 : (j + 16 * t) & in_page;
                const char *p = kb + (long)max(id, 0) * a.c.k_page + (long)off * a.c.k_row;
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[t][c] = *reinterpret_cast<const u4 *>(p + k_lane + 64 * c);
            }
        };
        auto load_v = [&](int j, int id0, int id1) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int id = t ? id1 : id0, off = id < 0 ? 0 : (j + 16 * t) & in_page;
                const char *p = vb + (long)max(id, 0) * a.c.v_page + (long)off * a.c.v_row;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int hf = 0; hf < VH; ++hf) {
                        const char *e = p + (v_lane + (uint32_t)r * (uint32_t)a.c.v_row) + 256 * hf;
                        if constexpr (VW == 8) { const u4 w = *reinterpret_cast<const u4 *>(e);
#pragma unroll
                            for (int i = 0; i < 4; ++i) vr[4 * t + r][hf][i] = w[i]; }
                        else { const uint2 w = *reinterpret_cast<const uint2 *>(e); vr[4 * t + r][hf][0] = w.x; vr[4 * t + r][hf][1] = w.y; }
                    }
            }
        };
        // o / l: the wave's sums of 2^(z - m) v and 2^(z - m); `held` of a head bounds the sum of 2^(z - m) over all its slots so far and stays at most 1 (see step)
        f4 o[QB][VH][VW]; float m[QB], l[QB], held[QB];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            m[b] = -INFINITY; l[b] = 0.f; held[b] = 0.f;
#pragma unroll
            for (int hf = 0; hf < VH; ++hf)
#pragma unroll
                for (int i = 0; i < VW; ++i) o[b][hf][i] = (f4){0.f, 0.f, 0.f, 0.f};
        }
        int j = (tile0 * WAVES + wave) * 32; const int j_end = min((tile0 + ntile) * TILE, n);
        float *score = !a.weight ? nullptr : ONE ? s_o + WAVES * heads * (D + 4) : a.score + ((long)s * a.n_head + h0) * a.score_row;          // of the unit's first head
        u4 q[QB][NS][KC]; float unscale[QB]; int id0 = -1, id1 = -1, nx0 = -1, nx1 = -1;
        // One step: the tile in kr / vr.  MORE: the next tile is requested on the way, K as soon as its registers are read, V at the end.  (The last tile is a step of its own and not a
        // condition around the loads: behind a condition the compiler waits for V of the next tile before the first product of K.)
        auto step = [&](auto more) {
            constexpr bool MORE = decltype(more)::value;
            f4 z[QB][2], low[QB][2];          // (low: the products of the second f16 terms)
#pragma unroll
            for (int b = 0; b < QB; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    z[b][t] = low[b][t] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        if constexpr (BF16) {
#pragma unroll
                            for (int k = NS - 1; k >= 0; --k) z[b][t] = mfma<BF16>(kr[t][c], q[b][k][c], z[b][t]);
                        } else { z[b][t] = mfma<BF16>(kr[t][c], q[b][0][c], z[b][t]); low[b][t] = mfma<BF16>(kr[t][c], q[b][1][c], low[b][t]); }
                    }
                }
            const int jn = j + TILE; int e0 = 0, e1 = 0;
            if constexpr (MORE) { load_k(jn, nx0, nx1); e0 = entry(jn + TILE); e1 = entry(jn + TILE + 16); }
            const bool whole = id0 >= 0 && id1 >= 0 && j + 32 <= n;          // (wave-uniform)
            uint32_t p[QB][NS][4]; float over[QB];
#pragma unroll
            for (int b = 0; b < QB; ++b) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if constexpr (!BF16) z[b][t][r] = fmaf(low[b][t][r], 1.0f / Split<false>::UP, z[b][t][r]);
                        float v = z[b][t][r] * unscale[b];
                        if constexpr (CAP) v = a.softcap * 1.44269504088896341f * tanh_of(v * a.inv_softcap);
                        z[b][t][r] = v;
                    }
                if (!whole) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) if ((t ? id1 : id0) < 0 || j + 16 * t + 4 * g + r >= n) {
                            z[b][t][r] = -INFINITY;
                            if (b == 0) {
#pragma unroll
                                for (int hf = 0; hf < VH; ++hf)
#pragma unroll
                                    for (int i = 0; i < VW / 2; ++i) vr[4 * t + r][hf][i] = 0u;          // (0 times what an unused slot holds may be NaN)
                            }
                        }
                }
                if (score && QH * b + col < heads) {
                    float *to = score + (long)(QH * b + col) * a.score_row + j + 4 * g;
#pragma unroll
                    for (int t = 0; t < 2; ++t) *reinterpret_cast<f4 *>(to + 16 * t) = z[b][t];
                }
                float top = fmaxf(fmaxf(fmaxf(z[b][0][0], z[b][0][1]), fmaxf(z[b][0][2], z[b][0][3])), fmaxf(fmaxf(z[b][1][0], z[b][1][1]), fmaxf(z[b][1][2], z[b][1][3])));
                top = over_rows(top, [](float p, float r) { return fmaxf(p, r); });
                // A step's own maximum is the reference of its probabilities: their terms are as exact in every step, and f carries their sums over to the reference m of o and l.  m is not
                // the maximum: it is raised (by 2^3 more than needed: a logarithmic number of times) where 2^top for each of the 32 slots would take `held` past 1.  A sum of 2^(z - m) v
                // is then no larger than the largest |v|: bf16 values may be as large as f32's.
                float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m[b]) * 32.0f;
                if (__ballot(!(held[b] + f <= 1.0f))) {
                    const float to = held[b] + f <= 1.0f ? m[b] : fmaxf(m[b], top + 5.0f) + 3.0f, down = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[b] - to);
                    m[b] = to; l[b] *= down; held[b] *= down; f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - to) * 32.0f;
#pragma unroll
                    for (int hf = 0; hf < VH; ++hf)
#pragma unroll
                        for (int i = 0; i < VW; ++i) o[b][hf][i] *= down;
                }
                held[b] += f; over[b] = f * (1.0f / (32.0f * P_SCALE));
                const float ref = top == -INFINITY ? 0.f : top;
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const float p0 = __builtin_amdgcn_exp2f(z[b][t][r] - ref) * P_SCALE, p1 = __builtin_amdgcn_exp2f(z[b][t][r + 1] - ref) * P_SCALE;
                        sum += p0 + p1;
                        uint32_t w[NS]; Split<BF16>::of(p0, p1, w);
#pragma unroll
                        for (int k = 0; k < NS; ++k) p[b][k][2 * t + r / 2] = w[k];
                    }
                l[b] = fmaf(over[b], sum, l[b]);
            }
#pragma unroll
            for (int hf = 0; hf < VH; ++hf)
#pragma unroll
                for (int i = 0; i < VW; ++i) {          // column i of every lane's 8 (4) elements: its 8 slots side by side
                    const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
                    u4 vt;
#pragma unroll
                    for (int w = 0; w < 4; ++w) vt[w] = __builtin_amdgcn_perm(vr[2 * w + 1][hf][i / 2], vr[2 * w][hf][i / 2], sel);
#pragma unroll
                    for (int b = 0; b < QB; ++b) {
                        auto product = [&](int k, f4 c) { return mfma<BF16>(vt, (u4){p[b][k][0], p[b][k][1], p[b][k][2], p[b][k][3]}, c); };
                        const f4 zero = (f4){0.f, 0.f, 0.f, 0.f};
                        if constexpr (BF16) o[b][hf][i] += over[b] * product(0, product(1, product(NS - 1, zero)));
                        else o[b][hf][i] += over[b] * product(0, zero) + (over[b] * (1.0f / Split<false>::UP)) * product(1, zero);
                    }
                }
            if constexpr (MORE) { load_v(jn, nx0, nx1); id0 = nx0; id1 = nx1; nx0 = id_of(e0, jn + TILE); nx1 = id_of(e1, jn + TILE + 16); j = jn; }
        };
        if (j < j_end) {
            const int e0 = entry(j), e1 = entry(j + 16), e2 = entry(j + TILE), e3 = entry(j + TILE + 16);
            id0 = id_of(e0, j); id1 = id_of(e1, j + 16); nx0 = id_of(e2, j + TILE); nx1 = id_of(e3, j + TILE + 16);
            load_k(j, id0, id1); load_v(j, id0, id1);
            __builtin_amdgcn_sched_barrier(0);          // (V too is requested before the split of the queries)
            const float pre_scale = CAP ? a.scale : a.scale * 1.44269504088896341f;
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                float up = 1.0f; unscale[b] = pre_scale;
                if constexpr (!BF16) {          // a power of two that puts the largest element into [2^14, 2^15): the f16 terms do not overflow, and elements down to 2^-28 of the largest keep their bits
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < KC; ++c) top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(x0[b][c].x), fabsf(x0[b][c].y)), fmaxf(fabsf(x0[b][c].z), fabsf(x0[b][c].w))),
                                                                       fmaxf(fmaxf(fabsf(x1[b][c].x), fabsf(x1[b][c].y)), fmaxf(fabsf(x1[b][c].z), fabsf(x1[b][c].w)))));
                    top = over_rows(top, [](float p, float r) { return fmaxf(p, r); });
                    const int e = top > 0.f ? min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100), 127) : 0;
                    up = __uint_as_float((uint32_t)(127 + 14 - e) << 23); unscale[b] = __uint_as_float((uint32_t)(127 - 14 + e) << 23) * pre_scale;
                }
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const float e[8] = {x0[b][c].x, x0[b][c].y, x0[b][c].z, x0[b][c].w, x1[b][c].x, x1[b][c].y, x1[b][c].z, x1[b][c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) { uint32_t t[NS]; Split<BF16>::of(e[2 * i] * up, e[2 * i + 1] * up, t);
#pragma unroll
                        for (int k = 0; k < NS; ++k) q[b][k][c][i] = t[k]; }
                }
            }
            while (j + TILE < j_end) step(std::true_type());
            step(std::false_type());
        }
        // the four waves' results: (m, l) through LDS, then the accumulators on the common maximum
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            l[b] = over_rows(l[b], [](float p, float r) { return p + r; });
            if (m[b] == -INFINITY && l[b] != l[b]) m[b] = 0.f;            // (scores that are all NaN: the maximum has passed them over, the result is NaN and not a row of nothing)
        }
        __syncthreads();                                                  // (the previous unit's reads of s_o are done)
#pragma unroll
        for (int b = 0; b < QB; ++b) if (g == 0) { s_m[wave][QH * b + col] = m[b]; s_l[wave][QH * b + col] = l[b]; }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int h = QH * b + col;
            const float m0 = s_m[0][h], m1 = s_m[1][h], m2 = s_m[2][h], m3 = s_m[3][h], M = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), to = M == -INFINITY ? 0.f : M;
            const float L = (s_l[0][h] * __builtin_amdgcn_exp2f(m0 - to) + s_l[1][h] * __builtin_amdgcn_exp2f(m1 - to)) +          // (0 for a wave that had nothing)
                            (s_l[2][h] * __builtin_amdgcn_exp2f(m2 - to) + s_l[3][h] * __builtin_amdgcn_exp2f(m3 - to));
            const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[b] - to) / L;            // (the rows are divided before they are added: see held)
            if (wave == 0 && g == 0) { s_row[0][h] = M; s_row[1][h] = L; }
            if (h < heads) {
                float *so = s_o + (wave * heads + h) * (D + 4);
#pragma unroll
                for (int hf = 0; hf < VH; ++hf)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int i = 0; i < VW; i += 4)      // element 128 hf + VW (4 g + r) + i
                            *reinterpret_cast<f4 *>(so + 128 * hf + VW * (4 * g + r) + i) = (f4){o[b][hf][i][r] * f, o[b][hf][i + 1][r] * f, o[b][hf][i + 2][r] * f, o[b][hf][i + 3][r] * f};
            }
        }
        __syncthreads();
        const bool alone = ONE || ntile == tiles;
        float *part = ONE ? nullptr : a.part + ((long)blockIdx.x * 2 + (first ? 0 : 1)) * HEADS * (D + 2);
        for (int e = threadIdx.x; e < heads * D / 4; e += 256) {
            const int h = e / (D / 4), d = (e - h * (D / 4)) * 4;
            const float Mh = s_row[0][h], L = s_row[1][h];
            const float *so = s_o + h * (D + 4) + d; const int next = heads * (D + 4);
            f4 v = (*reinterpret_cast<const f4 *>(so) + *reinterpret_cast<const f4 *>(so + next)) + (*reinterpret_cast<const f4 *>(so + 2 * next) + *reinterpret_cast<const f4 *>(so + 3 * next));
            if (alone) {
                *reinterpret_cast<f4 *>(a.dst + (long)s * a.d_seq + (long)(h0 + h) * a.d_head + d * 4) = v;
                if (!ONE && d == 0 && a.stat) a.stat[(long)s * a.n_head + h0 + h] = make_float2(Mh, L);
            } else {
                float *ph = part + h * (D + 2);
                if (d == 0) { ph[0] = Mh; ph[1] = L; }
                ph[2 + d] = v[0]; ph[3 + d] = v[1]; ph[4 + d] = v[2]; ph[5 + d] = v[3];
            }
        }
        if (ONE && a.weight) {          // (one unit to a KV head: the host has seen to it)
            const float *z = s_o + WAVES * heads * (D + 4);
            float *w = reinterpret_cast<float *>(a.weight + (long)s * a.w_seq + (long)hk * a.w_head);
            for (int i = threadIdx.x; i < n; i += 256) {          // one thread to a slot, the heads in order
                float sum = 0.f;
                for (int h = 0; h < heads; ++h) {
                    const float zi = z[h * (int)a.score_row + i];          // -inf: not attended to, whatever the row is
                    if (zi != -INFINITY) sum += __builtin_amdgcn_exp2f(zi - s_row[0][h]) / s_row[1][h];
                }
                if (sum != 0.f) w[i] += sum;
            }
        }
    }
}
// where the partial results of a query head lie: those of `count` neighbouring workgroups, the first at base + other, the next at base + step ...  A workgroup's slot 0 is its first unit,
// slot 1 a later (its last) one: only the first of the row's workgroups can have begun with another unit.  count 1: the row is done.
template <int D> struct RowParts {
    const float *base; long other, step; int count, tiles;
    __device__ RowParts(const AttnArgs &a, int h, int s) {
        const int p0 = a.prefix[s]; tiles = a.prefix[s + 1] - p0; count = 0; base = nullptr; other = 0; step = (2l << a.lg) * (D + 2);
        if (!tiles) return;
        const Shares shares(a.prefix[a.c.n_seq] * a.c.n_head_kv, a.n_wg);
        const int hk = h / a.group, in = h - hk * a.group, x0 = p0 * a.c.n_head_kv + hk * tiles, w0 = shares.owner(x0);
        count = shares.owner(x0 + tiles - 1) - w0 + 1;
        base = a.part + w0 * step + offset(a, in);
        other = shares.first(w0) < x0 ? step / 2 : 0;
    }
    __device__ const float *at(int i) const { return base + i * step + (i ? 0 : other); }
    // of head `in` of a group behind the group's first
    static __device__ long offset(const AttnArgs &a, int in) { const int b = in >> a.lg; return (((long)b * a.n_wg * 2 << a.lg) + (in - (b << a.lg))) * (D + 2); }
};
// weight[slot] += sum over the group of 2^(z - m) / l for 1024 slots of a KV head, four to a thread, the heads in order.  The rows' m and l are joined here once more, 64 heads at a
// time, 16 lanes to a head, which is cheaper than a third launch behind the join.  Nothing branches between the loads of the scores: 8 sequences of up to 4099 slots, 71 heads on one KV head of
// 64: 38 us with a branch per head and 16 heads at a time, 17 us so.
template <int D> static __device__ __forceinline__ void add_weights(const AttnArgs &a, int hk, int s, int chunk, float2 *s_row) {
    const int n = paged_len(a.c, s), j = chunk * 1024 + (int)threadIdx.x * 4, part = threadIdx.x & 15;
    if (chunk * 1024 >= n) return;
    const RowParts<D> row(a, hk * a.group, s);          // (the group's heads lie alike)
    f4 sum = (f4){0.f, 0.f, 0.f, 0.f};
    for (int h0 = 0; h0 < a.group; h0 += 64) {
        const int heads = min(64, a.group - h0);
        auto in = [&](int q) { return h0 + min(16 * q + ((int)threadIdx.x >> 4), heads - 1); };          // the lane's q-th head
        auto at = [&](int q, int i) { return *reinterpret_cast<const float2 *>(row.at(i) + RowParts<D>::offset(a, in(q))); };
        float2 first[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) if (16 * q < heads) first[q] = row.count == 1 ? a.stat[(long)s * a.n_head + hk * a.group + in(q)] : part < row.count ? at(q, part) : make_float2(-INFINITY, 0.f);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) if (16 * q < heads) {
            float m = first[q].x, l = first[q].y;
            if (row.count != 1) {
                for (int i = part + 16; i < row.count; i += 16) {
                    const float2 p = at(q, i); const float to = fmaxf(m, p.x);
                    if (to != -INFINITY) l = l * __builtin_amdgcn_exp2f(m - to) + p.y * __builtin_amdgcn_exp2f(p.x - to);
                    m = to;
                }
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) {
                    const float om = __shfl_xor(m, d, 64), ol = __shfl_xor(l, d, 64), to = fmaxf(m, om);
                    if (to != -INFINITY) l = l * __builtin_amdgcn_exp2f(m - to) + ol * __builtin_amdgcn_exp2f(om - to);
                    m = to;
                }
            }
            if (part == 0) s_row[16 * q + (threadIdx.x >> 4)] = make_float2(m, 1.0f / l);
        }
        __syncthreads();
        const float *z0 = a.score + ((long)s * a.n_head + hk * a.group + h0) * a.score_row + j;
        if (j < n) {
#pragma unroll 8
            for (int i = 0; i < heads; ++i) {
                const float2 st = s_row[i]; const f4 z = *reinterpret_cast<const f4 *>(z0 + i * a.score_row);
#pragma unroll
                for (int e = 0; e < 4; ++e) { const float p = __builtin_amdgcn_exp2f(z[e] - st.x) * st.y; sum[e] += z[e] != -INFINITY ? p : 0.0f; }          // (-inf: not attended to, whatever the row is)
            }
        }
    }
    float *w = reinterpret_cast<float *>(a.weight + (long)s * a.w_seq + (long)hk * a.w_head);
#pragma unroll
    for (int e = 0; e < 4; ++e) if (j + e < n && sum[e] != 0.f) w[j + e] += sum[e];
}
// grid (query heads, then with weights KV heads x chunks of 1024 slots; sequences): the rows that several workgroups share, the rows of nothing, the weights.  256 threads: the partial
// maxima and sums one to a thread, then D / 4 threads to a partial accumulator and 1024 / D of those at a time.
// WEIGHT: a kernel of its own, since the sums of the weights take twice the registers (64 ragged sequences without weights: 7.9 us with them in, 6.3 us).
template <int D, bool WEIGHT> __global__ void __launch_bounds__(256) paged_attn_join_kernel(AttnArgs a) {
    __shared__ float s_f[ATTN_MAX_WG], s_red[8]; __shared__ f4 s_v[256];
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if constexpr (WEIGHT) if (h >= a.n_head) { __shared__ float2 s_row[64]; const int chunks = (int)(a.score_row + 1023) / 1024, i = h - a.n_head; add_weights<D>(a, i / chunks, s, i % chunks, s_row); return; }
    float *out = reinterpret_cast<float *>(a.dst + (long)s * a.d_seq + (long)h * a.d_head);
    const RowParts<D> part(a, h, s);
    if (part.tiles == 0) { if (tid < D / 4) *reinterpret_cast<f4 *>(out + 4 * tid) = (f4){0.f, 0.f, 0.f, 0.f}; return; }
    const int count = part.count;
    if (count == 1) return;
    float M = -INFINITY;
    for (int i = tid; i < count; i += 256) { const float m = part.at(i)[0]; s_f[i] = m; M = fmaxf(M, m); }
    M = wave_max(M);
    if (lane == 0) s_red[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    float L = 0.f;
    for (int i = tid; i < count; i += 256) { const float m = s_f[i], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M) * part.at(i)[1]; s_f[i] = f; L += f; }
    L = wave_sum_dpp(L);
    if (lane == 0) s_red[4 + wave] = L;
    __syncthreads();
    L = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
    const float share = M == -INFINITY ? 0.f : 1.0f / L;          // (nothing to attend to: a row of zeros)
    constexpr int TD = D / 4, ROWS = 256 / TD;
    const int d = (tid % TD) * 4, row = tid / TD;
    f4 v = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = row; i < count; i += ROWS) {
        const float *p = part.at(i) + 2 + d; const float2 lo = *reinterpret_cast<const float2 *>(p), hi = *reinterpret_cast<const float2 *>(p + 2);
        const float f = s_f[i] * share;          // the partial rows are divided by their own sums: what is added here is no larger than the largest value
        v[0] += lo.x * f; v[1] += lo.y * f; v[2] += hi.x * f; v[3] += hi.y * f;
    }
    s_v[tid] = v;
    __syncthreads();
    if (row) return;
#pragma unroll
    for (int r = 1; r < ROWS; ++r) v += s_v[r * TD + tid];
    *reinterpret_cast<f4 *>(out + d) = v;
}
static int attn_check(const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *dst, AttnArgs *a) {
    ARG_CHECK(q && dst, "paged_attn: null argument");
    int rc = pg_cache_check("paged_attn", k_cache, v_cache, table, false, &a->c); if (rc) return rc;
    for (const cdna4_tensor *t : {q, dst}) {
        ARG_CHECK(pg_sizes_ok(t) && t->type == CDNA4_TYPE_F32 && t->ne[0] == a->c.D && t->ne[1] == q->ne[1] && t->ne[2] == a->c.n_seq && t->ne[3] == 1, "paged_attn: q and dst f32 [D, n_head, n_seq]");
        OP_CHECK(t->nb[0] == 4 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && (uintptr_t)t->data % 16 == 0, "paged_attn: rows of q and dst dense and 16-byte aligned");
    }
    ARG_CHECK(pg_disjoint_elems(dst, 4), "paged_attn: dst is written: its elements may not overlap");
    ARG_CHECK(q->ne[1] % a->c.n_head_kv == 0, "paged_attn: n_head a multiple of n_head_kv");
    OP_CHECK(q->ne[1] <= 16384, "paged_attn: at most 16384 query heads");
    if (weight && (rc = pg_slots_check("paged_attn", "weight", weight, CDNA4_TYPE_F32, a->c, true))) return rc;
    a->n_head = (int)q->ne[1]; a->group = a->n_head / a->c.n_head_kv; a->lg = 4; a->blocks = (a->group + QH - 1) / QH;
    const long slots = (long)a->c.W << a->c.page_shift, tiles = (slots + TILE - 1) / TILE;
    OP_CHECK(tiles * a->c.n_seq < (1l << 31) / std::max(a->c.n_head_kv * a->blocks, 1) && tiles * a->c.n_head_kv < (1l << 26), "paged_attn: too many slots in all");
    a->score_row = tiles * TILE;
    return CDNA4_OK;
}
// scratch: prefix sums | partial results of the workgroups | row statistics | scores (the last two with weights only)
struct AttnScratch { size_t part, stat, score, total; };
static AttnScratch attn_scratch(const AttnArgs &a, bool weight, int n_wg) {
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    AttnScratch s; s.part = up((size_t)(a.c.n_seq + 1) * 4);
    s.stat = s.part + up((size_t)n_wg * 2 * QH * (a.c.D + 2) * 4);
    s.score = s.stat + (weight ? up((size_t)a.c.n_seq * a.n_head * 8) : 0);
    s.total = s.score + (weight ? (size_t)a.c.n_seq * a.n_head * a.score_row * 4 : 0);
    return s;
}
int64_t cdna4_paged_attn_workspace(const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *dst) {
    PG_NORM(q, 4) PG_NORM(dst, 4) PG_NORM(weight, 4)
    AttnArgs a; const int rc = attn_check(q, k_cache, v_cache, table, weight, dst, &a); return rc ? rc : (int64_t)attn_scratch(a, weight != nullptr, ATTN_MAX_WG).total;
}
int cdna4_op_paged_attn(cdna4_context *ctx, const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const int32_t *n_kv, const cdna4_tensor *weight,
                        const cdna4_tensor *dst, float scale, float softcap, void *stream) {
    ARG_CHECK(ctx, "paged_attn: null argument");
    PG_NORM(q, 4) PG_NORM(dst, 4) PG_NORM(weight, 4)
    AttnArgs a; int rc = attn_check(q, k_cache, v_cache, table, weight, dst, &a); if (rc) return rc;
    if (pg_empty(q)) return CDNA4_OK;
    ARG_CHECK(n_kv && q->data && dst->data && (a.c.W == 0 || (a.c.table && (!weight || weight->data))), "paged_attn: null data");
    const PgRange args[] = {pg_range("dst", dst, 4, true), pg_range("weight", weight, 4, true), pg_range("q", q, 4, false), pg_range("k_cache", k_cache, 2, false),
                            pg_range("v_cache", v_cache, 2, false), pg_range("table", table, 4, false), pg_range("n_kv", n_kv, (long)a.c.n_seq * 4, false)};
    if ((rc = pg_apart("paged_attn", args))) return rc;
    if (a.c.W == 0) { a.c.table = n_kv; a.c.table_row = 0; }          // (no slots: the entry that is read for a missing one is anything)
    a.c.n_kv = n_kv; a.scale = scale; a.softcap = softcap; a.inv_softcap = softcap != 0.0f ? 1.0f / softcap : 0.0f;
    a.q = (const char *)q->data; a.q_head = q->nb[1]; a.q_seq = q->nb[2]; a.dst = (char *)dst->data; a.d_head = dst->nb[1]; a.d_seq = dst->nb[2];
    a.weight = weight ? (char *)weight->data : nullptr; a.w_head = weight ? weight->nb[1] : 0; a.w_seq = weight ? weight->nb[2] : 0;
    DEVICE_SCOPE(ctx);
    const long row_tiles = a.score_row / TILE, tiles = row_tiles * a.c.n_seq * a.c.n_head_kv; const int n_unit = a.c.n_head_kv * a.blocks;
    const bool bf = k_cache->type == CDNA4_TYPE_BF16, cap = softcap != 0.0f;
    hipStream_t st = (hipStream_t)stream;
    const size_t merge = (size_t)WAVES * std::min(QH, a.group) * (a.c.D + 4) * 4;
    // A workgroup per unit where a unit is little work, or where the units fill the chip and none is long.  Measured, us with a workgroup per unit / with equal shares and a join (f16, 32
    // query heads and 8 KV heads of 128; sequences x slots): 1 x 100: 6.2 / 9.2, 1 x 640: 10.2 / 11.2, 1 x 1024: 13.5 / 11.3, 8 x 1024: 14.2 / 14.7, 32 x 1024: 23.9 / 30.9, 64 x 512: 24.2 /
    // 29.4, 64 x 2048: 94 / 100, 256 x 2048: 359 / 373; bf16, 4 heads of 64, 1 x 768: 8.3 / 10.0; of 256, 1 x 512: 14.9 / 13.8, 128 x 2048: 355 / 377.
    // With weights: if a KV head is one unit and its scores fit LDS.
    const size_t one_lds = merge + (weight ? (size_t)a.group * a.score_row * 4 : 0);
    const bool one = (row_tiles * a.c.D <= 640 || (row_tiles <= 16 && (long)a.c.n_seq * n_unit >= ctx->num_cu)) && (!weight || a.group <= QH) && one_lds <= ONE_LDS;
#define ATTN(D_, B_, C_, O_, Q_, grid, lds) do { if ((lds) > 60 * 1024) HIP_TRY((pg_opt_in_lds<paged_attn_kernel<D_, B_, C_, O_, Q_>>(ctx->device, ONE_LDS))); \
                                                 hipLaunchKernelGGL((paged_attn_kernel<D_, B_, C_, O_, Q_>), grid, dim3(256), lds, st, a); } while (0)
#define ATTN_D(D_, O_, Q_, grid, lds) do { if (bf) { if (cap) ATTN(D_, true, true, O_, Q_, grid, lds); else ATTN(D_, true, false, O_, Q_, grid, lds); } \
                                           else { if (cap) ATTN(D_, false, true, O_, Q_, grid, lds); else ATTN(D_, false, false, O_, Q_, grid, lds); } HIP_TRY(hipGetLastError()); } while (0)
#define ATTN_ALL(O_, grid, lds) do { if (a.c.D == 64) ATTN_D(64, O_, 1, grid, lds); else if (a.c.D == 128) ATTN_D(128, O_, 1, grid, lds); else ATTN_D(256, O_, 1, grid, lds); } while (0)
    if (one) {
        a.n_wg = 0; a.prefix = nullptr; a.part = nullptr; a.stat = nullptr; a.score = nullptr;
        ATTN_ALL(true, dim3((unsigned)n_unit, (unsigned)a.c.n_seq), one_lds);
        return CDNA4_OK;
    }
    // Groups of 17 to 32 heads over much cache: 32 heads to a wave, so that it is read once (heads of 64, and of 128 in f16; for 256 there are not registers enough).  Two of those waves'
    // registers do not fit a SIMD (heads of 128), so each of its steps is in the open: with fewer tiles than 16 to a CU, or rows of which the ends count, two blocks of 16 are faster, and in
    // bf16, which has three terms for two, always.  us with blocks of 16 / 32 to a wave (sequences of up to as many slots, query heads on KV heads; f16): of 128: 64 x 8192, 160 on 8: 334 /
    // 300 (bf16: 276 / 298), 32 x 8192, 80 on 4: 90.6 / 83.8 (75.3 / 82.6), 64 x 8192, 20 on 1: 50.1 / 47.8 (44.2 / 47.2), 16 x 4099, 160 on 8: 51.0 / 59.2, 1 x 3000, 20 on 1: 12.4 / 14.7;
    // of 64: 64 x 8192, 160 on 8: 160 / 140 (157 / 139), 16 x 4099, 160 on 8: 34.2 / 29.3, 1 x 130000, 20 on 1: 19.4 / 21.7.
    // Larger groups (and the others): blocks of 16 heads that read the same tiles at the same time: workgroups that are a multiple of 8 apart share an XCD and its L2, so much of the cache
    // comes from memory once.  (Before a step's sums were its own, us with a numbering of all blocks one after the other / with this one: 64 x 8192, 32 on 1 of 128: 54.5 / 51.4, 1 x 130000,
    // 20 on 1 of 256: 50.4 / 43.5; bf16, 128 on 1 of 128: 80.8 / 51.8.)
    const bool two = a.group > QH && a.group <= 2 * QH && (a.c.D == 64 || (a.c.D == 128 && !bf)) && tiles >= 16l * ctx->num_cu && row_tiles * TILE >= 64 * a.c.D;
    if (two) { a.lg = 5; a.blocks = 1; }
    const int qb = two ? 2 : 1, per_cu = a.c.D == 256 || (a.c.D == 128 && two) ? 1 : 2;          // (what the registers allow)
    long most_wg = std::min<long>((long)ctx->num_cu * per_cu, ATTN_MAX_WG / qb) / a.blocks;       // (blocks: at most 1024)
    if (a.blocks > 1 && most_wg > 8) most_wg &= ~7l;
    a.n_wg = (int)std::max<long>(1, std::min(tiles, most_wg));
    const AttnScratch sc = attn_scratch(a, weight != nullptr, a.n_wg * a.blocks * qb);
    if ((rc = cdna4_ensure_ws(ctx, sc.total, st))) return rc;
    char *ws = (char *)ctx->ws;
    a.prefix = (int *)ws; a.part = (float *)(ws + sc.part); a.stat = weight ? (float2 *)(ws + sc.stat) : nullptr; a.score = weight ? (float *)(ws + sc.score) : nullptr;
    const size_t lds = (size_t)((a.c.n_seq + 4) & ~3) * 4 + (size_t)WAVES * std::min(QH * qb, a.group) * (a.c.D + 4) * 4;          // (at most (8192 + 4) * 4 + 4 * 32 * 132 * 4 bytes)
    const dim3 grid((unsigned)(a.n_wg * a.blocks));
    if (!two) ATTN_ALL(false, grid, lds);
    else if (a.c.D == 64) ATTN_D(64, false, 2, grid, lds);
    else { if (cap) ATTN(128, false, true, false, 2, grid, lds); else ATTN(128, false, false, false, 2, grid, lds); HIP_TRY(hipGetLastError()); }
    const dim3 join((unsigned)(a.n_head + (weight ? a.c.n_head_kv * ((a.score_row + 1023) / 1024) : 0)), (unsigned)a.c.n_seq);
#define JOIN(D_) do { if (weight) hipLaunchKernelGGL((paged_attn_join_kernel<D_, true>), join, dim3(256), 0, st, a); \
                      else hipLaunchKernelGGL((paged_attn_join_kernel<D_, false>), join, dim3(256), 0, st, a); } while (0)
    if (a.c.D == 64) JOIN(64); else if (a.c.D == 128) JOIN(128); else JOIN(256);
    HIP_TRY(hipGetLastError());
    return CDNA4_OK;
}
