// paged_attn.hip -- attention of one new token per sequence over a paged key / value cache.
#include "paged.cuh"
#include "fa_decode.cuh"
#include <cmath>

struct AttnArgs {
    PagedCache c; const char *q; long q_head, q_seq; char *dst; long d_head, d_seq; char *weight; long w_head, w_seq;
    int group; float scale, softcap;
};
template <bool BF16> static __device__ __forceinline__ float cache_f32(const char *p) {
    const uint32_t b = *reinterpret_cast<const uint16_t *>(p);
    return BF16 ? bf16_bits_to_float(b) : half_bits_to_float(b);
}
// One workgroup per (KV head, sequence), its query heads one after the other; a wave takes every fourth slot, a lane D / 64 elements of the row.
template <bool BF16> __global__ void __launch_bounds__(256) paged_attn_kernel(AttnArgs a) {
    __shared__ float s_m[4], s_l[4], s_o[4][256];
    const int hk = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.c.D / 64;
    const int n = paged_len(a.c, s), mask = (1 << a.c.page_shift) - 1;
    auto score = [&](const float *q, int j, int page) {
        const char *kr = a.c.k + (long)page * a.c.k_page + (long)hk * a.c.k_head + (long)(j & mask) * a.c.k_row;
        float d = 0.f;
        for (int e = 0; e < E; ++e) d = fmaf(q[e], cache_f32<BF16>(kr + 2 * (lane * E + e)), d);
        d = wave_sum_dpp(d) * a.scale;
        return a.softcap != 0.f ? a.softcap * tanhf(d / a.softcap) : d;
    };
    for (int g = 0; g < a.group; ++g) {
        const int h = hk * a.group + g;
        float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
        for (int e = 0; e < E; ++e) q[e] = reinterpret_cast<const float *>(a.q + (long)s * a.q_seq + (long)h * a.q_head)[lane * E + e];
        for (int j = wave; j < n; j += 4) {
            const int page = paged_page(a.c, s, j); if (page < 0) continue;
            const float x = score(q, j, page), mn = fmaxf(m, x), f = expf(m - mn), p = expf(x - mn);
            const char *vr = a.c.v + (long)page * a.c.v_page + (long)hk * a.c.v_head + (long)(j & mask) * a.c.v_row;
            l = l * f + p; m = mn;
            for (int e = 0; e < E; ++e) o[e] = fmaf(p, cache_f32<BF16>(vr + 2 * (lane * E + e)), o[e] * f);
        }
        __syncthreads();
        if (lane == 0) { s_m[wave] = m; s_l[wave] = l; }
        for (int e = 0; e < E; ++e) s_o[wave][lane * E + e] = o[e];
        __syncthreads();
        float M = -INFINITY, L = 0.f;
        for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w]);
        for (int w = 0; w < 4; ++w) L += s_m[w] == -INFINITY ? 0.f : s_l[w] * expf(s_m[w] - M);
        float *out = reinterpret_cast<float *>(a.dst + (long)s * a.d_seq + (long)h * a.d_head);
        for (int d = threadIdx.x; d < a.c.D; d += 256) {
            float v = 0.f;
            for (int w = 0; w < 4; ++w) v += s_m[w] == -INFINITY ? 0.f : s_o[w][d] * expf(s_m[w] - M);
            out[d] = L > 0.f || L != L ? v / L : 0.f;
        }
        if (a.weight && M != -INFINITY) {
            float *wr = reinterpret_cast<float *>(a.weight + (long)s * a.w_seq + (long)hk * a.w_head);
            for (int j = wave; j < n; j += 4) {
                const int page = paged_page(a.c, s, j); if (page < 0) continue;
                const float x = score(q, j, page);
                if (lane == 0) wr[j] += expf(x - M) / L;
            }
        }
    }
}
static int64_t attn_check(const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *dst, AttnArgs *a) {
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
    a->group = (int)(q->ne[1] / a->c.n_head_kv);
    return 0;
}
int64_t cdna4_paged_attn_workspace(const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const cdna4_tensor *weight, const cdna4_tensor *dst) {
    AttnArgs a; return attn_check(q, k_cache, v_cache, table, weight, dst, &a);
}
int cdna4_op_paged_attn(cdna4_context *ctx, const cdna4_tensor *q, const cdna4_tensor *k_cache, const cdna4_tensor *v_cache, const cdna4_tensor *table, const int32_t *n_kv, const cdna4_tensor *weight,
                        const cdna4_tensor *dst, float scale, float softcap, void *stream) {
    ARG_CHECK(ctx, "paged_attn: null argument");
    AttnArgs a; const int64_t bytes = attn_check(q, k_cache, v_cache, table, weight, dst, &a); if (bytes < 0) return (int)bytes;
    if (pg_empty(q)) return CDNA4_OK;
    ARG_CHECK(n_kv && q->data && dst->data && (a.c.W == 0 || (a.c.table && (!weight || weight->data))), "paged_attn: null data");
    ARG_CHECK(!pg_overlap(q, 4, dst, 4) && (!weight || a.c.W == 0 || (!pg_overlap(weight, 4, dst, 4) && !pg_overlap(weight, 4, q, 4))), "paged_attn: q, dst and weight may not overlap");
    a.c.n_kv = n_kv; a.scale = scale; a.softcap = softcap;
    a.q = (const char *)q->data; a.q_head = q->nb[1]; a.q_seq = q->nb[2]; a.dst = (char *)dst->data; a.d_head = dst->nb[1]; a.d_seq = dst->nb[2];
    a.weight = weight ? (char *)weight->data : nullptr; a.w_head = weight ? weight->nb[1] : 0; a.w_seq = weight ? weight->nb[2] : 0;
    DEVICE_SCOPE(ctx);
    const dim3 grid((unsigned)a.c.n_head_kv, (unsigned)a.c.n_seq);
    if (k_cache->type == CDNA4_TYPE_BF16) hipLaunchKernelGGL(paged_attn_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(paged_attn_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}
