// beam.hip -- one step of a beam search: the best continuations over beams and vocabulary.
#include "paged.cuh"
#include "fa_decode.cuh"
#include <algorithm>

struct BeamArgs {
    const char *logits; long row; const float *score; const int *done; int n_beam, n_out, pad; long n_vocab;
    float *score_out; int *parent, *token; double *top, *lse;        // largest logit and log sum exp (x - top) of every row
};
// the largest logit of every row and the log of its sum of exponentials, in 64 bits from the 32-bit sum
__global__ void __launch_bounds__(1024) beam_lse_kernel(BeamArgs a) {
    __shared__ float red[16];
    const float *x = reinterpret_cast<const float *>(a.logits + (long)blockIdx.x * a.row);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY;
    for (long i = threadIdx.x; i < a.n_vocab; i += 1024) m = fmaxf(m, x[i]);
    m = wave_max(m);
    if (lane == 0) red[wave] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i]);
    __syncthreads();
    float l = 0.f;
    for (long i = threadIdx.x; i < a.n_vocab; i += 1024) l += expf(x[i] - m);
    l = wave_sum_dpp(l);
    if (lane == 0) red[wave] = l;
    __syncthreads();
    if (threadIdx.x == 0) { double t = 0; for (int i = 0; i < 16; ++i) t += red[i]; a.top[blockIdx.x] = m; a.lse[blockIdx.x] = log(t); }
}
// a candidate and its place in the order: value descending, then beam, logit descending, token (within a beam the value grows with the logit, in 64 bits not always visibly)
struct Cand { double c; float x; int b, t; };
static __device__ __forceinline__ bool before(const Cand &p, const Cand &q) {
    if (p.c != q.c) return p.c > q.c;
    if (p.b != q.b) return p.b < q.b;
    if (p.x != q.x) return p.x > q.x;
    return p.t < q.t;
}
static __device__ __forceinline__ Cand shfl(const Cand &p, int d) { Cand q; q.c = __shfl_xor(p.c, d, 64); q.x = __shfl_xor(p.x, d, 64); q.b = __shfl_xor(p.b, d, 64); q.t = __shfl_xor(p.t, d, 64); return q; }
// n_out rounds over a group's candidates: the first one behind the last chosen
__global__ void __launch_bounds__(1024) beam_pick_kernel(BeamArgs a) {
    __shared__ Cand s_c[16];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Cand last = {};
    for (int o = 0; o < a.n_out; ++o) {
        Cand best = {-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
        for (int b = 0; b < a.n_beam; ++b) {
            const int r = g * a.n_beam + b; const float *x = reinterpret_cast<const float *>(a.logits + (long)r * a.row);
            const bool done = a.done && a.done[r];
            for (long t = threadIdx.x; t < a.n_vocab; t += 1024) {
                Cand q = {done ? (t == a.pad ? (double)a.score[r] : -INFINITY) : (double)a.score[r] + (((double)x[t] - a.top[r]) - a.lse[r]), done ? 0.f : x[t], b, (int)t};
                if (q.c != q.c || q.c == -INFINITY) { q.c = -INFINITY; q.x = -INFINITY; }
                if (o && !before(last, q)) continue;
                if (before(q, best)) best = q;
            }
        }
        for (int d = 32; d; d >>= 1) { const Cand q = shfl(best, d); if (before(q, best)) best = q; }
        __syncthreads();
        if (lane == 0) s_c[wave] = best;
        __syncthreads();
        best = s_c[0];
        for (int w = 1; w < 16; ++w) if (before(s_c[w], best)) best = s_c[w];
        last = best;
        if (threadIdx.x == 0) {
            const long k = (long)g * a.n_out + o;
            a.score_out[k] = (float)best.c; a.parent[k] = g * a.n_beam + best.b; a.token[k] = best.t;
        }
    }
}
static int64_t beam_check(const cdna4_tensor *x, int n_beam, int n_out, int pad, BeamArgs *a) {
    ARG_CHECK(x, "beam_select: null argument");
    ARG_CHECK(pg_sizes_ok(x) && x->type == CDNA4_TYPE_F32 && x->ne[0] >= 1 && x->ne[2] == 1 && x->ne[3] == 1, "beam_select: logits f32 [n_vocab, n_group * n_beam]");
    OP_CHECK(x->nb[0] == 4 && x->nb[1] % 4 == 0 && (uintptr_t)x->data % 4 == 0, "beam_select: dense rows");
    OP_CHECK(n_beam >= 1 && n_beam <= 256 && x->ne[0] * n_beam < (1l << 31) && x->ne[1] <= (1l << 20), "beam_select: 1 to 256 beams, n_beam * n_vocab < 2^31, at most 2^20 rows");
    ARG_CHECK(x->ne[1] % n_beam == 0, "beam_select: rows are groups of n_beam");
    OP_CHECK(n_out >= 1 && n_out <= 64 && n_out <= x->ne[0] * n_beam, "beam_select: 1 <= n_out <= min(64, n_beam * n_vocab)");
    ARG_CHECK(pad >= 0 && pad < x->ne[0], "beam_select: pad is a token");
    a->logits = (const char *)x->data; a->row = x->nb[1]; a->n_vocab = x->ne[0]; a->n_beam = n_beam; a->n_out = n_out; a->pad = pad;
    return x->ne[1] * 16;
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
    a.top = (double *)ctx->ws; a.lse = a.top + rows;
    hipLaunchKernelGGL(beam_lse_kernel, dim3((unsigned)rows), dim3(1024), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(beam_pick_kernel, dim3((unsigned)(rows / n_beam)), dim3(1024), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError()); return CDNA4_OK;
}
