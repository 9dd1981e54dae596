"""-m gpu: how far the paged attention is from 64 bits, beside elementary 32-bit torch on the same inputs, and that finite cache values give finite rows.

The bound of tests/paged_ref.py holds element by element and grows with the worst case of every product; here the root mean square of the error (relative to sum p |v| of the element, for
the gathered weights to p) may be at most twice that of the 32-bit form (measured in the same run) plus 2^-24, half a step of the result.  An emulation of the kernel's arithmetic on the same
kind of inputs puts it at 0.3 to 0.9 of the 32-bit form's; without any one term of a query or of a probability it is 3 times (third bf16 term of p) to 5000 times that."""
import numpy as np
import pytest
import torch

from test_gpu_paged import Case, g, host

pytestmark = pytest.mark.gpu


def plain(c, q, scale, softcap, dtype):
    """-> per sequence (out, p, sum p |v|) in `dtype`, elementary operations on the host"""
    kh, vh, table, n_kv = c.host()
    res = []
    for s, n in enumerate(n_kv):
        n = max(int(n), 0); pages = table[s, :-(-n // c.page)] if n else table[s, :0]
        k, v = (torch.from_numpy(np.ascontiguousarray(x[pages].transpose(1, 0, 2, 3).reshape(c.heads_kv, -1, c.D)[:, :n])).to(dtype) for x in (kh, vh))
        x = torch.from_numpy(q[s]).to(dtype).view(c.heads_kv, -1, c.D)
        z = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
        z = softcap * torch.tanh(z / softcap) if softcap else z
        if not n:
            res.append((torch.zeros(q.shape[1], c.D, dtype=dtype), z.reshape(q.shape[1], 0), torch.ones(q.shape[1], c.D, dtype=dtype))); continue
        p = torch.exp(z - z.amax(2, keepdim=True)); p = p / p.sum(2, keepdim=True)
        res.append((torch.matmul(p, v).reshape(q.shape[1], c.D), p.reshape(q.shape[1], n), torch.matmul(p, v.abs()).reshape(q.shape[1], c.D)))
    return res


def rms(x):
    return float(np.sqrt(np.mean(np.square(np.concatenate([np.asarray(y, dtype=np.float64).reshape(-1) for y in x])))))


def check(be, c, heads, q, softcap=0.0, weights=False, extra=0.0):
    scale = float(np.float32(c.D ** -0.5))
    weight = torch.zeros(len(c.n_kv), c.heads_kv, c.W * c.page, device="cuda") if weights else None
    got = host(be.paged_attn(g(q), *c.dev(), scale=scale, softcap=softcap, weight=weight))
    exact, single = plain(c, q, scale, softcap, torch.float64), plain(c, q, scale, softcap, torch.float32)
    mine = rms([(got[s] - e[0].numpy()) / e[2].clamp(min=1e-300).numpy() for s, e in enumerate(exact)])
    other = rms([(f[0].double() - e[0]).numpy() / e[2].clamp(min=1e-300).numpy() for e, f in zip(exact, single)])
    assert mine <= 2 * other + 2.0 ** -24 + extra, (mine, other)
    if weights:
        w, group = host(weight), heads // c.heads_kv
        def of(x):
            return x.double().view(c.heads_kv, group, -1).sum(1).numpy()
        least = 1e-6          # (of slots that carry nothing the 32-bit exponential has no digits either)
        mine = rms([(w[s][:, :e[1].shape[1]] - of(e[1])) / np.maximum(of(e[1]), least) for s, e in enumerate(exact)])
        other = rms([(of(f[1]) - of(e[1])) / np.maximum(of(e[1]), least) for e, f in zip(exact, single)])
        assert mine <= 2 * other + 2.0 ** -24, (mine, other)


def queries(c, heads, size):
    return c.rng.standard_normal((len(c.n_kv), heads, c.D)).astype(np.float32) * np.float32(size)


# (heads on KV heads, slots of the table): a workgroup per unit, shared tiles with a join, 32 heads to a wave
FORMS = {"unit": (2, 16, 0), "shared": (2, 16, 2500), "blocks": (1, 40, 2500)}


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("weights", [False, True])
def test_peaked_rows_are_as_close_as_32_bits(weights, D, dtype, form, backend):
    """scores of a few units: a handful of slots carry a row, so that no error averages out"""
    heads_kv, heads, most = FORMS[form]
    lens = [5, 20, 40, 100, 200, 0, 1] + ([most] if most else [])
    c = Case(lens, D=D, dtype=dtype, heads_kv=heads_kv, page=16, W=None if most else 14, seed=D)
    check(backend, c, heads, queries(c, heads, 6.0), weights=weights)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
def test_peaked_rows_with_32_heads_to_a_wave(D, dtype, backend):
    W = 64 * D // 64 + 1
    n_seq = 140 if D == 64 else 70
    lens = [int(x) for x in np.random.default_rng(D).integers(1, 200, n_seq)]
    c = Case(lens, D=D, heads_kv=1, page=64, dtype=dtype, seed=D)
    c.table = np.concatenate([c.table, np.full((n_seq, W - c.W), -1, np.int32)], axis=1); c.W = W
    check(backend, c, 32, queries(c, 32, 6.0), weights=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_long_rows_are_as_close_as_32_bits(softcap, dtype, backend):
    c = Case([9001, 4000, 700, 3], dtype=dtype, page=64, seed=3)
    check(backend, c, 8, queries(c, 8, 1.5), softcap=softcap, weights=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,n", [(64, 300), (128, 2048), (128, 8192), (256, 3000)])
@pytest.mark.parametrize("share", [0.9, 0.999, 0.999999])
def test_a_sink_of_no_value_leaves_the_others_their_digits(share, D, n, dtype, backend):
    """one slot takes nearly all the weight and its value is zero: the rest is the sum of many small probabilities.  All of a row's elements share the error of the sink's score (16 to 32 in
    units of log 2: up to four half steps of 2^-20, 2^-19 of the row): with values of both signs that is |sum p v| / sum p |v| ~ 1.25 / sqrt(n) of it"""
    c = Case([n], D=D, heads_kv=2, dtype=dtype, page=16, seed=n)
    q = queries(c, 4, 1.0)
    at = int(c.table[0, 0])
    for h in range(2):          # the first slot's key along the first of the head's two queries, as long as that share needs
        d = q[0, 2 * h].astype(np.float64); z = np.log(share / (1 - share) * n)
        c.k[at, h, 0] = g((d / (d @ d) * z * D ** 0.5).astype(np.float32)).to(dtype)
        q[0, 2 * h + 1] = q[0, 2 * h] * np.float32(1.01)
    c.v[at, :, 0] = 0.0
    check(backend, c, 4, q, extra=2.0 ** -19 * 1.25 / n ** 0.5)
    c.v[:] = 1.0; c.v[at, :, 0] = 0.0          # all others alike: what is always rounded one way adds up
    check(backend, c, 4, q, extra=2.0 ** -19)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [200, 3000])
def test_a_large_element_that_meets_zeros_leaves_the_others_their_digits(n, dtype, backend):
    """a query with one very large element where all keys are zero"""
    c = Case([n, 7], heads_kv=1, dtype=dtype, page=16, seed=n)
    c.k[:, :, :, 5] = 0.0
    q = queries(c, 4, 3.0); q[:, :, 5] = 1e7
    check(backend, c, 4, q, weights=True)


@pytest.mark.parametrize("form", ["unit", "shared", "blocks", "two"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("weights", [False, True])
def test_finite_bf16_values_give_finite_rows(weights, D, form, backend):
    """bf16 holds values up to the largest f32: their weighted mean is no larger than they are, whatever is summed on the way"""
    if form == "two":
        if D == 256:
            pytest.skip("heads of 256 take 16 to a wave")
        W = 64 * D // 64 + 1
        heads_kv, heads, lens = 1, 32, [int(x) for x in np.random.default_rng(D).integers(1, 400, 140 if D == 64 else 70)]
        lens[3] = 2100
    else:
        heads_kv, heads, most = FORMS[form]
        lens, W = [5, 200, 1, 33] + ([most, 9001] if most else []), None
    most = torch.finfo(torch.bfloat16).max
    for kind in ("equal", "rising", "signs", "small"):
        c = Case(lens, D=D, heads_kv=heads_kv, dtype=torch.bfloat16, page=64, seed=D)
        if W:
            c.table = np.concatenate([c.table, np.full((len(lens), W - c.W), -1, np.int32)], axis=1); c.W = W
        q = queries(c, heads, 1.5)
        sign = torch.sign(torch.randn(c.v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
        live = ~c.v.isnan()
        if kind == "equal":
            c.k[live] = 0.0; c.v[live] = most
        elif kind == "rising":          # every slot's score above the one before, slowly: the maximum is always new
            q[:] = 1.0
            for s, n in enumerate(lens):
                j = torch.arange(n, device="cuda"); page = g(c.table[s])[j // c.page].long()
                c.k[page, :, j % c.page] = (j * (min(0.05, 100.0 / n) / D ** 0.5))[:, None, None].to(torch.bfloat16).expand(n, heads_kv, D).contiguous()
            c.v[live] = most
        elif kind == "signs":
            c.v[live] = (sign * most)[live].to(torch.bfloat16)
        else:
            c.v.copy_((c.v.float() * 2.0 ** -100).to(torch.bfloat16))
        out = host(backend.paged_attn(g(q), *c.dev(), weight=torch.zeros(len(lens), heads_kv, c.W * c.page, device="cuda") if weights else None))
        exact = plain(c, q, float(np.float32(D ** -0.5)), 0.0, torch.float64)
        for s, e in enumerate(exact):          # 2^-15: some thousand half steps, far above the error of 32 bits and far below any overflow or underflow
            assert (np.abs(out[s] - e[0].numpy()) <= 2.0 ** -15 * e[2].numpy()).all(), (kind, s)
