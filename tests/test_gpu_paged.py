"""-m gpu: decoding over a paged key / value cache (store, attention of one new token, eviction by gathered weight, fork along beams) against tests/paged_ref.py in 64 bits on the same
inputs.  Whole numbers, moved and rounded values are equal bit for bit; the attention lies within the bound that paged_ref.attn derives for every element."""
import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def g(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype).to(DEV)


def host(x):
    return x.detach().cpu().double().numpy() if x.is_floating_point() else x.detach().cpu().numpy()


class Case:
    """A cache with random contents, private pages in a random order and the sequences' lengths.  junk: what every slot that is not in use holds."""

    def __init__(self, lens, D=128, heads_kv=2, page=16, dtype=torch.float16, token_major=False, W=None, seed=0, junk=float("nan"), spare=3):
        r = self.rng = np.random.default_rng(seed)
        self.page, self.D, self.heads_kv = page, D, heads_kv
        n_seq, most = len(lens), max([0] + list(lens))
        self.W = W if W is not None else -(-most // page) + 1
        self.n_pages = n_seq * self.W + spare
        perm = r.permutation(self.n_pages).astype(np.int32)
        self.table = perm[:n_seq * self.W].reshape(n_seq, self.W).copy()
        self.spare = perm[n_seq * self.W:].copy()
        self.n_kv = np.array(lens, np.int32)
        shape = (self.n_pages, page, heads_kv, D) if token_major else (self.n_pages, heads_kv, page, D)
        used = np.zeros((self.n_pages, page), bool)
        for s, n in enumerate(lens):
            for j in range(min(max(n, 0), self.W * page)):
                used[self.table[s, j // page], j % page] = True
        self.caches = []
        for _ in "kv":
            x = torch.from_numpy(r.standard_normal(shape).astype(np.float32)).to(dtype)
            u = torch.from_numpy(used)[:, :, None, None] if token_major else torch.from_numpy(used)[:, None, :, None]
            x = torch.where(u, x, torch.tensor(junk, dtype=dtype)).to(DEV)
            self.caches.append(x.transpose(1, 2) if token_major else x)
        self.k, self.v = self.caches

    def slots(self, extra=0, pos=False):
        n = self.W * self.page + extra
        if pos:
            return g(np.argsort(self.rng.random((len(self.n_kv), self.heads_kv, n)), axis=-1).astype(np.int32))
        return g(self.rng.random((len(self.n_kv), self.heads_kv, n)).astype(np.float32))

    def dev(self):
        return self.k, self.v, g(self.table), g(self.n_kv)

    def host(self):
        return host(self.k), host(self.v), self.table, self.n_kv


def check_attn(be, c, heads, scale=None, softcap=0.0, weight=None, q=None, out=None, call=None):
    q = g(c.rng.standard_normal((len(c.n_kv), heads, c.D)).astype(np.float32) * 1.5) if q is None else q
    w0 = None if weight is None else host(weight)
    k, v, table, n_kv = c.dev()
    got = be.paged_attn(q, k, v, table, n_kv, scale=scale, softcap=softcap, weight=weight, out=out)
    if w0 is not None:
        w0 = w0.copy()
    want, tol, wtol = ref.attn(host(q), *c.host(), scale=c.D ** -0.5 if scale is None else scale, softcap=softcap, weight=w0)
    bad = ~(np.abs(host(got) - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], host(got)[bad][:4], want[bad][:4], tol[bad][:4])
    if weight is not None:
        bad = ~(np.abs(host(weight) - w0) <= wtol)
        assert not bad.any(), (np.argwhere(bad)[:4], host(weight)[bad][:4], w0[bad][:4])
    return got


@pytest.mark.parametrize("heads_kv,heads", [(1, 1), (2, 6), (1, 8), (2, 14), (1, 16), (1, 17), (2, 40), (1, 71)])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.float16)])
def test_attn_groups_of_short_tables(D, dtype, heads_kv, heads, weights, backend):
    c = Case([37, 0, 200, 511], D=D, dtype=dtype, heads_kv=heads_kv, page=16, W=32, seed=heads)
    check_attn(backend, c, heads, weight=c.slots() if weights else None, softcap=15.0 if heads % 2 else 0.0)


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_attn_lengths(D, page, dtype, backend):
    check_attn(backend, Case(LENS, D=D, page=page, dtype=dtype, seed=D + page), heads=8, weight=None)


@pytest.mark.parametrize("D,heads_kv,heads,dtype", [(64, 1, 17, torch.float16), (128, 2, 40, torch.bfloat16), (256, 1, 33, torch.float16), (64, 1, 300, torch.bfloat16), (128, 3, 60, torch.float16)])
@pytest.mark.parametrize("weights", [False, True])
def test_attn_large_groups_over_long_tables(D, heads_kv, heads, dtype, weights, backend):
    """the blocks of 16 heads of a group have workgroups of their own: rows of many and of no tiles, more blocks than workgroups to a block"""
    c = Case([2700, 0, 129, 1], D=D, heads_kv=heads_kv, page=64, dtype=dtype, seed=heads)
    check_attn(backend, c, heads, weight=c.slots() if weights else None, softcap=20.0 if D == 256 else 0.0)


@pytest.mark.parametrize("D,heads_kv,heads,n_seq,dtype", [(64, 2, 40, 80, torch.float16), (64, 1, 32, 140, torch.bfloat16), (128, 1, 17, 66, torch.bfloat16), (128, 2, 62, 40, torch.float16), (128, 1, 31, 70, torch.float16)])
@pytest.mark.parametrize("weights", [False, True])
def test_attn_two_blocks_of_heads_to_a_wave(D, heads_kv, heads, n_seq, dtype, weights, backend):
    """groups of 17 to 32 heads and tables of many slots, of which few are in use"""
    W = 64 * D // 64 + 1
    r = np.random.default_rng(heads)
    lens = [int(x) for x in r.integers(0, 300, n_seq)]; lens[3] = 2100; lens[7] = 0; lens[8] = -1
    c = Case([max(n, 0) for n in lens], D=D, heads_kv=heads_kv, page=64, dtype=dtype, seed=heads)
    c.n_kv = np.array(lens, np.int32)
    c.table = np.concatenate([c.table, np.full((n_seq, W - c.W), c.n_pages, np.int32)], axis=1); c.W = W          # (wider tables: nothing behind the lengths is mapped)
    c.table[5, 0] = -1
    check_attn(backend, c, heads, weight=c.slots() if weights else None, softcap=25.0 if D == 64 else 0.0)


@pytest.mark.parametrize("heads_kv,heads", [(1, 1), (2, 2), (8, 8), (2, 6), (1, 8), (2, 14), (1, 16), (1, 17), (2, 40), (1, 71), (3, 12)])
@pytest.mark.parametrize("weights", [False, True])
def test_attn_groups(heads_kv, heads, weights, backend):
    c = Case([37, 0, 200, 513], heads_kv=heads_kv, page=32, seed=heads)
    check_attn(backend, c, heads, weight=c.slots() if weights else None)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("page", [16, 128, 4096])
def test_attn_pages_and_layouts(page, token_major, dtype, backend):
    c = Case([1, 700, 130, 4097 if page == 4096 else 260], heads_kv=2, page=page, token_major=token_major, dtype=dtype, seed=page)
    check_attn(backend, c, 8, softcap=20.0, weight=c.slots(extra=5))


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16)])
def test_attn_long_and_many(D, dtype, backend):
    """long rows are split over many workgroups and joined; a batch of many short ones shares a workgroup"""
    check_attn(backend, Case([9001, 3], D=D, page=64, dtype=dtype, seed=1), 8)
    c = Case([int(x) for x in np.random.default_rng(2).integers(0, 70, 300)], D=D, heads_kv=1, page=16, dtype=dtype, seed=2)
    check_attn(backend, c, 4, weight=c.slots())
    c = Case([2500, 0, 2500, 1], D=D, heads_kv=4, page=256, dtype=dtype, seed=3)
    check_attn(backend, c, 16, weight=c.slots())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attn_most_lds(dtype, backend):
    """the largest heads in groups of 16 and more, next to a long vector of lengths"""
    for n_seq, heads in ((3, 32), (900, 16)):
        c = Case([int(x) for x in np.random.default_rng(n_seq).integers(0, 40, n_seq)], D=256, heads_kv=1, page=16, dtype=dtype, seed=6)
        check_attn(backend, c, heads, softcap=30.0 if n_seq == 3 else 0.0, weight=c.slots())


def test_attn_many_sequences(backend):
    lens = [int(x) for x in np.random.default_rng(5).integers(0, 5, 700)]
    lens[477] = 700
    c = Case(lens, D=64, heads_kv=1, page=16, W=44, seed=4)
    check_attn(backend, c, 2, weight=c.slots())


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_attn_unmapped_pages_inactive_rows_and_oversized_lengths(junk, backend):
    c = Case([100, 100, 64, 90, 33], page=16, W=7, seed=7, junk=junk)
    c.table[0, 2] = -1; c.table[0, 6] = 1 << 30; c.table[2, :] = -5; c.table[4, 0] = c.n_pages        # holes, the last page, everything, the first page
    c.n_kv[1] = -3                                                                                   # inactive
    c.n_kv[3] = 1000                                                                                 # beyond the table: every slot
    for x in c.caches:
        x[g(c.table[3].astype(np.int64))] = 0.25
    out = check_attn(backend, c, 4, weight=c.slots())
    assert (host(out)[[1, 2]] == 0).all()


@pytest.mark.parametrize("size", [2e-6, 2e4])
def test_attn_smallest_and_largest_cache_values(size, backend):
    """f16 subnormals (K and V of 10^-6) and rows near the largest f16 keep their value: the bound of every element is relative to |k| and |v|"""
    for lens in ([300, 64], [2100, 2000]):
        c = Case(lens, seed=15, junk=0.0)
        for x in c.caches:
            x.copy_((x.float() * size).clamp(-65504, 65504).half())
        check_attn(backend, c, 8, scale=0.5 / size, weight=c.slots())


def test_attn_extreme_queries_and_masses(backend):
    """queries of very different sizes (one of zeros among them), a token that takes all the weight, equal scores"""
    c = Case([257, 257, 257, 40], seed=8)
    q = c.rng.standard_normal((4, 8, 128)).astype(np.float32)
    q[0] *= 1e-20; q[1, :, 3:] = 0; q[1, :, :3] *= 3e4; q[2] = 0; q[3, ::2] *= 100
    check_attn(backend, c, 8, q=g(q), weight=c.slots())
    check_attn(backend, c, 8, q=g(q), scale=-0.7, softcap=5.0)
    check_attn(backend, c, 8, q=g(q), scale=0.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attn_a_query_that_is_no_number_stays_in_its_row(dtype, backend):
    for lens in ([300, 40], [3000, 2000]):
        c = Case(lens, dtype=dtype, seed=11)
        q = c.rng.standard_normal((2, 8, 128)).astype(np.float32)
        want, tol, _ = ref.attn(q.astype(np.float64), *c.host(), scale=0.1)
        q[0, 1] = np.nan; q[1, 6, 5] = np.nan; q[1, 0, 0] = np.inf
        got = host(backend.paged_attn(g(q), *c.dev(), scale=0.1))
        bad = np.zeros((2, 8), bool); bad[0, 1] = bad[1, 6] = bad[1, 0] = True
        assert np.isnan(got[bad]).all() and (np.abs(got - want) <= tol)[~bad].all()


def test_attn_queries_near_the_largest_float(backend):
    """f16 terms of a query are taken of q scaled by a power of two, whatever its size"""
    c = Case([300, 40], seed=16)
    for size in (3e38, 1e36, 1e30, 1e-30):
        q = c.rng.uniform(-1, 1, (2, 8, 128)).astype(np.float32) * np.float32(size)
        check_attn(backend, c, 8, q=g(q), scale=float(np.float32(0.1) / np.float32(size)) if size < 1e37 else 1e-37)


def test_attn_weights_of_a_row_that_is_no_number(backend):
    """NaN reaches the slots that were attended to and no others"""
    for lens, W in (([100], 7), ([3000], 190)):
        c = Case(lens, page=16, W=W, seed=17)
        c.table[0, 2] = -1
        q = c.rng.standard_normal((1, 4, 128)).astype(np.float32); q[0, 1] = np.nan          # heads 0, 1 share the first KV head
        k, v, table, n_kv = c.dev(); w = c.slots(); before = w.clone()
        backend.paged_attn(g(q), k, v, table, n_kv, weight=w)
        n = lens[0]; hole = slice(32, 48)
        assert torch.equal(w[0, :, hole], before[0, :, hole]) and torch.equal(w[0, :, n:], before[0, :, n:])
        seen = torch.ones(n, dtype=torch.bool, device=DEV); seen[hole] = False
        assert w[0, 0, :n][seen].isnan().all() and not w[0, 1].isnan().any()


def test_attn_strided_arguments(backend):
    c = Case([70, 5, 129], heads_kv=2, page=32, seed=9)
    wide = g(c.rng.standard_normal((3, 24, 128)).astype(np.float32))
    out = torch.full((3, 2, 8, 128), 7.0, device=DEV)
    weight = c.slots(extra=11)
    untouched = weight.clone()
    check_attn(backend, c, 8, q=wide[:, 8:16], out=out[:, 1], weight=weight)
    assert (out[:, 0] == 7).all()
    for s, n in enumerate(c.n_kv):
        assert torch.equal(weight[s, :, n:], untouched[s, :, n:])
    table = torch.full((3, c.W + 9), -1, dtype=torch.int32, device=DEV)                  # rows of a wider table, heads cut from a wider cache
    table[:, :c.W] = g(c.table)
    got = backend.paged_attn(wide[:, :4].contiguous(), c.k[:, 1:], c.v[:, 1:], table[:, :c.W], g(c.n_kv))
    want, tol, _ = ref.attn(host(wide[:, :4]), host(c.k[:, 1:]), host(c.v[:, 1:]), c.table, c.n_kv, 128 ** -0.5)
    assert (np.abs(host(got) - want) <= tol).all()


def test_attn_past_32_bit_offsets(backend):
    """a pool of more than 4 GiB (K and V in one allocation), the pages of the sequence spread from its first to its last byte"""
    page, heads_kv, D, n_pages = 4096, 8, 128, 300
    pool = torch.zeros(n_pages, 2, heads_kv, page, D, dtype=torch.float16, device=DEV)             # 5 GB
    table = torch.tensor([[299, 0, 150]], dtype=torch.int32, device=DEV)
    for p in table[0].tolist():
        pool[p] = torch.randn(2, heads_kv, page, D, device=DEV).half()
    n, k, v = 2 * page + 77, pool[:, 0], pool[:, 1]
    q = torch.randn(1, 16, D, device=DEV)
    got = backend.paged_attn(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV))
    small = [pool[table[0].long(), i].cpu().double().numpy() for i in (0, 1)]
    want, tol, _ = ref.attn(host(q), small[0], small[1], np.array([[0, 1, 2]]), [n], D ** -0.5)
    assert (np.abs(host(got) - want) <= tol).all()


def test_attn_repeats_bit_for_bit_on_another_stream_and_in_a_graph(backend):
    c = Case([3000, 17, 0, 999], heads_kv=4, page=64, seed=10, W=64)
    k, v, table, n_kv = c.dev()
    q = g(c.rng.standard_normal((4, 16, 128)).astype(np.float32)); w0 = c.slots()
    base_w = w0.clone(); base = backend.paged_attn(q, k, v, table, n_kv, weight=base_w)
    for _ in range(3):
        w = w0.clone()
        assert torch.equal(backend.paged_attn(q, k, v, table, n_kv, weight=w), base) and torch.equal(w, base_w)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        w = w0.clone(); out = backend.paged_attn(q, k, v, table, n_kv, weight=w)
    other.synchronize()
    assert torch.equal(out, base) and torch.equal(w, base_w)
    backend.reserve_workspace(backend.paged_workspace(q, k, v, table, weight=w0))
    graph = torch.cuda.CUDAGraph(); w = w0.clone(); out = torch.empty_like(base)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        backend.paged_attn(q, k, v, table, n_kv, weight=w, out=out)
    for n in ([3000, 17, 0, 999], [4096, 1, 64, 0], [1, 2, 3, 4], [3000, 17, 0, 999]):               # the lengths live on the device: one graph serves all
        n_kv.copy_(g(np.array(n, np.int32))); w.copy_(w0); graph.replay(); torch.cuda.synchronize()
        w2 = w0.clone(); eager = backend.paged_attn(q, k, v, table, n_kv, weight=w2)
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(eager)) and torch.equal(torch.nan_to_num(w), torch.nan_to_num(w2))


# ---- store
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("D,heads_kv", [(64, 1), (128, 8), (256, 3)])
def test_store(D, heads_kv, token_major, dtype, backend):
    c = Case([0, 5, 16, 30, 47], D=D, heads_kv=heads_kv, token_major=token_major, dtype=dtype, seed=D, junk=1.0, W=5)
    counts = [1, 0, 37, 3, 40]                                           # the last one passes the end of its table: 33 of 40 fit
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    k, v = (c.rng.standard_normal((start[-1] + 2, heads_kv, D)).astype(np.float32) for _ in "kv")    # two rows behind the last sequence
    n_past = np.array([9, 8, 7, 1 << 20, 0], np.int32)
    weight, pos = c.slots(), c.slots(pos=True)
    kh, vh, _, _ = c.host(); wh, ph = host(weight), host(pos)
    want = ref.store(torch.from_numpy(k).to(dtype).double().numpy(), torch.from_numpy(v).to(dtype).double().numpy(), kh, vh, c.table, c.n_kv, start, n_past, wh, ph)
    kc, vc, table, n_kv = c.dev()
    got = backend.paged_store(g(k), g(v), kc, vc, table, n_kv, start=g(start), n_past=g(n_past), weight=weight, pos=pos)
    np.testing.assert_array_equal(host(got), want)
    for a, b in ((kc, kh), (vc, vh), (weight, wh), (pos, ph)):
        np.testing.assert_array_equal(host(a), b)


@pytest.mark.parametrize("D,heads_kv", [(64, 1), (64, 2), (64, 3), (128, 1), (128, 3), (64, 5), (256, 1), (256, 2), (64, 8), (128, 5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_store_of_few_heads(D, heads_kv, dtype, backend):
    """several tokens to a workgroup: sequences of none, one and many of them, tokens before the first and behind the last sequence, one token each"""
    counts = [0, 0, 1, 70, 0, 3, 1, 1, 0, 17, 129, 0]
    c = Case([5, 0, 16, 30, 1, -1, 15, 0, 7, 31, 3, 2], D=D, heads_kv=heads_kv, page=16, dtype=dtype, seed=D + heads_kv, junk=1.0, W=9)
    for lead in (0, 3):
        start = (np.concatenate([[0], np.cumsum(counts)]) + lead).astype(np.int32)
        k, v = (c.rng.standard_normal((start[-1] + 5, heads_kv, D)).astype(np.float32) for _ in "kv")
        n_past = np.arange(12, dtype=np.int32) * 11
        weight, pos = c.slots(), c.slots(pos=True)
        kh, vh, _, _ = c.host(); wh, ph = host(weight), host(pos)
        want = ref.store(torch.from_numpy(k).to(dtype).double().numpy(), torch.from_numpy(v).to(dtype).double().numpy(), kh, vh, c.table, c.n_kv, start, n_past, wh, ph)
        kc, vc, table, n_kv = c.dev()
        got = backend.paged_store(g(k), g(v), kc, vc, table, n_kv, start=g(start), n_past=g(n_past), weight=weight, pos=pos)
        np.testing.assert_array_equal(host(got), want)
        for a, b in ((kc, kh), (vc, vh), (weight, wh), (pos, ph)):
            np.testing.assert_array_equal(host(a), b)
    k, v = (c.rng.standard_normal((12, heads_kv, D)).astype(np.float32) for _ in "kv")
    kh, vh, _, _ = c.host()
    want = ref.store(torch.from_numpy(k).to(dtype).double().numpy(), torch.from_numpy(v).to(dtype).double().numpy(), kh, vh, c.table, c.n_kv)
    np.testing.assert_array_equal(host(backend.paged_store(g(k), g(v), kc, vc, table, n_kv)), want)
    np.testing.assert_array_equal(host(kc), kh); np.testing.assert_array_equal(host(vc), vh)


def test_store_one_token_each_with_inactive_rows_and_missing_pages(backend):
    c = Case([0, 15, 16, 40, 20, 47], junk=0.5, seed=3, W=3)
    c.n_kv[1] = -1; c.n_kv[5] = 48                                       # inactive; full
    c.table[2, 1] = -1; c.table[4, 1] = c.n_pages
    k, v = (c.rng.standard_normal((6, 2, 2, 128)).astype(np.float32) for _ in "kv")
    kh, vh, _, _ = c.host()
    want = ref.store(torch.from_numpy(k[:, 1]).half().double().numpy(), torch.from_numpy(v[:, 1]).half().double().numpy(), kh, vh, c.table, c.n_kv)
    kc, vc, table, n_kv = c.dev()
    got = backend.paged_store(g(k)[:, 1], g(v)[:, 1], kc, vc, table, n_kv)
    np.testing.assert_array_equal(host(got), want)
    np.testing.assert_array_equal(host(kc), kh); np.testing.assert_array_equal(host(vc), vh)


def test_store_rounds_to_nearest_even_and_keeps_what_is_not_finite(backend):
    for dtype in (torch.float16, torch.bfloat16):
        c = Case([0], heads_kv=1, D=64, dtype=dtype, junk=0.0)
        x = torch.tensor([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 65519.0, 65520.0, 1e38, -1e38, float("inf"), float("-inf"), 1e-8, -6e-8, 0.0, -0.0, 3e-5, 1e-40] * 4)
        k, v, table, n_kv = c.dev()
        backend.paged_store(x.view(1, 1, 64).to(DEV), -x.view(1, 1, 64).to(DEV), k, v, table, n_kv)
        at = int(c.table[0, 0])
        assert torch.equal(k[at, 0, 0].cpu().view(torch.int16), x.to(dtype).view(torch.int16)) and torch.equal(v[at, 0, 0].cpu().view(torch.int16), (-x).to(dtype).view(torch.int16))


# ---- evict
def run_evict(be, c, weight, pos, n_past, budget, sink, recent, in_place):
    kh, vh, _, _ = c.host(); w0, p0 = host(weight).astype(np.float32), host(pos)
    want_w, want_p, want_n = ref.evict(kh, vh, c.table, c.n_kv, w0, p0, n_past, budget, sink, recent)
    k, v, table, n_kv = c.dev()
    wo, po = (weight, pos) if in_place else (torch.full_like(weight, -7.0), torch.full_like(pos, -7))
    got = be.paged_evict(k, v, table, n_kv, weight, pos, g(n_past), budget, n_sink=sink, n_recent=recent, weight_out=None if in_place else wo, pos_out=None if in_place else po)
    np.testing.assert_array_equal(host(got), want_n)
    np.testing.assert_array_equal(host(k), kh); np.testing.assert_array_equal(host(v), vh)
    for s, n in enumerate(want_n):
        n = max(int(n), 0)
        for a, b, old in ((wo, want_w, w0), (po, want_p, p0)):
            a = a[s].cpu().numpy()
            np.testing.assert_array_equal(a[:, :n], b[s][:, :n])
            np.testing.assert_array_equal(a[:, n:], old[s][:, n:] if in_place else np.full_like(a[:, n:], -7))
    if not in_place:
        np.testing.assert_array_equal(host(weight).astype(np.float32), w0); np.testing.assert_array_equal(host(pos), p0)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (16, 2, 5), (63, 0, 63), (64, 4, 20), (100, 100, 0), (600, 4, 8)])
def test_evict(budget, sink, recent, in_place, backend):
    c = Case([0, 1, 63, 64, 65, 129, 1000, 601], heads_kv=3, page=16, D=64, seed=budget, junk=0.125)
    run_evict(backend, c, c.slots(extra=3), c.slots(extra=3, pos=True), np.array([5, 1, 70, 64, 90, 129, 1008, 700], np.int32), budget, sink, recent, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_ties_and_values_that_are_no_numbers(in_place, backend):
    """equal weights go by the slot, zeros of both signs are equal, NaN counts as -inf, infinities and negative weights keep their order"""
    values = np.array([0.0, -0.0, np.nan, -np.inf, np.inf, -1.5, 1e-45, 1.0, 1.0, 3e38, -np.nan], np.float32)
    for seed, budget in enumerate((3, 40, 77, 250)):
        c = Case([300, 78, 41, 251], heads_kv=2, page=32, D=64, seed=seed, junk=0.125)
        w = g(values[c.rng.integers(0, len(values), (4, 2, c.W * c.page))])
        run_evict(backend, c, w, c.slots(pos=True), np.array([400, 78, 41, 260], np.int32), budget, 1, 1, in_place)
    c = Case([500], heads_kv=1, page=32, D=64, junk=0.125)
    run_evict(backend, c, torch.zeros_like(c.slots()), c.slots(pos=True), np.array([10 ** 6], np.int32), 77, 0, 0, in_place)


@pytest.mark.parametrize("dtype,token_major,D", [(torch.float16, False, 256), (torch.bfloat16, True, 128)])
@pytest.mark.parametrize("n,budget", [(50000, 1024), (50000, 49000), (9000, 8999), (3000, 2999)])
def test_evict_long(n, budget, dtype, token_major, D, backend):
    c = Case([n, n // 2], heads_kv=1, page=256, D=D, dtype=dtype, token_major=token_major, junk=0.125, seed=n)
    w = torch.exp(3 * torch.randn(2, 1, c.W * c.page, device=DEV))
    run_evict(backend, c, w, c.slots(pos=True), np.array([n + 7, n], np.int32), budget, 4, budget // 3, True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [32769, 40002, 36871])
def test_evict_rows_that_do_not_fit_lds(n, in_place, backend):
    """odd lengths past 32768 slots, weights of which many are equal"""
    c = Case([n, 32768, 32770], heads_kv=1, page=64, D=64, junk=0.125, seed=n)
    w = torch.round(4 * torch.rand(3, 1, c.W * c.page + 3, device=DEV)) / 4
    for budget in (300, 20000):
        run_evict(backend, c, w[:, :, :c.W * c.page].contiguous() if in_place else w, c.slots(pos=True) if in_place else c.slots(extra=3, pos=True), np.array([n + 7, n, 100], np.int32), budget, 4, budget // 3, in_place)


def test_evict_inactive_oversized_unmapped(backend):
    c = Case([100, 100, 60, 112], page=16, W=7, D=64, seed=4, junk=0.125)
    c.n_kv[0] = -2; c.n_kv[1] = 5000; c.table[3, 0] = -1; c.table[3, 5] = 10 ** 9
    run_evict(backend, c, c.slots(), c.slots(pos=True), np.array([100, 100, 60, 100], np.int32), 50, 2, 3, False)


# ---- fork
@pytest.mark.parametrize("dtype,token_major,D,page", [(torch.float16, False, 128, 16), (torch.bfloat16, True, 64, 64), (torch.float16, True, 256, 32)])
def test_fork(dtype, token_major, D, page, backend):
    c = Case([0, 1, page - 1, page, page + 1, 3 * page, 3 * page + 7, 50], D=D, heads_kv=3, page=page, dtype=dtype, token_major=token_major, junk=0.5, spare=30, seed=page)
    c.n_kv[7] = -1
    parent = np.array([0, 1, 2, 3, 4, 5, 6, 7, 6, 6, -1, 8, 4, 4, 2 ** 31 - 1], np.int32)
    fresh = c.spare[:len(parent)].copy()
    fresh[9] = -1; fresh[12] = c.n_pages
    kh, vh, _, _ = c.host()
    want_t, want_n = ref.fork(kh, vh, c.table, c.n_kv, parent, fresh)
    k, v, table, n_kv = c.dev()
    got_t, got_n = backend.paged_fork(k, v, table, n_kv, g(parent), g(fresh))
    np.testing.assert_array_equal(host(got_t), want_t); np.testing.assert_array_equal(host(got_n), want_n)
    np.testing.assert_array_equal(host(k), kh); np.testing.assert_array_equal(host(v), vh)


def test_fork_of_an_unmapped_or_overfull_tail(backend):
    c = Case([40, 40, 48], page=16, W=3, junk=0.5, spare=8)
    c.table[0, 2] = -1; c.n_kv[2] = 500
    kh, vh, _, _ = c.host(); parent = np.array([0, 1, 2, 2], np.int32); fresh = c.spare[:4].copy()
    want_t, want_n = ref.fork(kh, vh, c.table, c.n_kv, parent, fresh)
    k, v, table, n_kv = c.dev()
    wide = torch.full((4, 5), 99, dtype=torch.int32, device=DEV)
    got_t, got_n = backend.paged_fork(k, v, table, n_kv, g(parent), g(fresh), table_out=wide[:, 1:4])
    np.testing.assert_array_equal(host(got_t), want_t); np.testing.assert_array_equal(host(got_n), want_n)
    assert (wide[:, [0, 4]] == 99).all()
    np.testing.assert_array_equal(host(k), kh); np.testing.assert_array_equal(host(v), vh)


def test_store_evict_and_fork_past_32_bit_offsets(backend):
    """the first and the last pages of a pool of more than 4 GiB"""
    page, heads_kv, D, n_pages = 4096, 8, 128, 300
    pool = torch.zeros(n_pages, 2, heads_kv, page, D, dtype=torch.float16, device=DEV)             # 5 GB
    k, v = pool[:, 0], pool[:, 1]
    table = torch.tensor([[299, 0]], dtype=torch.int32, device=DEV); n_kv = torch.tensor([4090], dtype=torch.int32, device=DEV)
    kn, vn = (torch.randn(20, heads_kv, D, device=DEV) for _ in "kv")
    n_kv = backend.paged_store(kn, vn, k, v, table, n_kv, start=torch.tensor([0, 20], dtype=torch.int32, device=DEV))
    assert n_kv.tolist() == [4110]
    for x, new in ((k, kn), (v, vn)):
        assert torch.equal(x[299, :, 4090:], new[:6].half().transpose(0, 1)) and torch.equal(x[0, :, :14], new[6:].half().transpose(0, 1))
        assert not x[299, :, :4090].any() and not x[0, :, 14:].any()
    table2, n2 = backend.paged_fork(k, v, table, n_kv, torch.tensor([0], dtype=torch.int32, device=DEV), torch.tensor([298], dtype=torch.int32, device=DEV))
    assert table2.tolist() == [[299, 298]] and n2.tolist() == [4110] and torch.equal(k[298, :, :14], k[0, :, :14]) and torch.equal(v[298, :, :14], v[0, :, :14]) and not v[298, :, 14:].any()
    weight = torch.zeros(1, heads_kv, 8192, device=DEV); weight[:, :, 4100:4110] = 1
    pos = torch.arange(8192, dtype=torch.int32, device=DEV).expand(1, heads_kv, 8192).contiguous()
    n3 = backend.paged_evict(k, v, table2, n2, weight, pos, n2, 4096)
    moved = torch.arange(4100, 4110, dtype=torch.int32, device=DEV).expand(heads_kv, 10)
    assert n3.tolist() == [4096] and torch.equal(pos[0, :, 4086:4096], moved)
    assert torch.equal(k[299, :, 4086:4096], kn[10:].half().transpose(0, 1)) and torch.equal(v[299, :, 4086:4096], vn[10:].half().transpose(0, 1))


def test_recorded_calls_replay(backend):
    """CallPlan: a store, an attention and a selection recorded once run again on what their tensors then hold"""
    c = Case([33, 5], page=16, W=6, seed=12, junk=0.0)
    k, v, table, n_kv = c.dev()
    kn, vn, q = torch.randn(2, 2, 128, device=DEV), torch.randn(2, 2, 128, device=DEV), torch.randn(2, 8, 128, device=DEV)
    x, score = torch.randn(2, 500, device=DEV), torch.zeros(2, device=DEV)
    out, after = torch.zeros_like(q), torch.zeros_like(n_kv); outs = (torch.zeros(1, 3, device=DEV), torch.zeros(1, 3, dtype=torch.int32, device=DEV), torch.zeros(1, 3, dtype=torch.int32, device=DEV))

    def step():
        backend.paged_store(kn, vn, k, v, table, n_kv, n_kv_out=after)
        backend.paged_attn(q, k, v, table, after, out=out)
        backend.beam_select(x, score, 2, 3, outs=outs)
    with backend.record() as plan:
        step()
    for i in range(3):
        n_kv.copy_(after)
        for y in (kn, vn, q, x):
            y.normal_()
        plan.replay(backend._check)
        got = out.clone(), after.clone(), [o.clone() for o in outs]
        step()
        assert torch.equal(got[0], out) and torch.equal(got[1], after) and all(torch.equal(a, b) for a, b in zip(got[2], outs)) and after.tolist() == [35 + i, 7 + i]


def test_fork_in_a_graph(backend):
    c = Case([40, 17, 64], page=16, W=6, junk=0.5, spare=12, seed=13)
    k, v, table, n_kv = c.dev()
    parent, fresh = g(np.array([0, 0, 1, 2], np.int32)), g(c.spare[:4].copy())
    table_out, n_out = torch.zeros(4, 6, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.paged_fork(k, v, table, n_kv, parent, fresh, table_out=table_out, n_kv_out=n_out)
    for i, (p, f) in enumerate((([0, 0, 1, 2], 0), ([2, 1, 1, -1], 4), ([1, 1, 1, 1], 8))):
        parent.copy_(g(np.array(p, np.int32))); fresh.copy_(g(c.spare[f:f + 4].copy()))
        kh, vh = host(k), host(v)
        graph.replay(); torch.cuda.synchronize()
        want_t, want_n = ref.fork(kh, vh, c.table, c.n_kv, p, c.spare[f:f + 4])
        np.testing.assert_array_equal(host(table_out), want_t); np.testing.assert_array_equal(host(n_out), want_n)
        np.testing.assert_array_equal(host(k), kh); np.testing.assert_array_equal(host(v), vh)


def test_tables_of_no_pages_and_batches_of_nothing(backend):
    """W = 0: nothing can be held; n_seq = 0, no tokens, no rows: nothing happens"""
    c = Case([16, 16], page=16, W=1, junk=0.5, seed=14)
    k, v, _, _ = c.dev(); k0, v0 = k.clone(), v.clone()
    table, n_kv = torch.empty(2, 0, dtype=torch.int32, device=DEV), torch.tensor([5, -1], dtype=torch.int32, device=DEV)
    q, rows = torch.randn(2, 4, 128, device=DEV), torch.randn(2, 2, 128, device=DEV)
    weight, pos = torch.empty(2, 2, 0, device=DEV), torch.empty(2, 2, 0, dtype=torch.int32, device=DEV)
    assert not backend.paged_attn(q, k, v, table, n_kv).any() and not backend.paged_attn(q, k, v, table, n_kv, weight=weight).any()
    assert backend.paged_store(rows, rows, k, v, table, n_kv, n_past=n_kv, weight=weight, pos=pos).tolist() == [0, -1]
    assert backend.paged_evict(k, v, table, n_kv, weight, pos, n_kv, 3).tolist() == [0, -1]
    t2, n2 = backend.paged_fork(k, v, table, n_kv, torch.tensor([0, 1, 5], dtype=torch.int32, device=DEV), torch.tensor([0, 1, 1], dtype=torch.int32, device=DEV))
    assert t2.shape == (3, 0) and n2.tolist() == [0, -1, -1]
    none, empty = torch.empty(0, 1, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV)
    assert backend.paged_attn(q[:0], k, v, none, empty).shape == (0, 4, 128)
    assert backend.paged_store(rows[:0], rows[:0], k, v, none, empty).numel() == 0
    full = g(c.table)
    assert backend.paged_store(rows[:0], rows[:0], k, v, full, n_kv, start=torch.zeros(3, dtype=torch.int32, device=DEV)).tolist() == [5, -1]
    t3, n3 = backend.paged_fork(k, v, full, n_kv, empty, empty)
    assert t3.shape == (0, 1) and n3.numel() == 0
    assert all(x.shape == (0, 2) for x in backend.beam_select(torch.empty(0, 10, device=DEV), torch.empty(0, device=DEV), 3, 2))
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ---- together, as they are used
def test_a_capped_cache_decodes(backend):
    """prompt, then 60 tokens with a cache of 48 slots a head: store, attention with gathered weights, eviction -- every step against the reference on its own copy of the state.  The
    reference follows the device's weights, so that a tie broken by the last bit does not make two histories."""
    heads_kv, heads, D, page, budget = 2, 6, 64, 16, 48
    c = Case([0, 0, 0], D=D, heads_kv=heads_kv, page=page, junk=0.0, W=5)
    k, v, table, n_kv = c.dev()
    weight, pos = torch.zeros(3, heads_kv, c.W * page, device=DEV), torch.zeros(3, heads_kv, c.W * page, dtype=torch.int32, device=DEV)
    past = torch.zeros(3, dtype=torch.int32, device=DEV)
    kh, vh, _, nh = c.host(); wh, ph, past_h = host(weight), host(pos), np.zeros(3, np.int32)
    for step in range(61):
        counts = np.array([50, 7, 1] if step == 0 else [1, 1, 1 if step % 3 else 0])
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        kn, vn = (torch.from_numpy(c.rng.standard_normal((start[-1], heads_kv, D)).astype(np.float32)) for _ in "kv")
        q = torch.from_numpy(c.rng.standard_normal((3, heads, D)).astype(np.float32))
        n_kv = backend.paged_store(kn.to(DEV), vn.to(DEV), k, v, table, n_kv, start=g(start), n_past=past, weight=weight, pos=pos)
        nh = ref.store(kn.half().double().numpy(), vn.half().double().numpy(), kh, vh, c.table, nh, start, past_h, wh, ph)
        past += g(counts.astype(np.int32)); past_h = past_h + counts.astype(np.int32)
        out = backend.paged_attn(q.to(DEV), k, v, table, n_kv, weight=weight)
        want, tol, wtol = ref.attn(q.double().numpy(), kh, vh, c.table, nh, D ** -0.5, weight=wh)
        assert (np.abs(host(out) - want) <= tol).all() and (np.abs(host(weight) - wh) <= wtol).all(), step
        wh = host(weight)
        n_kv = backend.paged_evict(k, v, table, n_kv, weight, pos, past, budget, n_sink=2, n_recent=16)
        w32, ph, nh = ref.evict(kh, vh, c.table, nh, wh.astype(np.float32), ph, past_h, budget, 2, 16)
        wh = w32.astype(np.float64)
        for a, b in ((k, kh), (v, vh), (weight, wh), (pos, ph), (n_kv, nh)):
            np.testing.assert_array_equal(host(a), b)
    assert nh.max() == budget


def test_a_beam_search_over_shared_pages(backend):
    """2 requests x 3 beams for 40 tokens: selection, fork, store, attention.  Every beam's attention equals that over its own unshared history."""
    groups, beams, heads_kv, heads, D, page, V = 2, 3, 2, 4, 64, 16, 1000
    rows, W = groups * beams, 5
    n_pages = 900
    r = np.random.default_rng(0)
    kc, vc = (torch.zeros(n_pages, heads_kv, page, D, dtype=torch.float16, device=DEV) for _ in "kv")
    free = iter(range(n_pages))
    table = np.full((rows, W), -1, np.int32); hist = []
    prompt = [21, 9]
    for gr in range(groups):
        kp, vp = (r.standard_normal((prompt[gr], heads_kv, D)).astype(np.float32) for _ in "kv")
        for b in range(beams):
            row = gr * beams + b
            table[row, :2] = [next(free), next(free)]; hist.append((list(kp), list(vp)))
    n_kv = torch.zeros(rows, dtype=torch.int32, device=DEV); dtable = g(table)
    start = g(np.cumsum([0] + [prompt[i // beams] for i in range(rows)]).astype(np.int32))
    n_kv = backend.paged_store(g(np.concatenate([np.array(h[0]) for h in hist])), g(np.concatenate([np.array(h[1]) for h in hist])), kc, vc, dtable, n_kv, start=start)
    score = g(np.where(np.arange(rows) % beams == 0, 0.0, -np.inf).astype(np.float32)); done = torch.zeros(rows, dtype=torch.int32, device=DEV)
    for step in range(40):
        logits = r.standard_normal((rows, V)).astype(np.float32) * 2
        ws, wp, wt = ref.beam(logits, score.cpu().numpy(), beams, beams, done.cpu().numpy(), pad=2)
        s2, parent, token = backend.beam_select(g(logits), score, beams, beams, done=done, pad=2)
        np.testing.assert_array_equal(host(parent), wp); np.testing.assert_array_equal(host(token), wt)
        np.testing.assert_allclose(host(s2), ws, rtol=1e-6, atol=1e-5)
        score = s2.reshape(-1); flat = parent.reshape(-1); done = ((done[flat.long()] != 0) | (token.reshape(-1) == 2)).int()
        fresh = g(np.array([next(free) for _ in range(rows)], np.int32))
        dtable, n_kv = backend.paged_fork(kc, vc, dtable, n_kv, flat, fresh)
        # a row whose pages are all full gets the page it appends to
        need = (n_kv % page == 0)
        dtable[torch.arange(rows, device=DEV)[need], (n_kv[need] // page).long()] = fresh[need]
        kn, vn = (r.standard_normal((rows, heads_kv, D)).astype(np.float32) for _ in "kv")
        n_kv = backend.paged_store(g(kn), g(vn), kc, vc, dtable, n_kv)
        hist = [(hist[p][0] + [kn[i]], hist[p][1] + [vn[i]]) for i, p in enumerate(flat.tolist())]
        q = r.standard_normal((rows, heads, D)).astype(np.float32)
        out = host(backend.paged_attn(g(q), kc, vc, dtable, n_kv))
        for i in range(rows):
            kk, vv = (torch.from_numpy(np.array(x)).half().double().numpy().transpose(1, 0, 2)[None] for x in hist[i])
            want, tol, _ = ref.attn(q[i:i + 1].astype(np.float64), kk, vv, np.array([[0]]), [kk.shape[2]], D ** -0.5)
            assert (np.abs(out[i] - want[0]) <= tol[0]).all(), (step, i)


def test_a_decode_step_in_one_graph(backend):
    """store + attention + eviction captured once and replayed: the lengths advance on the device"""
    heads_kv, heads, D, page, budget, n = 2, 4, 128, 32, 100, 3
    c = Case([90, 100, 3], D=D, heads_kv=heads_kv, page=page, junk=0.0, W=4)
    state = []
    for _ in range(2):
        state.append(dict(k=c.k.clone(), v=c.v.clone(), n=g(c.n_kv), past=g(c.n_kv), w=torch.zeros(n, heads_kv, 128, device=DEV), p=g(np.tile(np.arange(128, dtype=np.int32), (n, heads_kv, 1)))))
    table = g(c.table); kn, vn = (torch.zeros(n, heads_kv, D, device=DEV) for _ in "kv"); q = torch.zeros(n, heads, D, device=DEV)

    def step(s, out):
        m = backend.paged_store(kn, vn, s["k"], s["v"], table, s["n"], n_past=s["past"], weight=s["w"], pos=s["p"])
        s["past"].add_(1)
        backend.paged_attn(q, s["k"], s["v"], table, m, weight=s["w"], out=out)
        s["n"].copy_(backend.paged_evict(s["k"], s["v"], table, m, s["w"], s["p"], s["past"], budget, n_sink=1, n_recent=8))
    a, b = state
    outs = [torch.zeros(n, heads, D, device=DEV) for _ in state]
    backend.reserve_workspace(max(backend.paged_workspace(q, a["k"], a["v"], table, weight=a["w"]), backend.evict_workspace(a["k"], a["v"], table, a["w"], a["p"], budget, 1, 8)))
    epoch = backend.lib.cdna4_workspace_epoch(backend.ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, outs[1])
    for i in range(25):
        for x in (kn, vn, q):
            x.copy_(torch.from_numpy(c.rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        step(a, outs[0]); graph.replay(); torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]), i
        for key in a:
            assert torch.equal(a[key], b[key]), (i, key)
    assert a["n"].tolist() == [100, 100, 28] and epoch == backend.lib.cdna4_workspace_epoch(backend.ctx)
