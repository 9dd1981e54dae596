"""-m gpu: the selection of a beam search against tests/paged_ref.py in 64 bits: parents and tokens are equal, scores to the rounding of the result and of the sum of exponentials."""
import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu


def check(be, logits, score, n_beam, n_out, done=None, pad=0, rows=None):
    x = torch.from_numpy(logits).cuda() if rows is None else rows
    s = torch.from_numpy(score).cuda()
    got = be.beam_select(x, s, n_beam, n_out, done=None if done is None else torch.from_numpy(done).cuda(), pad=pad)
    ws, wp, wt = ref.beam(logits, score, n_beam, n_out, done, pad)
    np.testing.assert_array_equal(got[1].cpu().numpy(), wp); np.testing.assert_array_equal(got[2].cpu().numpy(), wt)
    # a score is rounded to f32 once (2^-24 of it); the sum of exponentials (each to 2^-22, an argument's rounding included for arguments down to -16: what is smaller adds nothing) is made
    # of partial sums of less than 2^8 terms in f32, 2^8 * 2^-24 relative, and its logarithm is off by as much: 2^-16 + 2^-22 < 2^-15
    np.testing.assert_allclose(got[0].cpu().numpy(), ws, rtol=2.0 ** -23, atol=2.0 ** -15)
    return got


@pytest.mark.parametrize("n_vocab", [1, 2, 63, 64, 65, 257, 1000, 4096, 8191, 8193, 32000, 151936])
@pytest.mark.parametrize("n_group,n_beam,n_out", [(1, 1, 1), (2, 4, 4), (3, 5, 10), (1, 8, 64), (2, 2, 33)])
def test_sizes(n_group, n_beam, n_out, n_vocab, backend):
    r = np.random.default_rng(n_vocab + n_out)
    n_out = min(n_out, n_beam * n_vocab)
    check(backend, (r.standard_normal((n_group * n_beam, n_vocab)) * 3).astype(np.float32), (-10 * r.random(n_group * n_beam)).astype(np.float32), n_beam, n_out)


@pytest.mark.parametrize("n_out", [1, 7, 64])
@pytest.mark.parametrize("n_vocab", [300, 40001])
def test_ties_go_to_the_lower_index(n_vocab, n_out, backend):
    r = np.random.default_rng(n_out)
    same = np.zeros(4, np.float32)
    check(backend, np.zeros((4, n_vocab), np.float32), same, 2, n_out)                                               # everything is equal
    check(backend, r.integers(0, 2, (4, n_vocab)).astype(np.float32)[[0, 0, 1, 1]], same, 2, n_out)                  # two values, two equal beams
    falling = -np.arange(n_vocab, dtype=np.float32)[None].repeat(4, 0) * 0.001                                       # the best ones lie side by side, at either end
    check(backend, falling, same, 4, n_out)
    check(backend, np.ascontiguousarray(falling[:, ::-1]), same, 4, n_out)
    x = np.full((2, n_vocab), -5.0, np.float32); x[0, ::256] = 1.0; x[1, 17::256] = 1.0                               # the best ones all in one thread's share
    check(backend, x, np.array([0.0, -0.5], np.float32), 2, n_out)


def test_masked_tokens_finished_beams_and_rows_of_nothing(backend):
    r = np.random.default_rng(1)
    x = r.standard_normal((12, 5000)).astype(np.float32)
    x[0] = -np.inf; x[1, 1:] = -np.inf; x[2, 100:] = -np.inf; x[3, 7] = np.nan; x[4, 9] = np.inf; x[5] = np.nan; x[6, ::2] = -np.finfo(np.float32).max; x[11, 1000:2000] = np.float32(1e-38) * np.arange(1000, dtype=np.float32); x[7] = np.finfo(np.float32).max
    score = (-3 * r.random(12)).astype(np.float32); score[8] = -np.inf; score[9] = np.nan
    done = (r.random(12) < 0.3).astype(np.int32); done[5] = 1; done[10] = -1
    for n_beam in (1, 3, 4, 12):
        for n_out in (1, 5, 40):
            check(backend, x, score, n_beam, n_out)
            check(backend, x, score, n_beam, n_out, done, pad=4999)
            check(backend, x, score, n_beam, n_out, np.ones(12, np.int32), pad=0)


def test_a_stretch_of_nan_makes_a_row_of_nothing(backend):
    r = np.random.default_rng(7)
    for n_vocab, rows in ((20000, 4), (20000, 300)):
        x = r.standard_normal((rows, n_vocab)).astype(np.float32)
        x[1, 8192:16384] = np.nan; x[2, 16384:] = -np.inf; x[3, 16384:] = -np.inf; x[3, 19999] = np.nan
        check(backend, x, np.zeros(rows, np.float32), 4, 6)
        check(backend, x, np.zeros(rows, np.float32), 1, 6)


def test_strides_and_many_beams(backend):
    r = np.random.default_rng(2)
    x = r.standard_normal((256, 1003)).astype(np.float32); score = -r.random(256).astype(np.float32)
    wide = torch.full((256, 1010), 50.0, device="cuda"); wide[:, 3:1006] = torch.from_numpy(x).cuda()                # rows that begin at odd addresses, larger values around them
    for n_beam, n_out in ((256, 64), (128, 3), (1, 2)):
        check(backend, x, score, n_beam, n_out, rows=wide[:, 3:1006])


def test_repeats_bit_for_bit_and_in_a_graph(backend):
    r = np.random.default_rng(3)
    x = torch.from_numpy(r.standard_normal((24, 32003)).astype(np.float32)).cuda(); score = torch.zeros(24, device="cuda")
    base = backend.beam_select(x, score, 6, 12)
    backend.reserve_workspace(backend.beam_workspace(x, 6, 12))
    outs = tuple(torch.zeros_like(t) for t in base)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.beam_select(x, score, 6, 12, outs=outs)
    for i in range(4):
        if i:
            x.copy_(torch.from_numpy(r.standard_normal((24, 32003)).astype(np.float32)))
        graph.replay(); torch.cuda.synchronize()
        eager = backend.beam_select(x, score, 6, 12)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        if not i:
            assert all(torch.equal(a, b) for a, b in zip(outs, base))


@pytest.mark.parametrize("n_group,n_beam,n_out,n_vocab", [(1, 256, 64, 20000), (1, 256, 50, 10000), (1, 200, 44, 14000), (2, 150, 45, 9000), (700, 1, 3, 4000), (3, 7, 23, 2049), (5, 3, 61, 2300), (300, 2, 17, 8193)])
def test_many_lists_and_cut_chunks(n_group, n_beam, n_out, n_vocab, backend):
    """more chunks of a group than the join has lanes, chunks with a few logits in them, waves without a finite one"""
    r = np.random.default_rng(n_vocab)
    x = (r.standard_normal((n_group * n_beam, n_vocab)) * 2).astype(np.float32); score = (-3 * r.random(n_group * n_beam)).astype(np.float32)
    check(backend, x, score, n_beam, n_out)
    x[:, n_vocab // 3:] = -np.inf; x[:, 5:300] = -np.inf; x[::2, :n_vocab // 3] = -np.inf; x[::2, -3:] = 1.0
    check(backend, x, score, n_beam, n_out)
    x[:] = np.round(r.standard_normal(x.shape)).astype(np.float32)                                                    # a few values, each many times
    check(backend, x, np.zeros_like(score), n_beam, n_out)
