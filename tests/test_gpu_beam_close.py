"""-m gpu: candidates of different beams that differ by less than 32 bits can tell come out in the order of their values in 64 bits."""
import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_vocab,n_beam,n_group", [(1000, 4, 100), (9001, 3, 60), (40000, 2, 40), (128256, 4, 70)])
def test_close_candidates_of_different_beams(n_vocab, n_beam, n_group, backend):
    """every group's beams have their best candidates at one value, up to the rounding of the scores: differences of up to 2^-22, and the sums of exponentials of the beams differ"""
    r = np.random.default_rng(n_vocab)
    x = (r.standard_normal((n_group * n_beam, n_vocab)) * r.uniform(0.5, 4, (n_group * n_beam, 1))).astype(np.float32)
    l = x.astype(np.float64); top = l.max(1)
    best = -np.log(np.exp(l - top[:, None]).sum(1))
    score = (-14.0 - best).astype(np.float32)
    c = np.sort((score.astype(np.float64) + best).reshape(n_group, n_beam), 1)
    assert np.diff(c, axis=1).max() < 2.0 ** -19 and np.diff(c, axis=1).min() > 1e-11          # (no pair so close that 64 bits could tell it differently)
    s, parent, token = backend.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), n_beam, n_beam)
    ws, wp, wt = ref.beam(x, score, n_beam, n_beam)
    np.testing.assert_array_equal(parent.cpu().numpy(), wp); np.testing.assert_array_equal(token.cpu().numpy(), wt)
    np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -24, atol=1e-10)          # one rounding to 32 bits
