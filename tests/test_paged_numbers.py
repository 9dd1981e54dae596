"""Whole numbers of the paged calls beyond 32 bits are refused by the binding and do not come back as small ones (no GPU)."""
import pytest
import torch

from conftest import load_package
from test_paged_refusals import be, cache  # noqa: F401


def test_numbers_beyond_32_bits_are_refused(be):  # noqa: F811
    Error = load_package().Cdna4Error
    k, table, n, slots = cache(9, 2, 16, 64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64)
    logits, score = torch.zeros(6, 100), torch.zeros(6)
    big = 1 << 32
    calls = [lambda x: be.evict_workspace(k, k, table, slots, slots.int(), 8 + x), lambda x: be.evict_workspace(k, k, table, slots, slots.int(), 8, n_sink=1 + x),
             lambda x: be.evict_workspace(k, k, table, slots, slots.int(), 8, n_recent=1 + x), lambda x: be.beam_workspace(logits, 3 + x, 5), lambda x: be.beam_workspace(logits, 3, 5 + x),
             lambda x: be.beam_workspace(logits, 3, 5, pad=1 + x)]
    for call in calls:
        assert call(0) > 0
        for x in (big, -big, 1 << 70):
            with pytest.raises(Error):
                call(x)
    for x in (big, -big):
        for call in (lambda: be.paged_evict(k, k, table, n, slots, slots.int(), n, 8 + x), lambda: be.paged_evict(k, k, table, n, slots, slots.int(), n, 8, n_sink=x),
                     lambda: be.paged_evict(k, k, table, n, slots, slots.int(), n, 8, n_recent=x), lambda: be.beam_select(logits, score, 3, 5 + x), lambda: be.beam_select(logits, score, 3 + x, 5),
                     lambda: be.beam_select(logits, score, 3, 5, pad=x)):
            with pytest.raises(Error, match="32 bits"):
                call()
    with pytest.raises(TypeError):
        be.beam_workspace(logits, 3.0, 5)
