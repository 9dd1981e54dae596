"""The paged decode step of the documentation for hosts, run on a backend that notes its calls: what the eviction holds as recent counts the token that the step stored (no GPU)."""
import glob
import os
import re

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Notes:
    calls = []

    def __init__(self, device):
        Notes.calls = []

    def paged_store(self, k, v, k_cache, v_cache, table, n_kv, start=None, n_past=None, weight=None, pos=None, n_kv_out=None):
        Notes.calls.append(("store", n_past.clone())); return n_kv + 1

    def paged_attn(self, q, k_cache, v_cache, table, n_kv, scale=None, softcap=0.0, weight=None, out=None):
        Notes.calls.append(("attn", n_kv.clone())); return q

    def paged_evict(self, k_cache, v_cache, table, n_kv, weight, pos, n_past, budget, n_sink=0, n_recent=0, weight_out=None, pos_out=None, n_kv_out=None):
        Notes.calls.append(("evict", n_past.clone())); return n_kv.clamp(max=budget)


class Torch:
    float16 = torch.float16

    @staticmethod
    def zeros(*size, dtype, device):
        return torch.zeros(*size, dtype=dtype)


def test_the_paged_decode_step():
    heading = "### Many sequences in one pool of pages"
    (text,) = [t for t in (open(p).read() for p in glob.glob(os.path.join(ROOT, "*.md"))) if heading in t]
    section = text[text.index(heading):]
    code = re.search(r"```python\n(.*?)```", section, re.S).group(1)
    past = torch.tensor([7, 100], dtype=torch.int32)
    names = dict(Cdna4Backend=Notes, torch=Torch, n_pages=3, n_head_kv=2, k=None, v=None, q=None, past=past, weight=None, pos=None, n_kv=torch.tensor([7, 90], dtype=torch.int32))
    for step in range(2):
        exec(code, names)
        (_, stored), (_, _), (_, held) = Notes.calls
        assert torch.equal(stored, torch.tensor([7, 100], dtype=torch.int32) + step) and torch.equal(held, stored + 1)
    assert names["past"].tolist() == [9, 102]
