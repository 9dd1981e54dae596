"""Measured cases of the operators that decode over a paged key / value cache: storing new tokens, the attention of one new token per sequence (with the weight that every
cached token has gathered so far), eviction by that weight, the selection of a beam search, and the fork of sequences along the chosen beams.

`run` computes an operator in elementary torch operations, or, where `own` is set, through the library's entry points.  `exact` states the same definitions in 64 bits."""
import functools
import importlib.util
import math
import os
import random
import sys

import torch

own = False
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -------------------------------------------------------------------------------------------------------------------------------------------------------------
def _store(n_seq, most, heads_kv, dim, page, dtype, layout, name=None):
    return _named(name, op="store", n_seq=n_seq, most=most, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout)


def _attn(n_seq, most, heads, heads_kv, dim, page, dtype, layout, weights, softcap, name=None):
    return _named(name, op="attn", n_seq=n_seq, most=most, heads=heads, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout, weights=weights, softcap=softcap)


def _evict(n_seq, most, budget, sink, recent, heads_kv, dim, page, dtype, layout, name=None):
    return _named(name, op="evict", n_seq=n_seq, most=most, budget=budget, sink=sink, recent=recent, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout)


def _beam(groups, beams, vocab, n_out, done, name=None):
    return _named(name, op="beam", groups=groups, beams=beams, vocab=vocab, n_out=n_out, done=done)


def _fork(n_seq, most, heads_kv, dim, page, dtype, layout, name=None):
    return _named(name, op="fork", n_seq=n_seq, most=most, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout)


def _named(name, **case):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one new token of each of 64 chats is written to one layer's cache: every decode step does it once a layer
        _store(64, 1, 8, 128, 64, "f16", "head", name="store, one token of 64 chats"),
        # ragged prompts of up to 4096 tokens are written to one layer's cache in one call
        _store(6, 4096, 8, 128, 16, "bf16", "token", name="store, six ragged prompts"),
        # a single chat, a few hundred tokens in: latency is all that counts
        _attn(1, 301, 32, 8, 128, 16, "f16", "head", False, 0.0, name="attn, one short chat"),
        # a server's batch of chats of very different lengths
        _attn(64, 8192, 32, 8, 128, 64, "f16", "head", False, 0.0, name="attn, 64 ragged chats"),
        # one long document with 8 query heads on each key head
        _attn(1, 131071, 64, 8, 128, 256, "bf16", "head", False, 0.0, name="attn, one long document"),
        # small heads, two to a key head, capped scores, token-major pages, and the gathered weights kept for the eviction below
        _attn(16, 4099, 16, 8, 64, 32, "f16", "token", True, 30.0, name="attn, 16 chats with weights"),
        # the steady state of a capped cache: some tokens over the budget go
        _evict(16, 4160, 4096, 4, 512, 8, 128, 64, "f16", "head", name="evict, 16 chats to 4096"),
        # prompts shrink to an eighth
        _evict(4, 32768, 4096, 16, 1024, 8, 128, 256, "bf16", "head", name="evict, long prompts to 4096"),
        # one request, four beams
        _beam(1, 4, 32000, 4, False, name="beam, one request of 4"),
        # a batch of requests, some beams finished
        _beam(32, 8, 128256, 16, True, name="beam, 32 requests of 8"),
        # one request's four beams go on from their parents
        _fork(4, 517, 8, 128, 64, "f16", "head", name="fork, 4 beams"),
        # a batch of 256 beams over long contexts
        _fork(256, 8192, 8, 128, 256, "bf16", "token", name="fork, 256 beams"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))


def draw(rng):
    op = rng.choice(["store", "attn", "attn", "evict", "beam", "fork"])
    dim, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
    dtype, layout, heads_kv = rng.choice(["f16", "bf16"]), rng.choice(["head", "token"]), rng.choice([1, 2, 4, 8])
    if op == "store":
        n_seq = _log(rng, 1, 200)
        return _store(n_seq, _log(rng, 1, max(1, 16000 // n_seq)), heads_kv, dim, page, dtype, layout)
    if op == "attn":
        n_seq = _log(rng, 1, 100)
        most = _log(rng, 1, min(130000, 130000 * 8 * 128 // (n_seq * heads_kv * dim)))
        heads = heads_kv * rng.choice([1, 2, 3, 4, 6, 8, 16, 20])
        return _attn(n_seq, most, heads, heads_kv, dim, page, dtype, layout, rng.random() < 0.4 and heads * n_seq * most < 1 << 27, rng.choice([0.0, 0.0, 30.0]))
    if op == "evict":
        n_seq = _log(rng, 1, 32)
        most = _log(rng, 20, min(32000, 130000 // n_seq))
        budget = _log(rng, 1, most)
        sink = rng.randint(0, min(budget, 8))
        return _evict(n_seq, most, budget, sink, rng.randint(0, (budget - sink) // 2), heads_kv, dim, page, dtype, layout)
    if op == "beam":
        groups, beams = _log(rng, 1, 40), rng.randint(1, 12)
        vocab = _log(rng, 500, min(152000, 32 * 8 * 128256 // (groups * beams)))
        return _beam(groups, beams, vocab, rng.randint(1, min(64, 2 * beams + 2)), rng.random() < 0.5)
    n_seq = _log(rng, 1, 200)
    return _fork(n_seq, _log(rng, 1, min(32000, 400000 // n_seq)), heads_kv, dim, page, dtype, layout)


def _lengths(c):
    """The tokens that each sequence holds (store: that it brings): spread over the whole range and the same for every seed, the longest among them."""
    rng = random.Random("%(op)s %(n_seq)d %(most)d" % c)
    if c["op"] == "evict":
        return [c["most"] if i == 0 else rng.randint(c["budget"], c["most"]) for i in range(c["n_seq"])]
    low = 0 if c["op"] == "attn" else 1
    return [c["most"] if i == 0 else rng.randint(low, c["most"]) for i in range(c["n_seq"])]


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    if c["op"] == "beam":
        rows = c["groups"] * c["beams"]
        s["logits"] = 2.5 * torch.randn(rows, c["vocab"], generator=g, device=DEV)
        s["score"] = -5.0 * torch.rand(rows, generator=g, device=DEV)
        s["done"] = (torch.rand(rows, generator=g, device=DEV) < 0.2).int() if c["done"] else None
        return s
    n_seq, page, heads_kv, dim, dtype = c["n_seq"], c["page"], c["heads_kv"], c["dim"], TYPES[c["dtype"]]
    lens = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
    before = torch.randint(0, 300, (n_seq,), generator=g, device=DEV).int() if c["op"] == "store" else 0 * lens
    width = -(-(c["most"] + (300 if c["op"] == "store" else 0)) // page)
    n_pages = n_seq * width + n_seq + 3
    perm = torch.randperm(n_pages, generator=g, device=DEV).int()
    s["table"] = perm[:n_seq * width].view(n_seq, width)
    for name in ("k_cache", "v_cache"):
        if c["layout"] == "head":
            s[name] = torch.randn(n_pages, heads_kv, page, dim, generator=g, device=DEV, dtype=dtype)
        else:      # the heads of a token side by side, seen as [pages, heads, slots, dim]
            s[name] = torch.randn(n_pages, page, heads_kv, dim, generator=g, device=DEV, dtype=dtype).transpose(1, 2)
    if c["op"] == "store":
        tokens = sum(_lengths(c))
        s["n_kv"], s["start"] = before, torch.cat([0 * lens[:1], lens.cumsum(0).int()])
        s["k"], s["v"] = (torch.randn(tokens, heads_kv, dim, generator=g, device=DEV) for _ in "kv")
        s["n_past"] = before + torch.randint(0, 50, (n_seq,), generator=g, device=DEV).int()
        s["weight"] = torch.rand(n_seq, heads_kv, width * page, generator=g, device=DEV)
        s["pos"] = torch.randint(0, 1 << 20, (n_seq, heads_kv, width * page), generator=g, device=DEV).int()
        return s
    s["n_kv"] = lens
    if c["op"] == "attn":
        s["q"] = torch.randn(n_seq, c["heads"], dim, generator=g, device=DEV) * 1.5
        s["scale"] = dim ** -0.5
        s["weight"] = torch.rand(n_seq, heads_kv, width * page, generator=g, device=DEV) if c["weights"] else None
    elif c["op"] == "evict":      # heavy-tailed weights of a long context, positions in disorder as earlier evictions leave them
        s["weight"] = torch.exp(3.0 * torch.randn(n_seq, heads_kv, width * page, generator=g, device=DEV) - 4.0)
        s["n_past"] = lens + torch.randint(0, 500, (n_seq,), generator=g, device=DEV).int()
        order = torch.rand(n_seq, heads_kv, width * page, generator=g, device=DEV)
        order = torch.where(torch.arange(width * page, device=DEV) < lens[:, None, None], order, 2.0)
        s["pos"] = order.argsort(-1).argsort(-1).int() + (s["n_past"] - lens)[:, None, None] * (order > 0.02)
        s["weight_out"], s["pos_out"] = torch.zeros_like(s["weight"]), torch.zeros_like(s["pos"])
    elif c["op"] == "fork":
        beams = 4
        first = torch.arange(n_seq, device=DEV) // beams * beams
        s["parent"] = (first + torch.randint(0, beams, (n_seq,), generator=g, device=DEV)).clamp(max=n_seq - 1).int()
        s["fresh"] = perm[n_seq * width:n_seq * width + n_seq].contiguous()
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return {"store": _own_store, "attn": _own_attn, "evict": _own_evict, "beam": _own_beam, "fork": _own_fork}[c["op"]](s, c, _backend())
    return {"store": _plain_store, "attn": _plain_attn, "evict": _plain_evict, "beam": _plain_beam, "fork": _plain_fork}[c["op"]](s, c)


@functools.lru_cache(None)
def _backend():
    name = "ik_llama_cpp_amd"
    if name not in sys.modules:
        folder = os.path.join(ROOT, "ik_llama.cpp_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name].Cdna4Backend(torch.cuda.current_device())


def _own_store(s, c, be):
    n_kv = be.paged_store(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["n_kv"], start=s["start"], n_past=s["n_past"], weight=s["weight"], pos=s["pos"])
    return s["k_cache"], s["v_cache"], s["weight"], s["pos"], n_kv


def _own_attn(s, c, be):
    out = be.paged_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["n_kv"], scale=s["scale"], softcap=c["softcap"], weight=s["weight"])
    return (out, s["weight"]) if c["weights"] else out


def _own_evict(s, c, be):
    n_kv = be.paged_evict(s["k_cache"], s["v_cache"], s["table"], s["n_kv"], s["weight"], s["pos"], s["n_past"], c["budget"], n_sink=c["sink"], n_recent=c["recent"],
                          weight_out=s["weight_out"], pos_out=s["pos_out"])
    return s["k_cache"], s["v_cache"], s["weight_out"], s["pos_out"], n_kv


def _own_beam(s, c, be):
    return be.beam_select(s["logits"], s["score"], c["beams"], c["n_out"], done=s["done"], pad=2)


def _own_fork(s, c, be):
    table, n_kv = be.paged_fork(s["k_cache"], s["v_cache"], s["table"], s["n_kv"], s["parent"], s["fresh"])
    return s["k_cache"], s["v_cache"], table, n_kv


def _plain_store(s, c):
    page, start, n_kv = c["page"], s["start"].long(), s["n_kv"].long()
    token = torch.arange(s["k"].shape[0], device=DEV)
    seq = torch.searchsorted(start, token, right=True) - 1
    nth = token - start[seq]
    slot = n_kv[seq] + nth
    where = s["table"][seq, slot // page].long()
    s["k_cache"][where, :, slot % page] = s["k"].to(s["k_cache"].dtype)
    s["v_cache"][where, :, slot % page] = s["v"].to(s["v_cache"].dtype)
    s["weight"][seq, :, slot] = 0.0
    s["pos"][seq, :, slot] = (s["n_past"][seq] + nth).int()[:, None]
    return s["k_cache"], s["v_cache"], s["weight"], s["pos"], (n_kv + start[1:] - start[:-1]).int()


def _rows(cache, table, page):
    """[sequences, heads, slots, dim] of a paged cache in 32 bits."""
    n_seq, width = table.shape
    x = cache[table.reshape(-1).long()].float()                                  # [n_seq * width, heads, page, dim]
    return x.view(n_seq, width, x.shape[1], page, x.shape[3]).transpose(1, 2).reshape(n_seq, x.shape[1], width * page, x.shape[3])


def _plain_attn(s, c):
    n_seq, heads, dim = s["q"].shape
    heads_kv, page = c["heads_kv"], c["page"]
    k = _rows(s["k_cache"], s["table"], page)
    q = s["q"].view(n_seq, heads_kv, heads // heads_kv, dim)
    scores = torch.matmul(k, q.transpose(2, 3).contiguous()) * s["scale"]         # [n_seq, heads_kv, slots, group]
    del k
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    valid = torch.arange(scores.shape[2], device=DEV) < s["n_kv"][:, None]
    scores = torch.where(valid[:, None, :, None], scores, -math.inf)
    top = scores.amax(2, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(2, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = _rows(s["v_cache"], s["table"], page)
    out = torch.matmul(p.transpose(2, 3).contiguous(), v).reshape(n_seq, heads, dim)
    if c["weights"]:
        s["weight"] += p.sum(3)
        return out, s["weight"]
    return out


def _plain_evict(s, c):
    page, budget, pos, weight = c["page"], c["budget"], s["pos"], s["weight"]
    slots = torch.arange(weight.shape[2], device=DEV)
    n_kv = s["n_kv"].long()[:, None, None]
    n_past = s["n_past"][:, None, None]
    held = (pos < c["sink"]) | (pos >= n_past - c["recent"])
    bits = (torch.where(weight.isnan(), -math.inf, weight) + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits)                       # ordered like the floats
    key = torch.where(held, 1 << 40, key)
    key = torch.where(slots < n_kv, key, -(1 << 40))
    order = key.sort(dim=-1, descending=True, stable=True).indices                  # ties: the lowest slot first
    rank = torch.empty_like(order).scatter_(2, order, slots.expand_as(order))
    over = n_kv > budget
    keep = torch.where(over, rank < budget, slots < n_kv)
    hole, mover = ~keep & (slots < budget) & over, keep & (slots >= budget) & over
    nth = torch.where(mover, mover.cumsum(2) - 1, weight.shape[2])
    movers = torch.zeros(*weight.shape[:2], weight.shape[2] + 1, dtype=torch.long, device=DEV).scatter_(2, nth, slots.expand_as(order))
    source = torch.where(hole, movers.gather(2, (hole.cumsum(2) - 1).clamp(min=0)), slots)[:, :, :budget]
    stays = (slots < n_kv)[:, :, :budget].expand_as(source)
    for out, x in ((s["weight_out"], weight), (s["pos_out"], pos)):
        out[:, :, :source.shape[2]] = torch.where(stays, x.gather(2, source), out[:, :, :source.shape[2]])
    seq, head, to = hole[:, :, :budget].nonzero(as_tuple=True)                    # the rows that move
    of = source[seq, head, to]
    here, there = s["table"][seq, of // page].long(), s["table"][seq, to // page].long()
    for cache in (s["k_cache"], s["v_cache"]):
        cache[there, head, to % page] = cache[here, head, of % page]
    return s["k_cache"], s["v_cache"], s["weight_out"], s["pos_out"], s["n_kv"].clamp(max=budget)


def _plain_beam(s, c):
    x = s["logits"].double()                                                      # neighbours in the order may differ by less than 32 bits tell
    x = x - x.amax(1, keepdim=True)
    lp = s["score"].double()[:, None] + x - x.exp().sum(1, keepdim=True).log()
    if s["done"] is not None:
        pad = torch.arange(c["vocab"], device=DEV) == 2
        kept = torch.where(pad, s["score"].double()[:, None], -math.inf)
        lp = torch.where(s["done"][:, None] != 0, kept, lp)
    flat = lp.view(c["groups"], c["beams"] * c["vocab"])
    score, at = flat.sort(dim=1, descending=True, stable=True)
    at, first = at[:, :c["n_out"]], torch.arange(c["groups"], device=DEV)[:, None] * c["beams"]
    return score[:, :c["n_out"]].float(), (first + at // c["vocab"]).int(), (at % c["vocab"]).int()


def _plain_fork(s, c):
    page, width, parent = c["page"], s["table"].shape[1], s["parent"].long()
    n_kv, pages = s["n_kv"][parent], s["table"][parent]
    full = (n_kv // page)[:, None]
    at = torch.arange(width, device=DEV)
    cut = (n_kv % page != 0)[:, None]
    table = torch.where(at < full, pages, torch.where((at == full) & cut, s["fresh"][:, None], -1)).int()
    tail = pages.gather(1, full.clamp(max=width - 1).long())[:, 0].long()
    copied = torch.arange(page, device=DEV) < (n_kv % page)[:, None]              # [rows, page]
    fresh = s["fresh"].long()
    for cache in (s["k_cache"], s["v_cache"]):
        cache[fresh] = torch.where(copied[:, None, :, None], cache[tail], cache[fresh])
    return s["k_cache"], s["v_cache"], table, n_kv


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------------------------------------------
def work(c):
    if c["op"] == "beam":
        rows = c["groups"] * c["beams"]
        n = rows * c["vocab"]
        return {"bytes": 4 * n + rows * 8 + c["groups"] * c["n_out"] * 12, "flops": 4 * n}
    lens, row = _lengths(c), c["heads_kv"] * c["dim"]
    total = sum(lens)
    entries = sum(-(-n // c["page"]) for n in lens) * 4
    if c["op"] == "store":
        return {"bytes": total * (2 * row * (4 + 2) + c["heads_kv"] * 8) + entries, "flops": 0}
    if c["op"] == "attn":
        weights = 2 * 4 * total * c["heads_kv"] if c["weights"] else 0
        return {"bytes": total * row * 4 + 2 * 4 * c["n_seq"] * c["heads"] * c["dim"] + weights + entries, "flops": 4 * total * c["heads"] * c["dim"]}
    if c["op"] == "evict":      # the expected share of the kept rows that lie behind the budget moves
        moved = sum(min(c["budget"], n) * (1 - min(1.0, c["budget"] / n)) for n in lens)
        return {"bytes": c["heads_kv"] * (8 * total + 8 * sum(min(c["budget"], n) for n in lens)) + moved * row * 2 * 2 * 2 + entries, "flops": total * c["heads_kv"]}
    tails = sum(n % c["page"] for n in lens)
    return {"bytes": 2 * entries + tails * row * 2 * 2 * 2, "flops": 0}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "beam":
        scores = []
        for g in range(c["groups"]):
            found = []
            for b in range(c["beams"]):
                r = g * c["beams"] + b
                base = float(s["score"][r])
                if s["done"] is not None and int(s["done"][r]):
                    found.append(torch.tensor([base], dtype=torch.float64, device=DEV))
                    continue
                row = s["logits"][r].to(torch.float64)
                found.append(torch.topk(row - torch.logsumexp(row, 0) + base, min(c["n_out"], c["vocab"])).values)
            best = torch.cat(found).sort(descending=True).values[:c["n_out"]]
            scores.append(torch.nn.functional.pad(best, (0, c["n_out"] - best.numel()), value=-math.inf))
        return torch.stack(scores), None, None
    if c["op"] == "attn":
        n_seq, heads, dim = s["q"].shape
        group = heads // c["heads_kv"]
        out = torch.zeros(n_seq, heads, dim, dtype=torch.float64, device=DEV)
        weight = s["weight"].double() if c["weights"] else None
        for i, n in enumerate(_lengths(c)):
            pages = s["table"][i, :-(-n // c["page"])].long()
            for h in range(c["heads_kv"] if n else 0):
                k, v = (s[x][pages, h].reshape(-1, dim)[:n].double() for x in ("k_cache", "v_cache"))
                for j in range(h * group, (h + 1) * group):
                    z = (k * s["q"][i, j].double()).sum(1) * s["scale"]
                    z = c["softcap"] * torch.tanh(z / c["softcap"]) if c["softcap"] else z
                    p = torch.softmax(z, 0)
                    out[i, j] = (v * p[:, None]).sum(0)
                    if c["weights"]:
                        weight[i, h, :n] += p
        return (out, weight) if c["weights"] else out
    if c["op"] == "store":      # the values before their rounding to the cache's type; the other operators move values and decide by them, they compute none
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        weight, first = s["weight"].double(), 0
        for i, n in enumerate(_lengths(c)):
            slots = torch.arange(int(s["n_kv"][i]), int(s["n_kv"][i]) + n, device=DEV)
            for cache, new in zip(caches, (s["k"], s["v"])):
                for h in range(c["heads_kv"]):
                    cache[s["table"][i].long()[slots // c["page"]], h, slots % c["page"]] = new[first:first + n, h].double()
            weight[i, :, slots] = 0
            first += n
        return caches[0], caches[1], weight, None, None
    return None
