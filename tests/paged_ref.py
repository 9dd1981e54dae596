"""The paged-cache operators in 64 bits on the host, one loop at a time, straight from their definitions (include/ggml_hip_cdna4.h).  Caches are float64 arrays [pages, heads, slots, D]."""
import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # largest relative rounding error of the cache types
EPS = 2.0 ** -24                                                       # ... and of f32


def page_of(table, n_pages, s, j, page):
    i = int(table[s, j // page])
    return i if 0 <= i < n_pages else -1


def length(table, n_kv, s, page):
    return min(max(int(n_kv[s]), 0), table.shape[1] * page)


def store(k, v, kc, vc, table, n_kv, start=None, n_past=None, weight=None, pos=None):
    """in place; returns the new lengths"""
    n_pages, _, page, _ = kc.shape
    out = np.empty(len(n_kv), np.int32)
    for s in range(len(n_kv)):
        a, b = (s, s + 1) if start is None else (int(start[s]), int(start[s + 1]))
        n = int(n_kv[s]); out[s] = n if n < 0 else min(n + max(b - a, 0), table.shape[1] * page)
        for i in range(a, min(b, len(k)) if n >= 0 else a):
            slot = n + i - a
            if slot >= table.shape[1] * page:
                break
            p = page_of(table, n_pages, s, slot, page)
            if p < 0:
                continue
            kc[p, :, slot % page] = k[i]; vc[p, :, slot % page] = v[i]
            if weight is not None:
                weight[s, :, slot] = 0
            if pos is not None:
                pos[s, :, slot] = n_past[s] + i - a
    return out


def gather(cache, table, n_kv, s, h):
    """(slots, rows) of the mapped slots of sequence s"""
    n_pages, _, page, _ = cache.shape
    at = [j for j in range(length(table, n_kv, s, page)) if page_of(table, n_pages, s, j, page) >= 0]
    return at, np.array([cache[int(table[s, j // page]), h, j % page] for j in at]).reshape(len(at), cache.shape[3])


def attn(q, kc, vc, table, n_kv, scale, softcap=0.0, weight=None):
    """-> out, its error bound, the bound of weight's (weight is updated in place).

    The bound: a score is a sum of D products in f32 of a query that is exact to 2^-22 (D + 8 half steps of f32 and the split), tanh and exp2 to 2^-21; a probability is off by twice
    the largest score error (numerator and denominator), a sum over n terms by n half steps."""
    n_seq, heads, D = q.shape
    group = heads // kc.shape[1]
    out = np.zeros((n_seq, heads, D)); tol = np.full((n_seq, heads, D), 1e-30); wtol = None if weight is None else np.zeros(weight.shape)
    for s in range(n_seq):
        for h in range(kc.shape[1]):
            at, k = gather(kc, table, n_kv, s, h); _, v = gather(vc, table, n_kv, s, h)
            if not at:
                continue
            for g in range(group):
                x = q[s, h * group + g]
                z = (k @ x) * scale
                dz = ((np.abs(k) @ np.abs(x)) * abs(scale) * ((D + 8) * EPS + 2.0 ** -21)).max()
                if softcap:
                    z = softcap * np.tanh(z / softcap); dz += abs(softcap) * 2.0 ** -21
                dz += np.abs(z).max() * 4 * EPS
                p = np.exp(z - z.max()); p /= p.sum()
                rel = 2 * dz + (len(at) + 64) * EPS + 2.0 ** -19
                out[s, h * group + g] = p @ v
                tol[s, h * group + g] += (p @ np.abs(v)) * rel
                if weight is not None:
                    weight[s, h, at] += p; wtol[s, h, at] += p * rel + 2 * EPS * np.abs(weight[s, h, at])
    return out, tol, wtol


def evict(kc, vc, table, n_kv, weight, pos, n_past, budget, sink=0, recent=0):
    """caches in place; -> weight, pos, lengths (copies; values behind the new lengths are the old ones)"""
    n_pages, heads, page, _ = kc.shape
    weight, pos = weight.copy(), pos.copy(); w0, p0 = weight.copy(), pos.copy()
    out = np.empty(len(n_kv), np.int32)
    for s in range(len(n_kv)):
        n = length(table, n_kv, s, page); out[s] = n_kv[s] if n_kv[s] < 0 else min(n, budget)
        if n <= budget:
            continue
        for h in range(heads):
            held = (p0[s, h, :n] < sink) | (p0[s, h, :n].astype(np.int64) >= int(n_past[s]) - recent)
            w = np.where(np.isnan(w0[s, h, :n]), -np.inf, w0[s, h, :n])
            kept = sorted(sorted(range(n), key=lambda j: (not held[j], 0.0 if held[j] else -w[j], j))[:budget])
            holes = sorted(set(range(budget)) - set(kept))
            for to, of in zip(holes, [j for j in kept if j >= budget]):
                weight[s, h, to] = w0[s, h, of]; pos[s, h, to] = p0[s, h, of]
                a, b = page_of(table, n_pages, s, of, page), page_of(table, n_pages, s, to, page)
                if a >= 0 and b >= 0:
                    kc[b, h, to % page] = kc[a, h, of % page]; vc[b, h, to % page] = vc[a, h, of % page]
    return weight, pos, out


def beam(logits, score, n_beam, n_out, done=None, pad=0):
    """order: value descending, beam, logit descending, token; what is not a number counts as -inf, and -inf candidates have no other order than their index"""
    groups, V = logits.shape[0] // n_beam, logits.shape[1]
    res = np.zeros((groups, n_out)), np.zeros((groups, n_out), np.int32), np.zeros((groups, n_out), np.int32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            c, l = np.empty((n_beam, V)), logits[g * n_beam:(g + 1) * n_beam].astype(np.float64)
            for b in range(n_beam):
                x = l[b] - l[b].max()
                c[b] = float(score[g * n_beam + b]) + (x - np.log(np.exp(x).sum()))
                if done is not None and done[g * n_beam + b]:
                    c[b] = -np.inf; c[b, pad] = score[g * n_beam + b]
            c[np.isnan(c)] = -np.inf
            l = np.where(c == -np.inf, -np.inf, l)
            beams, tokens = np.divmod(np.arange(c.size), V)
            best = np.lexsort((tokens, -l.reshape(-1), beams, -c.reshape(-1)))[:n_out]
            res[0][g], res[1][g], res[2][g] = c.reshape(-1)[best], g * n_beam + beams[best], tokens[best]
    return res


def fork(kc, vc, table, n_kv, parent, fresh):
    n_pages, _, page, _ = kc.shape
    out, lens = np.full((len(parent), table.shape[1]), -1, np.int32), np.full(len(parent), -1, np.int32)
    k0, v0 = kc.copy(), vc.copy()
    for i, p in enumerate(parent):
        if not 0 <= p < len(n_kv) or n_kv[p] < 0:
            continue
        n = lens[i] = length(table, n_kv, p, page)
        out[i, :n // page] = table[p, :n // page]
        if n % page:
            f = int(fresh[i]); ok = 0 <= f < n_pages
            out[i, n // page] = f if ok else -1
            of = page_of(table, n_pages, p, n - 1, page)
            if ok and of >= 0:
                kc[f, :, :n % page] = k0[of, :, :n % page]; vc[f, :, :n % page] = v0[of, :, :n % page]
    return out, lens
