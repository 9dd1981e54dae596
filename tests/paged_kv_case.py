"""Child process of tests/test_paged_overlaps.py on the stand-in HIP runtime: K and V caches in one pool.  Every layout is also laid out element by element on the host: what is accepted has no
byte twice.  Prints "kv ok <accepted> <refused>"."""
import itertools

from paged_refusal_case import F16, INVALID, OK, expect, mem, tensor

D, page, heads, pages = 64, 16, 2, 10
pool = mem(1 << 20)
count = {OK: 0, INVALID: 0}


def apart(nbk, nbv, off):
    def rows(nb, base):          # every row is D dense elements
        return [base + s * nb[1] + h * nb[2] + p * nb[3] for s, h, p in itertools.product(range(page), range(heads), range(pages))]
    x = sorted(rows(nbk, 0) + rows(nbv, off))
    return all(b - a >= 2 * D for a, b in zip(x, x[1:]))


def case(nbk, nbv, off, must=None):
    """must: what has to be answered; None: whatever, as long as nothing that overlaps is accepted"""
    ok = apart(nbk, nbv, off)
    if must is not None:
        assert ok == (must == OK), (nbk, nbv, off)
    want = must if must is not None else (INVALID if not ok else None)
    if want is None:
        return
    for op in ("store", "evict", "fork"):
        expect(op, want, kc=lambda a: tensor(F16, D, page, heads, pages, nb=nbk, data=pool), vc=lambda a: tensor(F16, D, page, heads, pages, nb=nbv, data=pool + off))
        expect(op, want, vc=lambda a: tensor(F16, D, page, heads, pages, nb=nbk, data=pool), kc=lambda a: tensor(F16, D, page, heads, pages, nb=nbv, data=pool + off))
    expect("attn", OK, kc=lambda a: tensor(F16, D, page, heads, pages, nb=nbk, data=pool), vc=lambda a: tensor(F16, D, page, heads, pages, nb=nbv, data=pool + off))          # (only read)
    count[want] += 1


r = 2 * D
head_major, token_major = (2, r, r * page, r * page * heads), (2, r * heads, r, r * page * heads)
full = r * page * heads
for nb in (head_major, token_major):
    case(nb, nb, 0, INVALID)                                           # one tensor for both
    case(nb, nb, full, INVALID)                                        # a page further
    case(nb, nb, r, INVALID)
    case(nb, nb, full * pages, OK)                                     # one behind the other
    case(nb, nb, full * pages - r, INVALID)
    wide = nb[:3] + (2 * full,)
    case(wide, wide, full, OK)                                         # [pages, 2, ...]
    case(wide, wide, 3 * full, OK)                                     # V a page further
    case(wide, wide, full - r, INVALID)
    case(wide, wide, 2 * full, INVALID)
case((2, r, 2 * r * page, 2 * full), (2, r, 2 * r * page, 2 * full), r * page, OK)             # [pages, heads, 2, page, D]
case((2, 2 * r, 2 * r * page, 2 * full), (2, 2 * r, 2 * r * page, 2 * full), r, OK)            # K and V of a slot side by side
case((2, 2 * r * heads, r, 2 * full), (2, 2 * r * heads, r, 2 * full), r * heads, OK)          # [pages, page, 2, heads, D]
case(head_major[:3] + (2 * full,), token_major[:3] + (2 * full,), full, OK)                    # different orders in a pool of pages
case((2, 2 * r * heads * pages, r, r * heads), (2, 2 * r * heads * pages, r, r * heads), r * heads * pages, OK)          # [page, 2, pages, heads, D]
for off in range(0, 5 * full, 16 * 61):
    for nb in (head_major, token_major, head_major[:3] + (2 * full,), (2, 2 * r, 2 * r * page, 2 * full), (2, 2 * r * heads, r, 3 * full)):
        case(nb, nb, off)
        case(nb, token_major, off)
print("kv ok", count[OK], count[INVALID])
