"""Child process of tests/test_paged_overlaps.py on the stand-in HIP runtime: arguments that share memory where a call writes.  Runs the cases of paged_refusal_case.py first (its helpers are
used).  Prints "overlaps ok <number>"."""
import paged_refusal_case as base
from paged_refusal_case import F16, F32, I32, INVALID, OK, expect, mem, tensor

before = base.cases


def at(name, off=0):
    return lambda a: (a[name] if isinstance(a[name], int) else a[name].data) + off


def f32(*ne):
    return lambda name, off=0: lambda a: tensor(F32, *ne, data=at(name, off)(a))


def i32(*ne):
    return lambda name, off=0: lambda a: tensor(I32, *ne, data=at(name, off)(a))


slots, pslots, rows, row, tab = f32(64, 2, 3), i32(64, 2, 3), f32(64, 8, 3), f32(64, 2, 3), i32(4, 3)
# what a call writes on what it reads or writes
for other in ("k", "v", "kc", "vc", "table", "n_kv", "n_past", "weight", "pos"):
    expect("store", INVALID, n_out=at(other))
for other in ("k", "v", "kc", "vc", "table", "n_kv", "n_past", "pos"):
    expect("store", INVALID, weight=slots(other))
for other in ("k", "v", "kc", "vc", "table", "n_kv", "n_past", "weight"):
    expect("store", INVALID, pos=pslots(other))
for other in ("kc", "vc"):
    expect("store", INVALID, k=row(other))
    expect("store", INVALID, v=row(other, 64))
    expect("store", INVALID, table=tab(other, 16))
    expect("store", INVALID, start=at(other, 32))
    expect("store", INVALID, n_kv=at(other, 32))
for other in ("q", "weight", "kc", "vc", "table", "n_kv"):
    expect("attn", INVALID, dst=rows(other))
for other in ("q", "kc", "vc", "table", "n_kv"):
    expect("attn", INVALID, weight=slots(other, 0))
for other in ("kc", "vc", "table", "n_kv", "weight", "pos", "n_past", "pos_out", "weight_out"):
    expect("evict", INVALID, n_out=at(other))
for other in ("kc", "vc", "table", "n_kv", "pos", "n_past"):
    expect("evict", INVALID, weight_out=slots(other))
for other in ("kc", "vc", "table", "n_kv", "weight", "n_past"):
    expect("evict", INVALID, pos_out=pslots(other))
for other in ("kc", "vc"):
    expect("evict", INVALID, weight=slots(other), weight_out=slots(other), pos_out=lambda a: a["pos"])
    expect("evict", INVALID, table=tab(other, 16))
for other in ("kc", "vc", "table", "n_kv", "parent", "fresh", "table_out"):
    expect("fork", INVALID, n_out=at(other))
for other in ("kc", "vc", "table", "n_kv", "parent", "fresh"):
    expect("fork", INVALID, table_out=tab(other))
for other in ("kc", "vc"):
    expect("fork", INVALID, parent=at(other, 4))
    expect("fork", INVALID, table=tab(other, 16))
# what is only read may be one and the same
expect("store", OK, n_past=lambda a: a["n_kv"], v=lambda a: a["k"])
expect("attn", OK, vc=lambda a: a["kc"])
expect("evict", OK, n_past=lambda a: a["n_kv"])
expect("evict", OK, weight_out=lambda a: a["weight"], pos_out=lambda a: a["pos"])
expect("fork", OK, fresh=lambda a: a["parent"])
# neighbours are apart; nothing is at the address of an empty tensor
expect("attn", OK, q=lambda a: tensor(F32, 64, 8, 3, data=a["dst"].data + 64 * 8 * 3 * 4))
expect("fork", OK, table=lambda a: tensor(I32, 0, 3), table_out=lambda a: tensor(I32, 0, 3, data=a["kc"].data))
print("overlaps ok", base.cases - before)
