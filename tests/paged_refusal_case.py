"""Child process of tests/test_paged_refusals.py, started with the stand-in HIP runtime preloaded ("device" memory is host memory, launches do nothing): what the paged-cache entry points
refuse, with a context, and what they accept.  No result of a kernel is looked at.  Prints "ok <number of cases>"."""
import ctypes as C
import os
import sys

sys.modules["torch"] = None          # (the library alone: torch would bring the real runtime)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from conftest import load_package  # noqa: E402

pkg = load_package()


class _Tensor(C.Structure):          # cdna4_tensor
    _fields_ = [("data", C.c_void_p), ("type", C.c_int), ("ne", C.c_int64 * 4), ("nb", C.c_int64 * 4)]


lib = pkg.load_library()
ctx = lib.cdna4_init(0)
assert ctx, lib.cdna4_last_error()
F32, F16, Q8_0, I32, BF16 = 0, 1, 8, 26, 30
OK, UNSUPPORTED, INVALID, NOMEM = 0, -1, -2, -4
keep, cases = [], 0


def mem(n):
    b = C.create_string_buffer(n + 64); keep.append(b)
    return (C.addressof(b) + 63) & ~63


def tensor(t, *ne, nb=None, data=None):
    es = {F32: 4, F16: 2, BF16: 2, I32: 4, Q8_0: 1}[t]
    if nb is None:
        nb = [es]
        for n in ne[:-1]:
            nb.append(nb[-1] * max(n, 1))
    ne, nb = list(ne), list(nb)
    size = sum((n - 1) * b for n, b in zip(ne, nb)) + es
    while len(ne) < 4:
        nb.append(nb[-1] * max(ne[-1], 1)); ne.append(1)
    return _Tensor(mem(max(size, 64)) if data is None else data, t, (C.c_int64 * 4)(*ne), (C.c_int64 * 4)(*nb))


def base():
    return dict(k=tensor(F32, 64, 2, 3), v=tensor(F32, 64, 2, 3), kc=tensor(F16, 64, 16, 2, 10), vc=tensor(F16, 64, 16, 2, 10), table=tensor(I32, 4, 3), n_kv=mem(64), start=None, n_past=mem(64),
                weight=tensor(F32, 64, 2, 3), pos=tensor(I32, 64, 2, 3), n_out=mem(64), q=tensor(F32, 64, 8, 3), dst=tensor(F32, 64, 8, 3), weight_out=tensor(F32, 64, 2, 3),
                pos_out=tensor(I32, 64, 2, 3), budget=8, sink=1, recent=2, parent=mem(64), fresh=mem(64), table_out=tensor(I32, 4, 3), logits=tensor(F32, 100, 6), score=mem(64), done=mem(64),
                n_beam=3, n_best=5, pad=1, so=mem(64), po=mem(64), to=mem(64), ctx=ctx)


def r(x):
    return C.byref(x) if isinstance(x, _Tensor) else x


def call(op, a):
    a = {k: r(v) for k, v in a.items()}
    if op == "store":
        return lib.cdna4_op_paged_store(a["ctx"], a["k"], a["v"], a["kc"], a["vc"], a["table"], a["n_kv"], a["start"], a["n_past"], a["weight"], a["pos"], a["n_out"], None)
    if op == "attn":
        return lib.cdna4_op_paged_attn(a["ctx"], a["q"], a["kc"], a["vc"], a["table"], a["n_kv"], a["weight"], a["dst"], 0.125, 0.0, None)
    if op == "evict":
        return lib.cdna4_op_paged_evict(a["ctx"], a["kc"], a["vc"], a["table"], a["n_kv"], a["weight"], a["pos"], a["n_past"], a["budget"], a["sink"], a["recent"], a["weight_out"], a["pos_out"],
                                        a["n_out"], None)
    if op == "fork":
        return lib.cdna4_op_paged_fork(a["ctx"], a["kc"], a["vc"], a["table"], a["n_kv"], a["parent"], a["fresh"], a["table_out"], a["n_out"], None)
    return lib.cdna4_op_beam_select(a["ctx"], a["logits"], a["score"], a["done"], a["n_beam"], a["n_best"], a["pad"], a["so"], a["po"], a["to"], None)


def expect(op, want, **change):
    global cases
    a = base(); a.update({k: (v(a) if callable(v) else v) for k, v in change.items()})
    got = call(op, a); cases += 1
    assert got == want, (op, want, got, list(change), lib.cdna4_last_error())
    assert want == OK or lib.cdna4_last_error()


PAGED = ("store", "attn", "evict", "fork")
for op in PAGED + ("beam",):
    expect(op, OK)
    expect(op, INVALID, ctx=None)
for op in PAGED:
    for name in ("kc", "vc", "table", "n_kv"):
        expect(op, INVALID, **{name: None})
    caches = lambda *s, **kw: {"kc": lambda a: tensor(*s, **kw), "vc": lambda a: tensor(*s, **kw)}  # noqa: E731
    expect(op, OK, **caches(BF16, 64, 16, 2, 10))
    expect(op, OK, **caches(F16, 64, 16, 2, 10, nb=(2, 256, 128, 4096)))                      # token-major
    expect(op, UNSUPPORTED, **caches(F32, 64, 16, 2, 10))
    expect(op, UNSUPPORTED, **caches(Q8_0, 64, 16, 2, 10))
    expect(op, UNSUPPORTED, vc=lambda a: tensor(BF16, 64, 16, 2, 10))
    expect(op, INVALID, vc=lambda a: tensor(F16, 64, 16, 2, 11))
    expect(op, UNSUPPORTED, **caches(F16, 80, 16, 2, 10))
    for page in (0, 8, 24, 8192):
        expect(op, UNSUPPORTED, **caches(F16, 64, page, 2, 10))
    expect(op, UNSUPPORTED, **caches(F16, 64, 16, 2, 0))
    expect(op, UNSUPPORTED, **caches(F16, 64, 16, 0, 10))
    expect(op, UNSUPPORTED, **caches(F16, 64, 16, 2, 10, nb=(4, 256, 4096, 8192)))            # not dense
    expect(op, UNSUPPORTED, **caches(F16, 64, 16, 2, 10, nb=(2, 136, 4352, 8704)))            # rows off 16 bytes
    expect(op, UNSUPPORTED, **caches(F16, 64, 16, 2, 10, nb=(2, 1 << 28, 128, 1 << 34), data=4096))
    expect(op, UNSUPPORTED, kc=lambda a: tensor(F16, 64, 16, 2, 10, data=a["kc"].data + 8))
    expect(op, INVALID, **caches(F16, 64, 16, 2, 10, nb=(2, -128, 2048, 4096), data=1 << 20))
    if op != "attn":                                                                           # (a cache that is only read may repeat itself)
        expect(op, INVALID, **caches(F16, 64, 16, 2, 10, nb=(2, 128, 0, 2048)))
        expect(op, INVALID, **caches(F16, 64, 16, 2, 10, nb=(2, 64, 2048, 4096)))
    else:
        expect(op, OK, **caches(F16, 64, 16, 2, 10, nb=(2, 128, 0, 2048)))
    expect(op, INVALID, table=lambda a: tensor(F32, 4, 3))
    expect(op, INVALID, table=lambda a: tensor(I32, 4, 3, nb=(8, 32)))
    expect(op, INVALID, kc=lambda a: tensor(F16, 64, 16, 2, 10, data=0) if False else _Tensor(None, F16, a["kc"].ne, a["kc"].nb))
    expect(op, UNSUPPORTED, table=lambda a: tensor(I32, (1 << 26) + 1, 3, data=4096))
    expect(op, UNSUPPORTED, table=lambda a: tensor(I32, 4, 8193))
# store
expect("store", OK, weight=None, pos=None, n_past=None, n_out=None)
expect("store", OK, start=lambda a: mem(64), k=lambda a: tensor(F32, 64, 2, 9), v=lambda a: tensor(F32, 64, 2, 9))
expect("store", OK, start=lambda a: mem(64), k=lambda a: tensor(F32, 64, 2, 0), v=lambda a: tensor(F32, 64, 2, 0))
expect("store", INVALID, k=None)
expect("store", INVALID, k=lambda a: tensor(F32, 64, 2, 9), v=lambda a: tensor(F32, 64, 2, 9))
expect("store", INVALID, start=lambda a: mem(64), k=lambda a: tensor(F32, 64, 2, 9))
expect("store", INVALID, k=lambda a: tensor(F16, 64, 2, 3))
expect("store", INVALID, k=lambda a: tensor(F32, 64, 1, 3))
expect("store", UNSUPPORTED, k=lambda a: tensor(F32, 64, 2, 3, nb=(4, 264, 528)))
expect("store", INVALID, n_past=None)
expect("store", INVALID, n_out=lambda a: a["n_kv"] + 8)
expect("store", INVALID, n_out=lambda a: a["n_past"] + 8)
expect("store", INVALID, start=lambda a: a["n_out"])
expect("store", INVALID, pos=lambda a: tensor(I32, 64, 2, 3, data=a["weight"].data + 256))
expect("store", INVALID, weight=lambda a: tensor(F32, 63, 2, 3))
expect("store", INVALID, weight=lambda a: tensor(F32, 64, 2, 3, nb=(4, 0, 256)))
expect("store", INVALID, pos=lambda a: tensor(F32, 64, 2, 3))
# attn
expect("attn", OK, weight=None)
expect("attn", INVALID, q=lambda a: tensor(F32, 64, 7, 3), dst=lambda a: tensor(F32, 64, 7, 3))
expect("attn", INVALID, q=lambda a: tensor(F16, 64, 8, 3))
expect("attn", INVALID, dst=lambda a: tensor(F32, 64, 8, 2))
expect("attn", INVALID, q=None)
expect("attn", INVALID, dst=None)
expect("attn", INVALID, dst=lambda a: a["q"])
expect("attn", INVALID, dst=lambda a: tensor(F32, 64, 8, 3, nb=(4, 256, 0)))
expect("attn", OK, q=lambda a: tensor(F32, 64, 8, 3, nb=(4, 256, 0)))
expect("attn", UNSUPPORTED, q=lambda a: tensor(F32, 64, 8, 3, nb=(4, 260, 2080)))
expect("attn", INVALID, weight=lambda a: tensor(F32, 64, 8, 3))
expect("attn", INVALID, weight=lambda a: tensor(F32, 64, 2, 3, data=a["dst"].data + 1024))
one = dict(kc=lambda a: tensor(F16, 64, 16, 1, 10, nb=(2, 128, 7, 2048)), vc=lambda a: tensor(F16, 64, 16, 1, 10, nb=(2, 128, 7, 2048)), q=lambda a: tensor(F32, 64, 8, 3),
           weight=lambda a: tensor(F32, 64, 1, 3, nb=(4, 1, 256)))
expect("attn", OK, **one)                                                                      # (strides of one-element dimensions do not count)
# evict
for name in ("weight", "pos", "weight_out", "pos_out", "n_past", "n_out"):
    expect("evict", INVALID, **{name: None})
expect("evict", OK, weight_out=lambda a: a["weight"], pos_out=lambda a: a["pos"])
expect("evict", INVALID, weight_out=lambda a: a["weight"])                                    # one in place, the other not
expect("evict", INVALID, weight_out=lambda a: tensor(F32, 64, 2, 3, data=a["weight"].data + 4))
expect("evict", INVALID, pos_out=lambda a: tensor(I32, 64, 2, 3, data=a["weight"].data))
expect("evict", INVALID, pos_out=lambda a: tensor(I32, 64, 2, 3, data=a["weight_out"].data))
expect("evict", INVALID, n_out=lambda a: a["n_kv"])
expect("evict", INVALID, n_out=lambda a: a["n_past"])
for budget, sink, recent, want in ((0, 0, 0, INVALID), (-1, 0, 0, INVALID), (8, 5, 4, INVALID), (8, -1, 0, INVALID), (8, 0, -1, INVALID), (8, 4, 4, OK), (1, 0, 0, OK), (2 ** 31 - 1, 2 ** 31 - 1, 0, OK),
                                   (2 ** 31 - 1, 2 ** 31 - 1, 1, INVALID)):
    expect("evict", want, budget=budget, sink=sink, recent=recent)
# fork
for name in ("parent", "fresh", "table_out", "n_out"):
    expect("fork", INVALID, **{name: None})
expect("fork", INVALID, table_out=lambda a: a["table"])
expect("fork", INVALID, table_out=lambda a: tensor(I32, 4, 3, data=a["table"].data + 44))
expect("fork", INVALID, table_out=lambda a: tensor(I32, 5, 3))
expect("fork", INVALID, table_out=lambda a: tensor(I32, 4, 3, nb=(4, 8)))
expect("fork", INVALID, table_out=lambda a: tensor(I32, 4, 3, data=a["parent"]))
expect("fork", INVALID, n_out=lambda a: a["n_kv"])
expect("fork", INVALID, n_out=lambda a: a["parent"] + 4)
expect("fork", OK, table_out=lambda a: tensor(I32, 4, 0))
expect("fork", OK, table_out=lambda a: tensor(I32, 4, 7))
# beam
for name in ("logits", "score", "so", "po", "to"):
    expect("beam", INVALID, **{name: None})
expect("beam", OK, done=None)
expect("beam", OK, logits=lambda a: tensor(F32, 100, 0))
for n_beam, n_best, pad, want in ((0, 5, 1, UNSUPPORTED), (4, 5, 1, INVALID), (257, 5, 1, UNSUPPORTED), (3, 0, 1, UNSUPPORTED), (3, 65, 1, UNSUPPORTED), (3, 64, 1, OK), (3, 5, 100, INVALID), (3, 5, -1, INVALID)):
    expect("beam", want, n_beam=n_beam, n_best=n_best, pad=pad, so=lambda a: mem(1024), po=lambda a: mem(1024), to=lambda a: mem(1024))
expect("beam", UNSUPPORTED, logits=lambda a: tensor(F32, 1, 6), n_best=4)
expect("beam", INVALID, logits=lambda a: tensor(F16, 100, 6))
expect("beam", UNSUPPORTED, logits=lambda a: tensor(F32, 100, 6, nb=(8, 800)))
expect("beam", UNSUPPORTED, logits=lambda a: tensor(F32, 1 << 30, 6, data=4096))
expect("beam", INVALID, po=lambda a: a["so"] + 16)
expect("beam", INVALID, so=lambda a: a["score"])
expect("beam", INVALID, to=lambda a: a["logits"].data + 400)
# a workspace that would have to grow under a capture is refused; the size functions say what to reserve
if os.environ.get("FAKE_HIP_CAPTURE"):
    hip = C.CDLL(None); st = C.c_void_p(); assert hip.hipStreamCreateWithFlags(C.byref(st), 0) == 0
    big = dict(logits=tensor(F32, 100000, 4000), so=mem(1 << 20), po=mem(1 << 20), to=mem(1 << 20), score=mem(1 << 16), done=mem(1 << 16)); a = base(); a.update(big)
    need = lib.cdna4_beam_select_workspace(r(a["logits"]), 4, 64, 0)
    a.update(n_beam=4, n_best=64, pad=0)
    args = [r(a[x]) for x in ("ctx", "logits", "score", "done", "n_beam", "n_best", "pad", "so", "po", "to")]
    epoch = lib.cdna4_workspace_epoch(ctx)
    assert hip.hipStreamBeginCapture(st, 0) == 0
    assert need <= (1 << 20) or lib.cdna4_op_beam_select(*args, st) == NOMEM, need
    g = C.c_void_p(); assert hip.hipStreamEndCapture(st, C.byref(g)) == 0
    assert lib.cdna4_workspace_epoch(ctx) == epoch and lib.cdna4_reserve_workspace(ctx, need) == OK
    assert hip.hipStreamBeginCapture(st, 0) == 0 and lib.cdna4_op_beam_select(*args, st) == OK
    cases += 2
print("ok", cases)
