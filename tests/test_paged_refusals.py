"""What the paged-cache operators refuse, without a GPU: the C entry points with a context on the stand-in HIP runtime (tests/paged_refusal_case.py in a child process), the size functions
and the binding's own checks on host tensors."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

from conftest import load_package

HERE = os.path.dirname(os.path.abspath(__file__))


def test_entry_points_refuse_what_they_do_not_serve(tmp_path):
    if torch.cuda.is_available():
        pytest.skip("a real GPU is present: the stand-in runtime is for machines without one")
    if not shutil.which("g++") or not os.path.exists("/opt/rocm/include/hip/hip_runtime_api.h"):
        pytest.skip("needs g++ and the HIP headers to build the stand-in runtime")
    fake = str(tmp_path / "libfakehip.so")
    subprocess.check_call(["g++", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", fake, os.path.join(HERE, "fake_hip", "fake_hip.cpp")])
    p = subprocess.run([sys.executable, os.path.join(HERE, "paged_refusal_case.py")], capture_output=True, text=True, timeout=300, env=dict(os.environ, LD_PRELOAD=fake, FAKE_HIP_CAPTURE="1"))
    assert p.returncode == 0 and p.stdout.startswith("ok "), (p.returncode, p.stdout[-500:], p.stderr[-3000:])
    assert int(p.stdout.split()[1]) >= 150


@pytest.fixture
def be():
    """the binding over host tensors: the size functions and the checks in front of the library need no device"""
    pkg = load_package()
    b = object.__new__(pkg.Cdna4Backend)
    b.torch, b.lib, b.ctx, b.comm, b.window, b.device = torch, pkg.load_library(), None, None, None, torch.device("cpu")
    args = pkg.cdna4.load_args()
    b._desc, b._vec, b._empty, b._dev = args.desc, args.vec, args.empty, -1
    b._stream = lambda: None
    return b


def cache(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_size_functions_answer_and_refuse(be):
    Error = load_package().Cdna4Error
    k, table, q, slots = cache(9, 2, 16, 64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 8, 64), torch.zeros(3, 2, 64)
    assert be.paged_workspace(q, k, k, table) >= 0 and be.paged_workspace(q, k, k, table, weight=slots) >= be.paged_workspace(q, k, k, table)
    assert be.paged_workspace(q, k.transpose(1, 2).contiguous().transpose(1, 2), k, table) >= 0
    assert be.evict_workspace(k, k, table, slots, slots.int(), 8, 1, 2) > 0
    assert be.beam_workspace(torch.zeros(6, 100), 3, 5) > 0
    for bad in (lambda: be.paged_workspace(q[:, :7], k, k, table), lambda: be.paged_workspace(q, k, k[:8], table), lambda: be.paged_workspace(q.half(), k, k, table),
                lambda: be.paged_workspace(q, k.float(), k.float(), table), lambda: be.paged_workspace(q, k, k, table, weight=slots[:, :, :63]),
                lambda: be.paged_workspace(q, k[:, :, ::2], k[:, :, ::2], table[:, :1].float()), lambda: be.paged_workspace(q, k[:, :, :, :32], k[:, :, :, :32], table),
                lambda: be.evict_workspace(k, k, table, slots, slots, 8), lambda: be.evict_workspace(k, k, table, slots, slots.int(), 0), lambda: be.beam_workspace(torch.zeros(6, 100), 4, 5),
                lambda: be.beam_workspace(torch.zeros(6, 100, dtype=torch.float16), 3, 5), lambda: be.beam_workspace(torch.zeros(6, 100)[:, ::2], 3, 5)):
        with pytest.raises(Error):
            bad()


def test_the_binding_refuses_other_devices_types_and_shapes(be):
    Error = load_package().Cdna4Error
    k, table, q, n = cache(9, 2, 16, 64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 8, 64), torch.zeros(3, dtype=torch.int32)
    elsewhere = torch.zeros(3, 8, 64, device="meta")
    for bad in (lambda: be.paged_attn(elsewhere, k, k, table, n), lambda: be.paged_attn(q, k, k, table, n.long()), lambda: be.paged_attn(q, k, k, table, n[:2]), lambda: be.paged_attn(q, k, k, table[0], n),
                lambda: be.paged_attn(q.double(), k, k, table, n), lambda: be.paged_attn(None, k, k, table, n), lambda: be.paged_attn(q.to_sparse(), k, k, table, n), lambda: be.paged_attn(q, k, k, table[0, 0], n), lambda: be.paged_attn(q, k, k, table, torch.zeros(6, dtype=torch.int32)[::2]),
                lambda: be.paged_store(q[:, :2], q[:, :2], k, k, table, n, start=n), lambda: be.paged_fork(k, k, table, n, n[:2], n), lambda: be.paged_fork(k, k, table, n, None, n),
                lambda: be.beam_select(torch.zeros(6, 100), torch.zeros(5), 3, 2), lambda: be.beam_select(torch.zeros(6, 100), torch.zeros(6), 0, 2),
                lambda: be.beam_select(torch.zeros(6, 100), torch.zeros(6), 3, -1), lambda: be.paged_evict(k, k, table, n, torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), n, 8)):
        with pytest.raises(Error):
            bad()


def test_descriptors_say_what_the_tensors_are(be):
    import struct
    for dtype, code, size in ((torch.float32, 0, 4), (torch.float16, 1, 2), (torch.bfloat16, 30, 2), (torch.int32, 26, 4)):
        x = torch.zeros(7, 6, 5, 4, dtype=dtype)
        for y in (x, x[2], x[2, 1], x.transpose(1, 2), x[:, ::2, 1:, :3], x[3:4, :1], x[:0], x.permute(3, 0, 2, 1)):
            ptr, ty, *rest = struct.unpack("@Pi8q", be._desc(y, "x", -1))
            ne, nb = list(y.shape)[::-1], [s * size for s in y.stride()][::-1]
            assert (ptr, ty) == (y.data_ptr(), code) and rest[:4] == ne + [1] * (4 - len(ne)) and rest[4:] == nb + [0] * (4 - len(nb))
    v = torch.arange(9, dtype=torch.int32)
    assert be._vec(v[2:7], "v", 5, 26, -1) == v.data_ptr() + 8 and be._vec(None, "v", 5, 26, -1) is None
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        fake = torch.zeros(2, 3)
    for bad in (lambda: be._desc(fake, "x", -1), lambda: be._desc(torch.zeros(2, 3, dtype=torch.float64), "x", -1), lambda: be._desc(torch.zeros(2, 3), "x", 0), lambda: be._desc("x", "x", -1),
                lambda: be._vec(v[::2], "v", 5, 26, -1), lambda: be._vec(v, "v", 9, 0, -1), lambda: be._vec(v, "v", 9, 26, 0), lambda: be._desc(torch.zeros(1, 1, 1, 2, 3), "x", -1)):
        with pytest.raises(load_package().Cdna4Error):
            bad()
    with pytest.raises(TypeError):
        be._desc(v, "x")


def test_a_negated_view_is_refused(be):
    z = torch.zeros(3, 4, dtype=torch.complex64).conj().imag          # float32 values whose memory holds their negatives
    assert z.is_neg()
    for bad in (lambda: be._desc(z, "x", -1), lambda: be._vec(z[0], "v", 4, 0, -1)):
        with pytest.raises(load_package().Cdna4Error):
            bad()
    be._desc(z.resolve_neg(), "x", -1)


def test_the_binding_part_is_loaded_by_the_first_paged_call():
    pkg = load_package()
    b = object.__new__(pkg.Cdna4Backend)
    b.torch, b.lib, b.ctx, b.comm, b.window, b._dev = torch, pkg.load_library(), None, None, None, -1
    assert "_desc" not in b.__dict__
    with pytest.raises(AttributeError):
        b.no_such_method
    assert b.beam_workspace(torch.zeros(6, 100), 3, 5) > 0 and "_desc" in b.__dict__
