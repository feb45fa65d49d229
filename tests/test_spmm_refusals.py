"""What the block-vector product refuses, on the host: Python checks of the
tensors against the plan, and C-ABI checks that come before any CUDA call."""
import ctypes as C
import weakref

import numpy as np
import pytest
import torch

import diagpu_b200 as dg


def host_plan(n_rows=8, n_cols=8, offsets=(-1, 0, 1)):
    """A plan without device tables: the Python checks see CPU tensors as its own."""
    p = dg.SpmmPlan.__new__(dg.SpmmPlan)
    p._h = C.c_void_p()
    p.n_rows, p.n_cols = n_rows, n_cols
    p.offsets = np.array(offsets, np.int32)
    p.device = torch.device("cpu")
    return p


def good(dtype=torch.float32, E=None):
    plan = host_plan()
    vals = torch.zeros((3, 32) if E is None else (E, 3, 32), dtype=dtype)
    return plan, vals, torch.zeros(4, 8, dtype=dtype)


def refused(match, f, *a, **k):
    with pytest.raises(dg.DiaError, match=match) as e:
        f(*a, **k)
    assert e.value.code == dg.DIA_ERR_INVALID


def test_operator_and_block():
    plan, vals, x = good()
    refused("act must be", dg.spmm, plan, vals, x, act="swish")
    refused("not float32", dg.spmm, plan, vals, x.double())
    refused("not float32", dg.spmm, plan, vals, x.int())
    refused("vals must be", dg.spmm, plan, vals[:2], x)
    refused("vals must be", dg.spmm, plan, vals[None], x)
    refused("contiguous", dg.spmm, plan, vals.half(), x)
    refused("contiguous", dg.spmm, plan, torch.zeros(32, 3).t(), x)
    refused("x has shape", dg.spmm, plan, vals, torch.zeros(4, 7))
    refused("2-D", dg.spmm, plan, vals, torch.zeros(8))
    refused("adjacent", dg.spmm, plan, vals, torch.zeros(8, 4).t())
    refused("bias must be", dg.spmm, plan, vals, x, bias=torch.zeros(7))
    refused("residual has shape", dg.spmm, plan, vals, x, residual=torch.zeros(3, 8))
    refused("residual must be", dg.spmm, plan, vals, x, residual=torch.zeros(4, 8).half())


def test_experts():
    plan, vals, x = good(E=2)
    seg = torch.tensor([0, 1, 4])
    refused("vals must be", dg.spmm, plan, vals, x)
    refused("seg must be", dg.spmm, plan, vals, x, seg=seg[:2])
    refused("seg must be", dg.spmm, plan, vals, x, seg=seg.int())
    refused("seg must be", dg.spmm, plan, vals, x, seg=torch.zeros(6, dtype=torch.int64)[::2])
    refused("bias must be", dg.spmm, plan, vals, x, seg=seg, bias=torch.zeros(8))


def test_backward():
    plan, vals, x = good()
    dy = torch.zeros(4, 8)
    refused("must be given", dg.spmm_backward, plan, vals, x, None)
    refused("must be given", dg.spmm_backward, plan, vals, x, dy, act="gelu")
    refused("dy has shape", dg.spmm_backward, plan, vals, x, dy[:3])
    refused("z has shape", dg.spmm_backward, plan, vals, x, dy, z=dy[:3], act="relu")


def test_plan():
    refused("CUDA device", dg.SpmmPlan, 4, 4, [0], device="cpu")
    L = dg.lib()
    h = C.c_void_p()

    def create(nr, nc, off, plan=C.byref(h)):
        a = np.array(off, np.int32)
        return L.dia_spmm_plan_create(nr, nc, len(off), a.ctypes.data_as(C.c_void_p), plan)

    assert create(4, 4, [0], None) == dg.DIA_ERR_INVALID
    assert create(-1, 4, [0]) == dg.DIA_ERR_INVALID
    assert create(4, 4, [0, 1, 0]) == dg.DIA_ERR_INVALID
    assert "twice" in L.dia_last_error().decode()
    assert create(1 << 30, 1 << 30, [0]) == dg.DIA_ERR_UNSUPPORTED
    assert L.dia_spmm_plan_create(4, 4, 1, None, C.byref(h)) == dg.DIA_ERR_INVALID
    assert L.dia_spmm_plan_destroy(None) == dg.DIA_OK


def test_c_abi_before_cuda():
    L = dg.lib()

    def fwd(dtype=0, M=4, E=1, seg=None, act=0):
        return L.dia_spmm(None, dtype, M, E, seg, None, 8, None, 32, None, act, None, 8, None, 8,
                          None, 8, None, 0, None)

    def bwd(dtype=0, M=4, E=1, seg=None, act=0):
        return L.dia_spmm_backward(None, dtype, M, E, seg, None, 8, None, 32, None, 8, act, None,
                                   8, None, 8, None, None, None, 0, None)

    for f in (fwd, bwd):
        for bad, word in ((dict(dtype=3), "dtype"), (dict(act=5), "activation"),
                          (dict(act=-1), "activation"), (dict(M=-1), "rows"),
                          (dict(M=1 << 31), "rows"), (dict(E=0), "experts"),
                          (dict(E=2), "seg"), (dict(), "null plan")):
            assert f(**bad) == dg.DIA_ERR_INVALID
            assert word in L.dia_last_error().decode(), bad
    assert L.dia_spmm_workspace(None, 0, 4, 1, 8) == -1
    assert L.dia_spmm_backward_workspace(None, 0, 4, 1, 8, 32, 8, 0) == -1
    assert L.dia_test_spmm_form(3) == dg.DIA_ERR_INVALID


@pytest.mark.parametrize("nr,nc", [((1 << 63) - 1, (1 << 63) - 1), (1 << 62, 1 << 62),
                                   ((1 << 63) - 1, 1), (1, 1 << 40), (1 << 40, 0)])
def test_plan_sizes_past_32_bits(nr, nc):
    """No sum of two sizes wraps around into a size that is taken."""
    L, h, off = dg.lib(), C.c_void_p(), np.zeros(1, np.int32)
    rc = L.dia_spmm_plan_create(nr, nc, 1, off.ctypes.data_as(C.c_void_p), C.byref(h))
    assert rc == dg.DIA_ERR_UNSUPPORTED and not h.value


def test_workspace_lives_until_the_call_returns(monkeypatch):
    """Another thread on the same stream must not be given the workspace before
    the call has put its kernels on the stream: the tensor is alive in the C
    entry."""
    made, seen = [], []

    class Entries:
        @staticmethod
        def dia_spmm_workspace(*a):
            return 512

        dia_spmm_backward_workspace = dia_spmm_workspace

        @staticmethod
        def entry(*a):
            work, size = a[-3:-1]
            seen.append((size, [r() for r in made if r() is not None
                                and r().data_ptr() == work and r().numel() == size]))
            return 0

        dia_spmm = dia_spmm_backward = entry

    def new(stream, like, shape, dtype=None):
        t = torch.empty(shape, dtype=dtype or like.dtype)
        made.append(weakref.ref(t))
        return t

    monkeypatch.setattr(dg, "lib", lambda: Entries)
    monkeypatch.setattr(dg, "_spmm_new", new)
    monkeypatch.setattr(dg, "_spmm_stream", lambda plan, stream: 0)
    plan, vals, x = good()
    dg.spmm(plan, vals, x)
    dg.spmm_backward(plan, vals, x, torch.zeros(4, 8))
    assert [(size, len(alive)) for size, alive in seen] == [(512, 1), (512, 1)]


def test_workspace_queries():
    """They refuse what the calls refuse."""
    plan, vals, x = good()
    dy = torch.zeros(4, 8)
    for f, a in ((dg.spmm_workspace, ()), (dg.spmm_backward_workspace, (dy,))):
        refused("not float32", f, plan, vals.double(), x.double(), *(t.double() for t in a))
        refused("vals must be", f, plan, vals[:2], x, *a)
        refused("vals must be", f, plan, vals[0], x, *a)
        refused("contiguous", f, plan, vals.half(), x, *a)
        refused("2-D", f, plan, vals, x[0], *a)
    refused("act must be", dg.spmm_backward_workspace, plan, vals, x, dy, "swish")
