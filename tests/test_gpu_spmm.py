"""A DIA operator times a block of vectors (spmm, spmm_backward) against its
definition in 64 bits on the CPU.

Tolerances are elementwise bounds.  u is half a step of the block's type, a an
fp32 sum's unit (2^-24; 2^-22 for 16-bit types, whose sums may run on tensor
cores, which align products before adding and cut rather than round).  With S
the sum of |terms| of one output, a sum of K terms is off by at most (K+4) a S
in any order.  An activation and its derivative are evaluated to within e|z|
and e (e = 2^-18; 2^-13 for 16-bit types, a quarter of fp16's half step), and
change by at most 1.13 times a change of z.  dz is rounded to the block's
type.  Storing rounds once more (fp16 also flushes to steps of 2^-24)."""
import math

import numpy as np
import pytest
import torch

import diagpu_b200 as dg

pytestmark = pytest.mark.gpu

# type and form (dia_test_spmm_form): CUDA cores, or tensor cores where they can run
FORMS = {"fp32": (torch.float32, 0), "fp16": (torch.float16, 1), "fp16-tc": (torch.float16, 2),
         "bf16": (torch.bfloat16, 1), "bf16-tc": (torch.bfloat16, 2),
         "bf16-rule": (torch.bfloat16, 0)}
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(params=FORMS)
def t(request):
    dtype, form = FORMS[request.param]
    dg.check(dg.lib().dia_test_spmm_form(form))
    yield dtype
    dg.check(dg.lib().dia_test_spmm_form(0))
    assert dg.device_status() == 0      # no wait of a kernel ran out


def unit(t):
    return torch.finfo(t).eps / 2


def sum_unit(t):
    return 2.0 ** -24 if t == torch.float32 else 2.0 ** -22


def act_err(t):
    return 2.0 ** -18 if t == torch.float32 else 2.0 ** -13


def tiny(t):
    return 2.0 ** -24 if t == torch.float16 else 1e-37


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def dact64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return (0.5 * torch.special.erfc(-z * math.sqrt(0.5))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def spans(off, n, m):
    for k, d in enumerate(off):
        lo, hi = max(0, -d), min(n, m - d)
        if hi > lo:
            yield k, d, lo, hi


def product64(off, n, m, vals, x, parts, bias=None):
    """z and the sum of |terms|."""
    z = torch.zeros(x.shape[0], n, dtype=torch.float64)
    S = torch.zeros_like(z)
    for e, a, b in parts:
        for k, d, lo, hi in spans(off, n, m):
            p = vals[e, k, lo:hi] * x[a:b, lo + d:hi + d]
            z[a:b, lo:hi] += p
            S[a:b, lo:hi] += p.abs()
        if bias is not None:
            z[a:b] += bias[e]
            S[a:b] += bias[e].abs()
    return z, S


def gradient64(off, n, m, vals, x, dz, parts):
    dx, dv = torch.zeros_like(x), torch.zeros_like(vals)
    db = torch.zeros(vals.shape[0], n, dtype=torch.float64)
    for e, a, b in parts:
        db[e] = dz[a:b].sum(0)
        for k, d, lo, hi in spans(off, n, m):
            dx[a:b, lo + d:hi + d] += vals[e, k, lo:hi] * dz[a:b, lo:hi]
            dv[e, k, lo:hi] = (dz[a:b, lo:hi] * x[a:b, lo + d:hi + d]).sum(0)
    return dx, dv, db


def near(got, want, tol, what):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), (got - want).abs()[bad][:4].tolist(),
                                 tol[bad][:4].tolist(), bad.nonzero()[:4].tolist())


class Case:
    """Inputs on the GPU and, exactly the same values, in 64 bits on the CPU."""

    def __init__(self, t, M, n, m, off, *, seed=0, seg=None, ld=None, shift=0, junk=None,
                 mult=True):
        g = torch.Generator().manual_seed(seed)
        self.t, self.M, self.n, self.m, self.off, self.seg = t, M, n, m, list(off), seg
        self.E = 1 if seg is None else len(seg) - 1
        K = len(self.off)
        stride = max(32, (n + 31) // 32 * 32)
        v = torch.zeros(self.E, K, stride, dtype=torch.float64)
        if junk is not None:
            v += junk
        for k, d, lo, hi in spans(self.off, n, m):
            v[:, k, lo:hi] = torch.randn(self.E, hi - lo, generator=g, dtype=torch.float64)
        self.vals = v.to(t).cuda()
        self.ld, self.shift = ld, shift
        self.x = self.block(torch.randn(M, m, generator=g))
        self.dy = self.block(torch.randn(M, n, generator=g))
        self.zin = self.block(torch.randn(M, n, generator=g) * 2)
        self.res = self.block(torch.randn(M, n, generator=g))
        self.bias = torch.randn(self.E, n, generator=g).to(t).cuda()
        if seg is None:
            self.parts = [(0, 0, M)]
            self.dseg = None
        else:
            self.parts = [(e, seg[e], seg[e + 1]) for e in range(self.E)]
            self.dseg = torch.tensor(seg, dtype=torch.int64).cuda()
        self.plan = dg.SpmmPlan(n, m, np.array(self.off, np.int32))

    def block(self, v):
        """v on the GPU in rows of ld elements (None: adjacent), `shift` elements
        past an aligned address."""
        M, w = v.shape
        ld = w if self.ld is None else w + self.ld
        buf = torch.full((M * ld + self.shift + 8,), 7.0, dtype=self.t, device="cuda")
        b = buf[self.shift:self.shift + M * ld].view(M, ld)[:, :w]
        b.copy_(v)
        return b

    def v(self, a):
        return a.double().cpu()

    def pv(self):
        return self.vals if self.seg is not None else self.vals[0]

    def rows(self):
        r = torch.zeros(self.M, dtype=torch.bool)
        for _, a, b in self.parts:
            r[a:b] = True
        return r

    def product(self, act="none", bias=False, res=False, z=False):
        out = self.block(torch.full((self.M, self.n), 3.0))
        zb = self.block(torch.full((self.M, self.n), 5.0)) if z else None
        b = None if not bias else (self.bias if self.seg is not None else self.bias[0])
        r = dg.spmm(self.plan, self.pv(), self.x, bias=b, act=act,
                    residual=self.res if res else None, seg=self.dseg, out=out, z=zb)
        y = r[0] if z else r
        t, K, u = self.t, len(self.off), unit(self.t)
        z64, S = product64(self.off, self.n, self.m, self.v(self.vals), self.v(self.x),
                           self.parts, self.v(self.bias) if bias else None)
        ez = (K + 4) * sum_unit(t) * S
        f = act64(z64, act)
        want = f + (self.v(self.res) if res else 0)
        tol = 1.13 * ez + (act_err(t) * z64.abs() if act not in ("none", "relu") else 0)
        tol = tol + 2.0 ** -23 * (f.abs() + want.abs())
        on = self.rows()
        near(y[on], want[on], (tol + u * (want.abs() + tol) + tiny(t))[on], "y")
        assert bool((y[~on].cpu() == 3).all())
        if z:
            near(r[1][on], z64[on], (ez + u * (z64.abs() + ez) + tiny(t))[on], "z")
            assert bool((r[1][~on].cpu() == 5).all())
        return y

    def gradient(self, act="none", bias=True):
        t, K, u, n, m = self.t, len(self.off), unit(self.t), self.n, self.m
        dx = self.block(torch.full((self.M, m), 3.0))
        dv = torch.full_like(self.vals, 9.0)
        db = torch.full_like(self.bias, 9.0) if bias else None
        z = self.zin if act != "none" else None
        sq = (lambda a: a) if self.seg is not None else (lambda a: a[0])
        dg.spmm_backward(self.plan, self.pv(), self.x, self.dy, z=z, act=act, seg=self.dseg,
                         dx=dx, dvals=sq(dv), dbias=sq(db) if bias else None)
        dy, x, vals = self.v(self.dy), self.v(self.x), self.v(self.vals)
        dz = dy if act == "none" else dy * dact64(self.v(self.zin), act)
        ed = torch.zeros_like(dz)
        if act != "none":
            ed = 1.01 * u * dz.abs() + tiny(t)
            if act != "relu":
                ed += 1.01 * act_err(t) * dy.abs()
        gx, gv, gb = gradient64(self.off, n, m, vals, x, dz, self.parts)
        sx, sv, sb = gradient64(self.off, n, m, vals.abs(), x.abs(), dz.abs(), self.parts)
        tx, tv, tb = gradient64(self.off, n, m, vals.abs(), x.abs(), ed, self.parts)
        on = self.rows()
        long = max([b - a for _, a, b in self.parts], default=0)
        for got, want, S, T, terms, what in ((dx[on], gx[on], sx[on], tx[on], K, "dx"),
                                             (dv, gv, sv, tv, long, "dvals"),
                                             (db, gb, sb, tb, long, "dbias")):
            if got is None:
                continue
            e = T + (terms + 4) * sum_unit(t) * (S + T)
            near(got, want, e + u * (want.abs() + e) + tiny(t), what)
        assert bool((dx[~on].cpu() == 3).all())
        return dx, dv, db


def band(w):
    return list(range(-w, w + 1))


# name: (M, n_rows, n_cols, offsets)
SHAPES = {
    "one": (1, 1, 1, [0]),
    "one row": (1, 128, 128, band(3)),
    "odd": (5, 37, 37, band(4)),
    "unsorted": (9, 64, 64, [5, -3, 0, 1, 40, -63]),
    "no diagonal": (3, 40, 40, []),
    "outside": (4, 40, 33, [0, 33, 100, -40, -39, 2 ** 30, -2 ** 31]),
    "wide": (7, 100, 260, [0, 1, 2, 100, 159, 259, -99]),
    "tall": (66, 260, 100, [0, -1, -159, 99, -259, -160, -161]),
    "tile": (128, 128, 128, band(64)),
    "tile+1": (129, 129, 136, band(64)),
    "wide band": (200, 328, 328, band(130)),
    "scattered": (130, 640, 640, [-512, -377, -200, -111, -64, -7, 0, 1, 13, 90, 255, 511]),
    "stencil": (257, 512, 512, [i + 8 * j + 64 * k for i in (-1, 0, 1) for j in (-1, 0, 1)
                                for k in (-1, 0, 1)]),
    "long": (700, 264, 264, band(20)),
    "odd widths": (300, 131, 203, [-40, -39, 0, 1, 2, 3, 70, 71, 90]),
}


@pytest.mark.parametrize("shape", SHAPES)
def test_product(shape, t):
    Case(t, *SHAPES[shape], seed=1).product(bias=True)


@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(shape, t):
    Case(t, *SHAPES[shape], seed=2).gradient(act="silu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [2, 150])
def test_epilogue(M, act, t):
    c = Case(t, M, 200, 200, band(9), seed=3)
    c.product(act=act, bias=True, res=True, z=True)
    c.product(act=act, z=True)
    c.product(act=act, res=True)
    c.gradient(act=act)
    c.gradient(act=act, bias=False)


@pytest.mark.parametrize("ld,shift", [(8, 0), (1, 0), (None, 1), (24, 8), (3, 3), (64, 2)])
def test_strides_and_alignment(ld, shift, t):
    c = Case(t, 140, 136, 144, band(12), seed=4, ld=ld, shift=shift)
    c.product(act="gelu", bias=True, res=True, z=True)
    c.gradient(act="gelu")


SEGS = {
    "one expert": [0, 150],
    "empty ones": [0, 0, 1, 1, 64, 64, 64, 150, 150],
    "rows around": [3, 40, 140],
    "no rows": [0, 0, 0],
    "none at the end": [10, 10],
    "many": list(range(0, 151)),
    "ragged": [0, 2, 7, 8, 71, 149, 149, 150],
}


@pytest.mark.parametrize("name", SEGS)
def test_experts(name, t):
    c = Case(t, 150, 136, 136, band(10), seed=5, seg=SEGS[name])
    c.product(act="silu", bias=True, res=True, z=True)
    c.gradient(act="silu")


def test_experts_long_and_short(t):
    c = Case(t, 1500, 72, 72, band(3), seed=6, seg=[0, 1100, 1101, 1101, 1500])
    c.product(act="gelu", bias=True)
    c.gradient(act="gelu")


# Long blocks: a CTA of the tensor-core form goes around its accumulators, keeps
# an operator for many tiles or reads a large one again, takes a stretch of the
# tiles or every so-manieth; parts of the gradient are joined.
LONG = {
    "band": (60000, 136, 136, band(4)),
    "scattered": (30000, 264, 264, [-250, -201, -130, -64, -3, 0, 55, 120, 199, 260]),
    "stretches": (600, 6400, 6400, [-2, -1, 0, 1, 700]),
}


@pytest.mark.parametrize("shape", LONG)
def test_long_blocks(shape, t):
    c = Case(t, *LONG[shape], seed=21)
    c.product(act="silu", bias=True, res=True, z=True)
    c.gradient(act="silu")
    c.gradient(act="none")


def test_long_blocks_of_experts(t):
    c = Case(t, 20000, 136, 136, [-70, -8, 0, 1, 2, 65], seed=22,
             seg=[0, 9000, 9000, 9001, 9700, 20000])
    c.product(act="gelu", bias=True, res=True, z=True)
    c.gradient(act="gelu")


@pytest.mark.parametrize("M", [3, 140])
def test_unread_values(M, t):
    """Bits outside the matrix, in the padding and in rows outside every expert
    do not reach a result."""
    nan = float("nan")
    c = Case(t, M, 130, 120, band(20), seed=7, junk=nan, seg=[1, 2, M - 1])
    for b in (c.x, c.dy, c.zin, c.res):
        b[0] = nan
        b[M - 1] = nan
    c.product(act="gelu", bias=True, res=True)
    outside = c.vals.isnan()
    dx = torch.zeros(M, 120, dtype=t, device="cuda")
    dv = torch.full_like(c.vals, 9.0)
    db = torch.full_like(c.bias, 9.0)
    dg.spmm_backward(c.plan, c.vals, c.x, c.dy, z=c.zin, act="gelu", seg=c.dseg, dx=dx, dvals=dv,
                     dbias=db)
    assert bool(dx.isfinite().all() and dv.isfinite().all() and db.isfinite().all())
    assert bool((dv[outside] == 0).all())


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinite_values_stay_where_they_belong(value, M, t):
    """An infinite or undefined feature reaches exactly the outputs that a
    diagonal joins to it.  The rest keep their values; a sum that the tensor
    cores' zeros met it in is computed again, in another order, so each of the
    two is within the sums' bound of the same number, and storing rounds both."""
    n, off = 200, [-33, -2, 0, 5, 6, 70]
    c = Case(t, M, n, n, off, seed=8)
    x0, dy0 = c.x.clone(), c.dy.clone()
    y0 = dg.spmm(c.plan, c.vals[0], c.x)
    dx0, dv0, _ = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)
    K, u = len(off), unit(t)
    sx, sv, _ = gradient64(off, n, n, c.v(c.vals).abs(), c.v(c.x).abs(), c.v(c.dy).abs(), c.parts)
    sy = product64(off, n, n, c.v(c.vals), c.v(c.x), c.parts)[1]

    def kept(got, want, S, terms):
        """got and want where neither is a hit"""
        w = want.double().cpu()
        tol = 2 * (terms + 4) * sum_unit(t) * S
        near(got, w, tol + 2 * u * (w.abs() + tol) + tiny(t), "kept")

    c.x[1, 100] = value
    y = dg.spmm(c.plan, c.vals[0], c.x)
    hit = torch.zeros(M, n, dtype=torch.bool, device="cuda")
    hit[1, [100 - d for d in off]] = True
    assert bool((~y[hit].isfinite()).all())
    kept(y[~hit], y0[~hit], sy[~hit.cpu()], K)
    if not math.isnan(value):      # one infinite term: the sum is that infinity
        sign = torch.stack([c.vals[0, k, 100 - d] for k, d in enumerate(off)]).sign() * value
        assert torch.equal(torch.stack([y[1, 100 - d] for d in off]), sign)
    _, dv, _ = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)
    hit = torch.zeros(len(off), 224, dtype=torch.bool, device="cuda")
    for k, d in enumerate(off):
        hit[k, 100 - d] = True
    assert bool((~dv[hit].isfinite()).all())
    kept(dv[~hit], dv0[~hit], sv[0][~hit.cpu()], M)
    c.x.copy_(x0)
    c.dy[2, 90] = value
    dx, dv, _ = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)
    hit = torch.zeros(M, n, dtype=torch.bool, device="cuda")
    hit[2, [90 + d for d in off]] = True
    assert bool((~dx[hit].isfinite()).all())
    kept(dx[~hit], dx0[~hit], sx[~hit.cpu()], K)
    assert bool((~dv[:, 90].isfinite()).all())
    keep = torch.ones(224, dtype=torch.bool, device="cuda")
    keep[90] = False
    kept(dv[:, keep], dv0[:, keep], sv[0][:, keep.cpu()], M)


@pytest.mark.parametrize("seg", [[0, 90, 20, 200], [-5, 50, 100, 10 ** 12], [200, 0, 200, 0],
                                 [0, 200, 0, 200]])
def test_bad_segments_stay_inside(seg, t):
    """A seg that decreases or leaves the block gives some result, without a
    read or write outside the buffers."""
    c = Case(t, 200, 136, 136, band(6), seed=9, seg=[0, 50, 100, 200])
    s = torch.tensor(seg, dtype=torch.int64).cuda()
    guard = torch.full((3, 200, 136), 3.0, dtype=t, device="cuda")
    dg.spmm(c.plan, c.vals, c.x, seg=s, out=guard[1])
    dg.spmm_backward(c.plan, c.vals, c.x, c.dy, seg=s, dx=guard[1])
    torch.cuda.synchronize()
    assert bool((guard[0] == 3).all() and (guard[2] == 3).all())


@pytest.mark.parametrize("M", [1, 600])
def test_same_bits_every_time(M, t):
    c = Case(t, M, 264, 264, band(30), seed=10)
    a = dg.spmm(c.plan, c.vals[0], c.x, act="gelu")
    ga = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="gelu", bias_grad=True)
    for _ in range(3):
        assert torch.equal(a, dg.spmm(c.plan, c.vals[0], c.x, act="gelu"))
        gb = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="gelu", bias_grad=True)
        assert all(torch.equal(p, q) for p, q in zip(ga, gb))


def test_result_over_the_residual():
    c = Case(torch.bfloat16, 140, 136, 136, band(6), seed=11)
    want = dg.spmm(c.plan, c.vals[0], c.x, act="silu", residual=c.res)
    r = c.res.clone()
    dg.spmm(c.plan, c.vals[0], c.x, act="silu", residual=r, out=r)
    assert torch.equal(r, want)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_streams_and_graphs(t):
    """Two streams at once with one plan; then forward and backward captured
    into a graph and replayed on new inputs, beside a second graph of the same
    plan with buffers of its own."""
    a, b = (Case(t, 300, 200, 200, band(12), seed=s) for s in (12, 13))
    want = []
    for c in (a, b):
        y, z = dg.spmm(c.plan, c.vals[0], c.x, act="gelu", save_z=True)
        want.append((y, *dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=z, act="gelu",
                                          bias_grad=True)))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got = []
        for c, s in zip((a, b), side):
            y, z = dg.spmm(a.plan, c.vals[0], c.x, act="gelu", save_z=True, stream=s)
            got.append((y, *dg.spmm_backward(a.plan, c.vals[0], c.x, c.dy, z=z, act="gelu",
                                             bias_grad=True, stream=s)))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, z = dg.spmm(a.plan, c.vals[0], c.x, act="gelu", save_z=True)
            outs.append((y, *dg.spmm_backward(a.plan, c.vals[0], c.x, c.dy, z=z, act="gelu",
                                              bias_grad=True)))
        graphs.append(g)
    x = a.x.clone()
    a.x.copy_(b.x)
    for s, g in zip(side, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[1], want[1]))
    a.x.copy_(x)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[0], want[0]))


class Layer(torch.autograd.Function):
    """How a program trains such a layer."""

    @staticmethod
    def forward(ctx, plan, act, seg, x, vals, bias, residual):
        y, z = dg.spmm(plan, vals, x, bias=bias, act=act, residual=residual, seg=seg, save_z=True)
        ctx.plan, ctx.act = plan, act
        ctx.save_for_backward(x, vals, z, *([seg] if seg is not None else []))
        return y

    @staticmethod
    def backward(ctx, dy):
        x, vals, z, *seg = ctx.saved_tensors
        dx, dvals, dbias = dg.spmm_backward(ctx.plan, vals, x, dy.contiguous(), z=z, act=ctx.act,
                                            seg=seg[0] if seg else None, bias_grad=True)
        return None, None, None, dx, dvals, dbias, dy


@pytest.mark.parametrize("grouped", [False, True])
def test_layers_trained_together(grouped):
    """Two layers with a residual, as a model runs them: the loss's derivative
    along random directions against differences of the same loss in 64 bits.
    The step h = 1e-5 leaves about h^2 and 1e-16 / h of the loss's size, and the
    fp32 gradients K * 2^-24 of theirs: 1e-4 of the gradients' norm covers all."""
    M, n, m = 40, 96, 80
    seg = [0, 11, 11, 40] if grouped else None
    up = Case(torch.float32, M, n, m, band(5), seed=14, seg=seg)
    down = Case(torch.float32, M, m, n, band(7), seed=15, seg=seg)
    sq = (lambda a: a) if grouped else (lambda a: a[0])
    theta = [up.x.clone(), sq(up.vals).clone(), sq(up.bias).clone(), sq(down.vals).clone(),
             sq(down.bias).clone()]
    theta = [p.requires_grad_() for p in theta]
    x, v1, b1, v2, b2 = theta
    target = torch.randn(M, m, generator=torch.Generator().manual_seed(3)).cuda()
    h = Layer.apply(up.plan, "gelu", up.dseg, x, v1, b1, torch.zeros(M, n, device="cuda"))
    y = Layer.apply(down.plan, "none", down.dseg, h, v2, b2, x)
    ((y - target) ** 2).sum().backward()

    def loss(p):
        x, v1, b1, v2, b2 = p
        f = lambda a, dims: a if a.dim() == dims else a[None]
        z, _ = product64(up.off, n, m, f(v1, 3), x, up.parts, f(b1, 2))
        z2, _ = product64(down.off, m, n, f(v2, 3), act64(z, "gelu"), down.parts, f(b2, 2))
        return float(((z2 + x - target.double().cpu()) ** 2).sum())

    base = [p.detach().double().cpu() for p in theta]
    g = torch.Generator().manual_seed(16)
    for j in range(len(base)):
        d = torch.randn(base[j].shape, generator=g, dtype=torch.float64)
        d /= d.norm()
        step = 1e-5
        lo = loss([b - step * d if i == j else b for i, b in enumerate(base)])
        hi = loss([b + step * d if i == j else b for i, b in enumerate(base)])
        grad = theta[j].grad.double().cpu()
        assert abs((hi - lo) / (2 * step) - float((grad * d).sum())) <= 1e-4 * float(grad.norm())


def test_matches_spmv():
    """One fp32 vector: the same operator through spmv."""
    n, off = 5000, [-70, -1, 0, 1, 70]
    A = dg.DiaRows.synth(n, n, np.array(off, np.int32), seed=1)
    x = dg.synth_vector(n, seed=2)
    y = dg.spmm(dg.SpmmPlan(n, n, off), A.vals, x[None])
    ref = dg.spmv(A, x)[:n]
    S = product64(off, n, n, A.vals.double().cpu()[None], x.double().cpu()[None],
                  [(0, 0, 1)])[1][0]
    near(y[0], ref.double().cpu(), 2 * 9 * 2.0 ** -24 * S, "spmv")


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31: views far apart in one buffer."""
    n, M, off = 64, 3, band(2)
    ld = (1 << 30) + 8
    buf = torch.empty(2 * ld + n, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((M, n), (ld, 1))
    g = torch.Generator(device="cuda").manual_seed(5)
    x.copy_(torch.randn(M, n, generator=g, device="cuda"))
    v = torch.randn(5, 64, generator=g, device="cuda").bfloat16()
    plan = dg.SpmmPlan(n, n, off)
    assert torch.equal(dg.spmm(plan, v, x), dg.spmm(plan, v, x.contiguous()))
    a = dg.spmm_backward(plan, v, x, x, bias_grad=True)
    b = dg.spmm_backward(plan, v, x.contiguous(), x.contiguous(), bias_grad=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals_on_the_device():
    c = Case(torch.bfloat16, 20, 64, 64, band(2), seed=17)
    plan, v, x = c.plan, c.vals[0], c.x

    def refused(code, f, *a, **k):
        with pytest.raises(dg.DiaError) as e:
            f(*a, **k)
        assert e.value.code == code

    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, v, x.cpu())
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, v.cpu(), x)
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, torch.zeros(5, 48, dtype=x.dtype, device="cuda"), x)
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, torch.zeros(5, 32, dtype=x.dtype, device="cuda"), x)
    odd = torch.zeros(5 * 64 + 1, dtype=x.dtype, device="cuda")[1:].view(5, 64)
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, odd, x)
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, v, x[:1].expand(20, 64))
    refused(dg.DIA_ERR_INVALID, dg.spmm, plan, v, x, out=torch.zeros(20, 63, dtype=x.dtype,
                                                                      device="cuda"))
    ws = dg.spmm_backward_workspace(plan, v, x, c.dy, "silu")
    assert ws > 0
    work = torch.empty(ws - 1, dtype=torch.uint8, device="cuda")
    refused(dg.DIA_ERR_CAPACITY, dg.spmm_backward, plan, v, x, c.dy, z=c.zin, act="silu",
            work=work)
    work = torch.empty(ws + 1, dtype=torch.uint8, device="cuda")[1:]
    refused(dg.DIA_ERR_INVALID, dg.spmm_backward, plan, v, x, c.dy, z=c.zin, act="silu",
            work=work)


def test_a_wait_that_runs_out():
    """Failure detection without a fault: with a limit of 1 ms and one copy
    withheld, the tensor-core product and gradient stop, report DIA_TC_TIMEOUT
    and leave the GPU usable: the next calls are right."""
    L = dg.lib()
    c = Case(torch.bfloat16, 600, 264, 264, band(6), seed=23)
    dg.check(L.dia_test_spmm_form(2))
    try:
        dg.device_status(clear=True)
        for f in (lambda: dg.spmm(c.plan, c.vals[0], c.x, act="silu"),
                  lambda: dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="silu"),
                  lambda: dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)):
            dg.check(L.dia_test_tc_wait(1_000_000, 1))
            try:
                f()
                torch.cuda.synchronize()
            finally:
                dg.check(L.dia_test_tc_wait(0, 0))
            assert dg.device_status(clear=True) & dg.DIA_TC_TIMEOUT
            c.product(act="silu", bias=True, res=True)
            c.gradient(act="silu")
            assert dg.device_status() == 0
    finally:
        dg.check(L.dia_test_spmm_form(0))


@pytest.mark.parametrize("n,m,off", [(0, 8, [0, 1]), (8, 0, [0, -1]), (0, 0, []), (0, 0, [0])])
@pytest.mark.parametrize("M", [0, 3, 200])
def test_empty_sides(M, n, m, off, t):
    c = Case(t, M, n, m, off, seed=24)
    c.product(act="relu", bias=True, res=True, z=True)
    c.gradient(act="relu")


@pytest.mark.parametrize("M", [4, 300])
def test_single_gradients(M, t):
    """The C entry's outputs may each be left out: the others stay the same."""
    c = Case(t, M, 136, 144, band(5), seed=25)
    L, code = dg.lib(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[t]
    dx, dv, db = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="silu",
                                  bias_grad=True)
    st = c.vals.shape[-1]
    ws = L.dia_spmm_backward_workspace(c.plan._h, code, M, 1, 144, st, 136, 2)
    work = torch.empty(ws, dtype=torch.uint8, device="cuda")
    for want in (dx, dv, db):
        out = torch.full_like(want, 9.0)
        p = [o.data_ptr() if w is want else None for w, o in ((dx, out), (dv, out), (db, out))]
        for x in (c.x.data_ptr(),) if want is dv else (c.x.data_ptr(), None):
            out.fill_(9.0)
            dg.check(L.dia_spmm_backward(c.plan._h, code, M, 1, None, x, 144,
                                         c.vals.data_ptr() if want is dx else None, st,
                                         c.dy.data_ptr(), 136, 2, c.zin.data_ptr(), 136, p[0], 144,
                                         p[1], p[2], work.data_ptr(), ws,
                                         torch.cuda.current_stream().cuda_stream))
            u = unit(t)
            # dbias alone is summed on the CUDA cores, in another order
            assert bool(((out.double() - want.double()).abs()
                         <= 2 * u * want.double().abs() + (M + 4) * sum_unit(t) * 200).all())
            if want is not db:
                assert torch.equal(out, want)


def test_refused_gradient_buffers():
    c = Case(torch.bfloat16, 20, 64, 64, band(2), seed=17)
    odd = torch.zeros(5 * 64 + 1, dtype=c.x.dtype, device="cuda")[1:].view(5, 64)
    with pytest.raises(dg.DiaError) as e:
        dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, dvals=odd)
    assert e.value.code == dg.DIA_ERR_INVALID


def test_results_on_another_stream_have_their_own_memory():
    """What a call on a given stream allocates is not memory that the current
    stream still writes."""
    c = Case(torch.bfloat16, 256, 512, 512, band(3), seed=41)
    want = dg.spmm(c.plan, c.vals[0], c.x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        old = [torch.empty_like(want) for _ in range(4)]
        torch.cuda._sleep(20_000_000)
        for o in old:
            o.fill_(float("nan"))
        del old, o
        got = dg.spmm(c.plan, c.vals[0], c.x, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("M,tensor", [(8, False), (1024, True)])
def test_wide_operators(M, tensor):
    """Few rows under an operator of many boxes stay on the CUDA cores, which
    want no workspace; either form's sums are the same to rounding."""
    n, side = 32768, 32
    off = [i + side * j + side * side * k
           for i in (-1, 0, 1) for j in (-1, 0, 1) for k in (-1, 0, 1)]
    c = Case(torch.bfloat16, M, n, n, off, seed=43)
    assert (dg.spmm_workspace(c.plan, c.vals[0], c.x) > 0) == tensor
    got = dg.spmm(c.plan, c.vals[0], c.x).double()
    want = torch.zeros(M, n, dtype=torch.float64, device="cuda")
    size = torch.zeros(M, n, dtype=torch.float64, device="cuda")
    x, v = c.x.double(), c.vals[0].double()
    for k, d in enumerate(off):
        lo, hi = max(0, -d), min(n, n - d)
        p = v[k, lo:hi] * x[:, lo + d:hi + d]
        want[:, lo:hi] += p
        size[:, lo:hi] += p.abs()
    # the result's rounding to bf16, and 27 fp32 additions, each off by at most
    # a step (the tensor cores may cut off instead of rounding)
    u = unit(c.x.dtype)
    limit = u * want.abs() + (1 + u) * 27 * 2.0 ** -23 * size
    assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("act", ACTS[1:])
def test_lowest_and_largest_values(act, t):
    """Pre-activations of the type's lowest and largest value, as masks leave
    them: the activation is 0 or z, its derivative 0 or 1, exactly."""
    M, n = 40, 136
    c = Case(t, M, n, n, [0], seed=47)
    top = torch.finfo(t).max
    z = c.block(torch.zeros(M, n))
    z[:, ::2], z[:, 1::2] = -top, top
    c.vals[0, 0].fill_(0.0)
    c.vals[0, 0, :n] = 1.0
    y, zz = dg.spmm(c.plan, c.vals[0], z, act=act, save_z=True)
    assert torch.equal(zz, z)
    assert bool((y[:, ::2] == 0).all()) and bool((y[:, 1::2] == top).all())
    dx, dv, _ = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=z, act=act)
    dz = c.dy.clone()
    dz[:, ::2] = 0
    assert torch.equal(dx, dz)
    assert bool(dv.isfinite().all())


@pytest.mark.parametrize("M", [3, 300])
def test_first_use_of_a_plan_on_another_stream(M, t):
    """A new plan's tables are on the device when it is returned: its first
    calls are on a stream that does not wait for the default one.  The offsets
    are many, so that the tables are more than one staging buffer."""
    n, off = 2000, list(range(-1900, 1900, 2))
    c = Case(t, M, n, n, off, seed=51)
    want = dg.spmm(c.plan, c.vals[0], c.x)
    grads = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        plan = dg.SpmmPlan(n, n, np.array(off, np.int32))
        got = dg.spmm(plan, c.vals[0], c.x, stream=side)
        back = dg.spmm_backward(plan, c.vals[0], c.x, c.dy, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(p, q) for p, q in zip(back[:2], grads[:2]))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_plans_come_and_go_during_capture(t):
    """A plan that is dropped, and one that is made, while a graph is captured
    leave the capture alone."""
    c = Case(t, 140, 136, 136, band(6), seed=52)
    want = dg.spmm(c.plan, c.vals[0], c.x)
    old = dg.SpmmPlan(64, 64, [0, 1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        del old
        plan = dg.SpmmPlan(136, 136, c.off)
        got = dg.spmm(plan, c.vals[0], c.x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("act", ACTS[2:])
def test_activations_to_their_last_bits(act, M, t):
    """Values and derivatives on [-6, 6] as an identity operator gives them,
    bounded by the result itself, so that a negative z's small one counts too.

    With a = 2^-23 (fp32) an argument z sqrt(1/2) is off by a of itself, which
    erfc, whose logarithm's slope is below 2 x + 1 / x, makes (z^2 + 2) a; with
    the function's own 4 a and three multiplications (8 + z^2) a.  Likewise
    exp(-2 u) is off by 6 |u| a for u of the tanh form (six roundings), the
    logistic function by (8 + 6 |u|) a.  16-bit types: 2^-16, the bound that the
    polynomial of the normal distribution is fitted to, and for the logistic
    functions the fp32 bounds once more for the hardware's functions.  A derivative's
    terms carry these bounds each, and 1 - s is off by a."""
    n = 700
    c = Case(t, M, n, n, [0], seed=61)
    c.vals[0, 0].fill_(0.0)
    c.vals[0, 0, :n] = 1.0
    z = torch.linspace(-6, 6, M * n, dtype=torch.float64).view(M, n)
    c.x, c.zin = c.block(z), c.block(z)
    c.dy = c.block(torch.ones(M, n))
    z, u, a = c.v(c.zin), unit(t), 2.0 ** -23
    half = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    if act == "gelu":
        e = 2.0 ** -16 + torch.zeros_like(z) if t != torch.float32 else (8 + z * z) * a
    else:
        e = (8 + 6 * (half if act == "gelu_tanh" else z / 2).abs()) * a
        e = e if t == torch.float32 else 2 * e
    want = act64(z, act)
    tol = (e + u * (1 + e)) * want.abs() + tiny(t)
    near(dg.spmm(c.plan, c.vals[0], c.x, act=act), want, tol, "value")

    want = dact64(z, act)
    if act == "gelu":
        slope = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        slope = slope + z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        err = e * slope
    else:
        s = torch.sigmoid(2 * half if act == "gelu_tanh" else z)
        grow = torch.ones_like(z)
        if act == "gelu_tanh":
            grow = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
        # s + z grow s (1 - s): s twice, grow's three roundings, 1 - s
        err = e * s + z.abs() * grow * s * ((1 - s) * (2 * e + 3 * a) + 2 * a)
    dx = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act=act)[0]
    near(dx, want, err + u * (want.abs() + err) + tiny(t), "derivative")


def alike(got, want, what):
    """Both NaN, or the same infinity, at every place."""
    got, want = got.double().cpu(), want.double().cpu()
    ok = (got == want) | (got.isnan() & want.isnan())
    assert bool(ok.all()), (what, int((~ok).sum()), got[~ok][:4].tolist(), want[~ok][:4].tolist())


def best_ms(f, n=4):
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    f()
    best = math.inf
    for _ in range(n):
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def time_against_cores(f):
    """Time of f in the tensor-core form over that in the CUDA-core form."""
    L = dg.lib()
    try:
        dg.check(L.dia_test_spmm_form(1))
        cores = best_ms(f)
        dg.check(L.dia_test_spmm_form(2))
        return best_ms(f) / cores
    finally:
        dg.check(L.dia_test_spmm_form(0))
        assert dg.device_status() == 0


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_gradient_of_a_block_that_overflowed(value, t):
    """dy as a step of too large a loss scale leaves it: every entry of the
    diagonals' gradient is what its own terms give."""
    M, n, off = 300, 264, band(20)
    c = Case(t, M, n, n, off, seed=62)
    c.dy.fill_(value)
    dv = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)[1]
    want = gradient64(off, n, n, c.v(c.vals), c.v(c.x), c.v(c.dy), c.parts)[1][0]
    alike(dv, want, "dvals")


def test_time_of_a_gradient_that_overflowed():
    """It costs no walk over the rows for each entry (with one, five times the
    CUDA-core form's time, which does not look at its values)."""
    M, n, off = 4096, 2048, band(64)
    c = Case(torch.float16, M, n, n, off, seed=63)
    c.dy.fill_(float("inf"))
    dv = torch.zeros_like(c.vals[0])
    L, st = dg.lib(), c.vals.shape[-1]
    work = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")

    def f():
        dg.check(L.dia_spmm_backward(c.plan._h, 1, M, 1, None, c.x.data_ptr(), n, None, st,
                                     c.dy.data_ptr(), n, 0, None, n, None, n, dv.data_ptr(), None,
                                     work.data_ptr(), work.numel(),
                                     torch.cuda.current_stream().cuda_stream))

    assert time_against_cores(f) < 2


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_product_of_a_block_that_overflowed(value, t):
    """No input is finite: sums, z and results are what their own terms give,
    gradients of the inputs likewise."""
    M, n, off = 300, 264, [-250, -64, -1, 0, 1, 2, 3, 200]
    c = Case(t, M, n, n, off, seed=64)
    c.x.fill_(value)
    c.dy.fill_(value)
    v, x = c.v(c.vals), c.v(c.x)
    y, z = dg.spmm(c.plan, c.vals[0], c.x, bias=c.bias[0], act="relu", residual=c.res, save_z=True)
    want = product64(off, n, n, v, x, c.parts, c.v(c.bias))[0]
    alike(z, want, "z")
    finite = act64(want, "relu").isfinite()
    alike(torch.where(finite.cuda(), 0, y), act64(want, "relu") + torch.where(finite, 0, c.v(c.res))
          - torch.where(finite, act64(want, "relu"), 0), "y")
    dx = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)[0]
    alike(dx, gradient64(off, n, n, v, x, c.v(c.dy), c.parts)[0], "dx")


def test_time_of_a_product_that_overflowed():
    """Sums over their own terms are shared out over the lanes (one lane a row
    took 55 times the CUDA-core form's time and twice that with z kept, this nine
    times)."""
    c = Case(torch.float16, 4096, 2048, 2048, band(64), seed=65)
    c.x.fill_(float("inf"))
    y, z = torch.empty_like(c.x), torch.empty_like(c.x)
    assert time_against_cores(lambda: dg.spmm(c.plan, c.vals[0], c.x, out=y)) < 25
    assert time_against_cores(lambda: dg.spmm(c.plan, c.vals[0], c.x, out=y, z=z)) < 25


def test_waits_outlast_sums_over_their_own_terms():
    """A wait's limit does not run while the sums that it waits for are being
    computed again: 2 ms, a block without a finite value, six tiles a CTA of
    527 diagonals."""
    M, n, off = 40000, 264, band(263)
    c = Case(torch.bfloat16, M, n, n, off, seed=66)
    c.x.fill_(float("inf"))
    L = dg.lib()
    want = product64(off, n, n, c.v(c.vals), c.v(c.x[:1]), [(0, 0, 1)])[0].expand(M, n)
    dg.check(L.dia_test_spmm_form(2))
    try:
        dg.spmm(c.plan, c.vals[0], c.x)         # the kernel is loaded
        torch.cuda.synchronize()
        dg.device_status(clear=True)
        dg.check(L.dia_test_tc_wait(2_000_000, 0))
        y = dg.spmm(c.plan, c.vals[0], c.x)
        torch.cuda.synchronize()
        assert dg.device_status(clear=True) == 0
    finally:
        dg.check(L.dia_test_tc_wait(0, 0))
        dg.check(L.dia_test_spmm_form(0))
    alike(y, want, "y")


@pytest.mark.parametrize("side,M", [(128, 256), (256, 512), (256, 32), (64, 2048), (96, 8192)])
def test_workspace_has_a_limit(side, M):
    """An operator packed for the tensor cores takes no more room than the block
    and its result, or 2 GB: scattered diagonals of large operators would take
    fifty times their own.  Sizes only; nothing of them is allocated."""
    n = side ** 3
    plan = dg.SpmmPlan(n, n, [i + side * j + side * side * k for i in (-1, 0, 1)
                              for j in (-1, 0, 1) for k in (-1, 0, 1)])
    L, block = dg.lib(), 2 * 2 * M * n
    most = max(block, 1 << 31)
    assert 0 <= L.dia_spmm_workspace(plan._h, 2, M, 1, n) <= most
    # and dz in 32 bits; features enough for every SM leave the rows in one part
    assert 0 <= L.dia_spmm_backward_workspace(plan._h, 2, M, 1, n, n, n, 2) <= most + block


# Sizes at which a kernel takes its other path: more diagonals than a CTA keeps
# offsets of (512), more boxes than it keeps places of (64).
LARGE = {
    "diagonals, 1 row": (1, 700, 700, list(range(-550, 550))),
    "diagonals, 2 rows": (2, 700, 700, list(range(-550, 550))),
    "diagonals": (20, 700, 700, list(range(-550, 550))),
    "diagonals, tiles": (300, 700, 700, list(range(-550, 550))),
    "boxes": (200, 9200, 9200, list(range(-4550, 4550, 130))),
}


@pytest.mark.parametrize("shape", LARGE)
def test_many_diagonals_and_boxes(shape, t):
    c = Case(t, *LARGE[shape], seed=67)
    c.product(act="silu", bias=True, res=True, z=True)
    c.gradient(act="silu")


def test_many_diagonals_of_experts(t):
    c = Case(t, 150, 300, 300, list(range(-290, 290)), seed=68, seg=[0, 1, 40, 40, 149])
    c.product(act="relu", bias=True)
    c.gradient(act="relu")


# The many-row CUDA-core kernel, which begins at 196608 results: rows and bases
# that its vector accesses do not take, and each of its feature tiles (256, 512
# and 1024: the widest that fits and leaves every SM a CTA).
@pytest.mark.parametrize("off", [band(4), [-300, -40, 0, 1, 77, 400]], ids=["band", "scattered"])
@pytest.mark.parametrize("M,n,ld,shift", [(300, 701, 1, 0), (300, 700, None, 1), (300, 702, 3, 2),
                                          (600, 700, 4, 0), (8, 100000, None, 0),
                                          (1200, 2100, None, 0), (1201, 2101, 1, 1)])
def test_many_rows_on_the_cores(M, n, ld, shift, off, t):
    c = Case(t, M, n, n, off, seed=69, ld=ld, shift=shift)
    c.product(act="gelu", bias=True, res=True, z=True)
    c.gradient(act="gelu")


def test_offsets_past_32_bits_on_the_tensor_cores():
    """As above, where TMA and the tensor cores' epilogue step from row to row."""
    n, M, off = 64, 3, band(2)
    ld = (1 << 30) + 8
    buf = torch.empty(2 * ld + n, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((M, n), (ld, 1))
    g = torch.Generator(device="cuda").manual_seed(5)
    x.copy_(torch.randn(M, n, generator=g, device="cuda"))
    v = torch.randn(5, 64, generator=g, device="cuda").bfloat16()
    plan, near = dg.SpmmPlan(n, n, off), x.contiguous()
    dg.check(dg.lib().dia_test_spmm_form(2))
    try:
        want = dg.spmm(plan, v, near, act="silu", residual=near, save_z=True)
        got = dg.spmm(plan, v, x, act="silu", residual=x, save_z=True)
        a = dg.spmm_backward(plan, v, x, x, z=x, act="silu", bias_grad=True)
        b = dg.spmm_backward(plan, v, near, near, z=near, act="silu", bias_grad=True)
        dg.spmm(plan, v, near, out=x)
        assert torch.equal(x, dg.spmm(plan, v, near))
        assert dg.device_status() == 0
    finally:
        dg.check(dg.lib().dia_test_spmm_form(0))
    assert all(torch.equal(p, q) for p, q in zip((*got, *a), (*want, *b)))


@pytest.mark.parametrize("M", [1, 300])
def test_an_error_is_reported_once(M, t):
    """A call of the library that failed (here one that allocates, during a
    capture) has reported its error; the next call, which is good, does not
    report it again."""
    c = Case(t, M, 700, 700, band(3), seed=70)
    A = dg.DiaRows.synth(64, 64, np.array([0, 1], np.int32), seed=1)
    calls = (lambda: (dg.spmm(c.plan, c.vals[0], c.x),),
             lambda: dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy)[:2])
    for f in calls:
        want = f()
        torch.cuda.synchronize()
        with pytest.raises(Exception):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                dg.SpmspmPlan(A, A)
        assert all(torch.equal(p, q) for p, q in zip(f(), want))


WIDE = [-250, -201, -130, -64, -3, 0, 55, 120, 199, 260]


@pytest.mark.parametrize("M,off,seg,shift", [
    (3, band(2), None, 0), (300, band(2), None, 0), (300, WIDE, None, 0),
    (300, band(2), None, 1), (300, WIDE, None, 1), (1500, band(2), None, 0),
    (300, band(2), [3, 70, 70, 71, 290], 0), (300, WIDE, [0, 1, 200, 300], 0)])
def test_gradients_keep_dz_in_32_bits(M, off, seg, shift, t):
    """The gradients' error is the sums' and one rounding: dz = dy silu'(z) is not
    rounded to the block's type before them.  silu' is off by less than 2^-16 (1 +
    |z|) (the logistic function by 2^-19 of itself), a dz of two halves by 2^-18,
    and where fp16's second half underflows by half a step of 2^-24.  Operators of
    a few boxes and of many, parts, experts, blocks that TMA does not take."""
    n = 264
    c = Case(t, M, n, n, off, seed=71, seg=seg, shift=shift)
    sq = (lambda a: a) if seg is not None else (lambda a: a[0])
    dx, dv = c.block(torch.full((M, n), 3.0)), torch.full_like(c.vals, 9.0)
    db = torch.full_like(c.bias, 9.0)
    dg.spmm_backward(c.plan, c.pv(), c.x, c.dy, z=c.zin, act="silu", seg=c.dseg, dx=dx,
                     dvals=sq(dv), dbias=sq(db))
    dy, x, vals, z, u = c.v(c.dy), c.v(c.x), c.v(c.vals), c.v(c.zin), unit(t)
    dz = dy * dact64(z, "silu")
    ed = 2.0 ** -16 * (1 + z.abs()) * dy.abs() + 2.0 ** -18 * dz.abs()
    ed = ed + (2.0 ** -25 if t == torch.float16 else 0)
    want = gradient64(off, n, n, vals, x, dz, c.parts)
    S = gradient64(off, n, n, vals.abs(), x.abs(), dz.abs(), c.parts)
    T = gradient64(off, n, n, vals.abs(), x.abs(), ed, c.parts)
    on, rows = c.rows(), max(b - a for _, a, b in c.parts)
    for got, w, s, e, terms, what in ((dx[on], want[0][on], S[0][on], T[0][on], len(off), "dx"),
                                      (dv, want[1], S[1], T[1], rows, "dvals"),
                                      (db, want[2], S[2], T[2], rows, "dbias")):
        e = e + (2 * terms + 4) * sum_unit(t) * (s + e)     # two halves: twice the terms
        near(got, w, e + u * (w.abs() + e) + tiny(t), what)
    assert bool((dx[~on].cpu() == 3).all())


@pytest.mark.parametrize("n,M,off,act", [
    (65536, 512, [-500, -377, -200, -64, 0, 13, 90, 255, 500], "silu"),
    (65536, 512, [-500, -377, -200, -64, 0, 13, 90, 255, 500], "none"),
    (65536, 512, band(16), "relu"), (4096, 4096, band(64), "gelu"), (2048, 4096, band(64), "relu")])
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
def test_gradient_stages_are_read_when_they_are_full(n, M, off, act, t):
    """Thousands of CTAs whose warps make or sum dz from a ring of three stages: no
    warp takes an earlier round of a stage for the one that it waits for.  The
    same bits every time and no wait that runs out; for dz = dy or 0 the CUDA-core
    form's bits, since sums of small whole numbers are exact in any order."""
    g = torch.Generator(device="cuda").manual_seed(72)
    plan, K = dg.SpmmPlan(n, n, off), len(off)
    r = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").to(t)
    v, x, dy, z = r(K, n), r(M, n), r(M, n), r(M, n)
    L = dg.lib()

    def run():
        return dg.spmm_backward(plan, v, x, dy, z=z, act=act, bias_grad=True)

    try:
        dg.check(L.dia_test_spmm_form(1))
        cores = run()
        dg.check(L.dia_test_spmm_form(2))
        first = run()
        for _ in range(20):
            assert all(torch.equal(p, q) for p, q in zip(run(), first))
        assert dg.device_status() == 0
    finally:
        dg.check(L.dia_test_spmm_form(0))
    if act in ("none", "relu"):
        assert all(torch.equal(p, q) for p, q in zip(first, cores))


@pytest.mark.parametrize("off", [band(2), WIDE], ids=["made in the gradient", "made before"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), "large"])
def test_dz_past_the_type(value, off, t):
    """dz that is not finite reaches the results that its terms reach; finite dz
    past the largest number of fp16 (dy times a derivative up to 1.1) stays
    finite, in either form."""
    M, n = 300, 264
    c = Case(t, M, n, n, off, seed=73)
    c.zin[:, ::3] = 2.4
    if value == "large":
        top = torch.finfo(t).max if t == torch.float16 else 65504.0
        c.dy[:, ::3] = top
        c.vals.mul_(2.0 ** -10)
        c.x.mul_(2.0 ** -14)
    else:
        c.dy[::7, ::5] = value
    dx, dv, db = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="silu", bias_grad=True)
    dz = c.v(c.dy) * dact64(c.v(c.zin), "silu")
    want = gradient64(off, n, n, c.v(c.vals), c.v(c.x), dz, c.parts)
    for got, w, what in ((dx, want[0], "dx"), (dv, want[1][0], "dvals"), (db, want[2][0], "dbias")):
        got = got.double().cpu()
        if value == "large":
            # sums of dbias pass the type; the others are finite and near
            fits = w.abs() < 0.9 * torch.finfo(t).max
            assert what == "dbias" or bool(fits.all())
            err = (got - w)[fits].norm() / w[fits].norm()
            assert bool(got[fits].isfinite().all()) and float(err) <= 2 * unit(t) + 2.0 ** -14
        else:
            bad = ~w.isfinite()
            alike(torch.where(bad, got, 0), torch.where(bad, w, 0), what)
            assert bool(got[~bad].isfinite().all())


@pytest.mark.parametrize("M", [4, 300])
@pytest.mark.parametrize("shift", [0, 1])
def test_pairs_of_gradients(M, shift, t):
    """Two of the C entry's outputs without the third: the same as all three,
    but for the order of the sums where another form takes the rest."""
    n, m = 136, 144
    c = Case(t, M, n, m, band(5), seed=74, shift=shift)
    L, code = dg.lib(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[t]
    want = dg.spmm_backward(c.plan, c.vals[0], c.x, c.dy, z=c.zin, act="silu", bias_grad=True)
    st = c.vals.shape[-1]
    ws = L.dia_spmm_backward_workspace(c.plan._h, code, M, 1, m, st, n, 2)
    work = torch.empty(ws, dtype=torch.uint8, device="cuda")
    for left in range(3):
        out = [torch.full_like(w, 9.0) for w in want]
        p = [None if k == left else o.data_ptr() for k, o in enumerate(out)]
        dg.check(L.dia_spmm_backward(c.plan._h, code, M, 1, None, c.x.data_ptr(), m,
                                     c.vals.data_ptr(), st, c.dy.data_ptr(), n, 2,
                                     c.zin.data_ptr(), n, p[0], m, p[1], p[2], work.data_ptr(), ws,
                                     torch.cuda.current_stream().cuda_stream))
        for k, (o, w) in enumerate(zip(out, want)):
            if k == left:
                assert bool((o == 9).all())
                continue
            S = (11, M, M)[k] * (float(c.vals.abs().max()), float(c.x.abs().max()), 1.0)[k]
            S *= 1.2 * float(c.dy.abs().max())
            lim = 2 * unit(t) * w.double().abs() + (M + 15) * sum_unit(t) * S + 2.0 ** -16 * S
            assert bool(((o.double() - w.double()).abs() <= lim + tiny(t)).all())
