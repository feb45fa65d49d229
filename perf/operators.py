"""Measured operators: a diagonal (DIA) operator times a block of vectors.

A block holds one vector (token) per row.  The operator's diagonals are stored
as ``vals[k, i] = A[i, i + d_k]``, padded to a stride that is a multiple of 32.

* product:   z = x A^T + bias,  y = act(z) + residual, z kept for training;
* gradient:  dz = dy act'(z),  dx = dz A,  dvals[k, i] = sum_t dz[t, i] x[t, i + d_k],
  dbias = sum_t dz;
* grouped ("experts" > 0): the rows are sorted by expert, ragged and some empty,
  and every expert has diagonal values of its own.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def _case(name, op, tokens, rows, cols, pattern, width, dtype, act="none", bias=False,
          residual=False, save=False, experts=0):
    return dict(name=name, op=op, tokens=tokens, rows=rows, cols=cols, pattern=pattern,
                width=width, dtype=dtype, act=act, bias=bias, residual=residual, save=save,
                experts=experts)


def listed():
    return [
        # one new token through a square band layer (129 diagonals, the dense-band width)
        _case("decode_band_bf16", "product", 1, 4096, 4096, "band", 64, "bf16", "silu",
              bias=True, residual=True),
        # a small block of vectors under an operator of 32 scattered diagonals
        _case("block8_scatter_fp32", "product", 8, 4096, 4096, "scatter", 32, "fp32"),
        # training forward of a band layer over a batch of sequences
        _case("prompt_band_bf16", "product", 4096, 4096, 4096, "band", 64, "bf16", "gelu",
              bias=True, residual=True, save=True),
        # a prompt of odd length through scattered diagonals
        _case("prompt_scatter_fp16", "product", 2047, 4096, 4096, "scatter", 32, "fp16", "relu",
              bias=True),
        # a block of 64 states under a 27-point stencil on a 64^3 grid
        _case("block64_stencil_fp32", "product", 64, 262144, 262144, "stencil", 64, "fp32"),
        # down-projection: a band around each of the two halves of the inputs
        _case("down_band_bf16", "product", 1000, 2048, 4096, "band", 32, "bf16", "gelu_tanh",
              bias=True, residual=True),
        # training backward of the band layer
        _case("grad_band_bf16", "gradient", 4096, 4096, 4096, "band", 64, "bf16", "gelu",
              bias=True),
        # gradients of scattered diagonals in full precision, odd number of vectors
        _case("grad_scatter_fp32", "gradient", 511, 4096, 4096, "scatter", 32, "fp32", "silu",
              bias=True),
        # a batch routed to 8 experts
        _case("experts_prompt_bf16", "product", 8192, 2048, 2048, "band", 32, "bf16", "silu",
              bias=True, save=True, experts=8),
        # 64 new tokens routed to 64 small experts: many hold one token or none
        _case("experts_decode_fp16", "product", 64, 1024, 1024, "band", 16, "fp16", "gelu",
              experts=64),
        # training backward of the routed batch
        _case("experts_grad_bf16", "gradient", 4096, 2048, 2048, "band", 32, "bf16", "silu",
              bias=True, experts=8),
        # small experts trained in full precision
        _case("experts_grad_fp32", "gradient", 257, 513, 512, "band", 8, "fp32", "relu",
              experts=16),
    ]


_MOST = 4096 * 4096 * 129   # products of the largest listed case


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("product", "gradient"))
    experts = rng.choice((0, 0, _log(rng, 2, 64)))
    pattern = rng.choice(("band", "band", "scatter", "stencil"))
    if pattern == "stencil":
        width = _log(rng, 4, 24)                        # grid side: width^3 unknowns
        rows = cols = width ** 3
    else:
        rows = _log(rng, 128, 8192)
        if rng.random() < 0.7:                          # widths are mostly multiples of 64
            rows = max(128, rows // 64 * 64)
        cols = rows if rng.random() < 0.7 else max(128, rows * rng.choice((1, 2, 4)) // 2)
        width = _log(rng, 1, 64)
    c = _case("", op, 1, rows, cols, pattern, width, rng.choice(("bf16", "bf16", "fp16", "fp32")),
              rng.choice(_ACTS), bias=rng.random() < 0.5, residual=rng.random() < 0.5,
              save=rng.random() < 0.5, experts=experts)
    if op == "gradient":
        c["residual"] = c["save"] = False
    per = _diagonals(c) * rows * (2 if op == "gradient" else 1)
    c["tokens"] = _log(rng, 1, max(1, min(8192, _MOST // (2 * per))))
    del c["name"]
    return c


def _offsets(c):
    """Host int32 offsets, ascending."""
    rows, cols, w = c["rows"], c["cols"], c["width"]
    if c["pattern"] == "band":
        # a band around the diagonal of every square block of the rectangle
        side = min(rows, cols)
        centres = range(0, cols, side) if cols >= rows else range(0, -rows, -side)
        off = {m + j for m in centres for j in range(-w, w + 1)}
    elif c["pattern"] == "scatter":
        g = np.random.default_rng(w)
        off = set(int(v) for v in g.choice(np.arange(-512, 513), size=w, replace=False)) | {0}
    else:
        off = {i + w * j + w * w * k for i in (-1, 0, 1) for j in (-1, 0, 1) for k in (-1, 0, 1)}
    return np.array(sorted(d for d in off if -rows < d < cols), np.int32)


def _diagonals(c):
    return len(_offsets(c))


def _entries(c):
    """Entries inside the matrix."""
    off = _offsets(c).astype(np.int64)
    return int((np.minimum(c["rows"], c["cols"] - off) - np.maximum(0, -off)).clip(0).sum())


def _lengths(c, seed):
    """Rows of each expert: a few busy experts, some without any."""
    g = np.random.default_rng(seed + 17)
    p = g.exponential(size=c["experts"]) ** 2
    return g.multinomial(c["tokens"], p / p.sum())


def prepare(case, seed):
    c, t = case, _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    off = _offsets(c)
    T, n, m, K, E = c["tokens"], c["rows"], c["cols"], len(off), max(1, c["experts"])
    stride = (n + 31) // 32 * 32

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)

    s = dict(case=c, seg=None, eid=None, bias=None, residual=None, z=None, dy=None)
    s["x"] = normal(T, m)
    s["vals"] = torch.zeros(E, K, stride, dtype=t, device="cuda")
    for k, d in enumerate(off.tolist()):
        lo, hi = max(0, -d), min(n, m - d)
        if hi > lo:
            s["vals"][:, k, lo:hi] = normal(E, hi - lo, scale=K ** -0.5)
    if c["experts"]:
        ln = _lengths(c, seed)
        s["seg"] = torch.from_numpy(np.concatenate([[0], np.cumsum(ln)]).astype(np.int64)).cuda()
        s["eid"] = torch.from_numpy(np.repeat(np.arange(E), ln)).cuda()
    else:
        s["vals"] = s["vals"][0]
    if c["op"] == "product":
        if c["bias"]:
            s["bias"] = normal(E, n, scale=0.1) if c["experts"] else normal(n, scale=0.1)
        if c["residual"]:
            s["residual"] = normal(T, n)
    else:
        s["dy"] = normal(T, n)
        s["z"] = normal(T, n) if c["act"] != "none" else None
    # columns of x that each entry reads, and rows of the operator that each column meets
    d = torch.from_numpy(off).cuda().long()[:, None]
    col = torch.arange(n, device="cuda")[None, :] + d
    row = torch.arange(m, device="cuda")[None, :] - d
    s["col"], s["col_in"] = col.clamp(0, m - 1), (col >= 0) & (col < m)
    s["row"], s["row_in"] = row.clamp(0, n - 1), (row >= 0) & (row < n)
    if own:
        import diagpu_b200 as dg
        s["plan"] = dg.SpmmPlan(n, m, off)
    return s


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _dact(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        u = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + u) + 0.5 * z * (1 - u * u) * a * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_product(s):
    c, x, n, t = s["case"], s["x"].float(), s["case"]["rows"], s["x"].dtype
    v = torch.where(s["col_in"], s["vals"][..., :n].float(), 0)
    bias = s["bias"].float() if s["bias"] is not None else None
    if s["eid"] is not None:
        v = v[s["eid"]]
        bias = bias[s["eid"]] if bias is not None else None
    z = x[:, s["col"]].mul_(v).sum(1)
    if bias is not None:
        z = z + bias
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (y.to(t), z.to(t)) if c["save"] else y.to(t)


def _plain_gradient(s):
    c, x, n, t = s["case"], s["x"].float(), s["case"]["rows"], s["x"].dtype
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _dact(s["z"].float(), c["act"])
    vals = s["vals"]
    v = torch.where(s["row_in"], vals.float().gather(-1, s["row"].expand(*vals.shape[:-1], -1)), 0)
    g = dz[:, s["row"]].mul_(v if s["eid"] is None else v[s["eid"]])
    dx = g.sum(1)
    g = x[:, s["col"]].mul_(s["col_in"]).mul_(dz[:, None, :])
    dvals = torch.zeros(vals.shape, device=x.device)
    dbias = None
    if s["eid"] is None:
        dvals[:, :n] = g.sum(0)
        dbias = dz.sum(0)
    else:
        dvals[:, :, :n] = torch.zeros_like(dvals[:, :, :n]).index_add_(0, s["eid"], g)
        dbias = torch.zeros(vals.shape[0], n, device=x.device).index_add_(0, s["eid"], dz)
    out = (dx.to(t), dvals.to(t))
    return out + (dbias.to(t),) if c["bias"] else out


def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_product(s) if c["op"] == "product" else _plain_gradient(s)
    import diagpu_b200 as dg
    if c["op"] == "product":
        return dg.spmm(s["plan"], s["vals"], s["x"], bias=s["bias"], act=c["act"],
                       residual=s["residual"], seg=s["seg"], save_z=c["save"])
    dx, dvals, dbias = dg.spmm_backward(s["plan"], s["vals"], s["x"], s["dy"], z=s["z"],
                                        act=c["act"], seg=s["seg"], bias_grad=c["bias"])
    return (dx, dvals, dbias) if c["bias"] else (dx, dvals)


def work(case):
    c, b = case, _SIZE[case["dtype"]]
    T, n, m, E, nnz = c["tokens"], c["rows"], c["cols"], max(1, c["experts"]), _entries(case)
    bias = E * n if c["bias"] else 0
    used = min(E, T) * nnz                              # an expert without rows is not read
    if c["op"] == "product":
        return dict(bytes=b * (T * m + used + bias
                               + T * n * (1 + int(c["residual"]) + int(c["save"]))),
                    flops=2 * T * nnz)
    return dict(bytes=b * (2 * T * m + T * n * (1 + int(c["act"] != "none")) + used + E * nnz + bias),
                flops=4 * T * nnz)


def exact(case, seed):
    """Diagonal by diagonal over shifted slices, in 64 bits."""
    s, c = prepare(case, seed), case
    T, n, m = c["tokens"], c["rows"], c["cols"]
    off = _offsets(c).tolist()
    x = s["x"].double()
    vals = s["vals"].double().reshape(-1, len(off), s["vals"].shape[-1])
    ends = [0, T] if s["seg"] is None else s["seg"].tolist()
    parts = [(e, ends[e], ends[e + 1]) for e in range(len(ends) - 1)]
    if c["op"] == "product":
        z = torch.zeros(T, n, dtype=torch.float64, device="cuda")
        for e, t0, t1 in parts:
            for k, d in enumerate(off):
                lo, hi = max(0, -d), min(n, m - d)
                z[t0:t1, lo:hi] += vals[e, k, lo:hi] * x[t0:t1, lo + d:hi + d]
            if s["bias"] is not None:
                z[t0:t1] += s["bias"].double().reshape(-1, n)[e]
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return (y, z) if c["save"] else y
    dz = s["dy"].double()
    if s["z"] is not None:
        dz = dz * _dact(s["z"].double(), c["act"])
    dx = torch.zeros_like(x)
    dvals = torch.zeros_like(vals)
    dbias = torch.zeros(vals.shape[0], n, dtype=torch.float64, device="cuda")
    for e, t0, t1 in parts:
        dbias[e] = dz[t0:t1].sum(0)
        for k, d in enumerate(off):
            lo, hi = max(0, -d), min(n, m - d)
            dx[t0:t1, lo + d:hi + d] += vals[e, k, lo:hi] * dz[t0:t1, lo:hi]
            dvals[e, k, lo:hi] = (dz[t0:t1, lo:hi] * x[t0:t1, lo + d:hi + d]).sum(0)
    out = (dx, dvals.reshape(s["vals"].shape))
    return out + (dbias.reshape((-1, n) if c["experts"] else (n,)),) if c["bias"] else out
