"""Norms around a block with gate and residual, and their gradients, against the formulas in 64 bits (gradients by
differentiating them, and by their differences).

An fp32 pass over a row of D elements has relative errors of a few 2^-23 per term and of the row's statistics: 2^-19 of
the sizes of the terms that are added, plus the output's rounding; sums over R rows add R 2^-24 of their terms' sizes."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu
REL = 2.0 ** -19

CASES = [
    # rows, dim, post, pre, gate rows, type, pad, shift, weights
    (1, 1, 1, 1, 1, 0, 0, 0, True), (3, 5, 2, 1, 2, 0, 1, 1, True), (1, 4096, 1, 1, 1000, 2, 0, 0, True),
    (5, 64, 2, 2, 0, 1, 0, 0, True), (70, 127, 1, 2, 7, 1, 0, 0, True), (33, 512, 0, 1, 1, 2, 8, 0, True),
    (129, 1024, 1, 0, 129, 0, 0, 0, True), (40, 1280, 2, 2, 16, 1, 0, 0, True), (65, 1283, 2, 1, 30, 0, 0, 0, True),
    (17, 2048, 1, 1, 5, 2, 0, 8, True), (9, 2050, 2, 2, 4, 1, 2, 0, False), (6, 4100, 1, 2, 3, 0, 0, 0, True),
    (4, 8192, 2, 2, 0, 2, 0, 0, True), (3, 8191, 1, 1, 2, 1, 0, 0, True), (4000, 96, 2, 1, 1, 2, 0, 0, True),
    (5000, 64, 1, 2, 700, 0, 0, 0, True), (4099, 128, 2, 2, 3, 1, 0, 0, True), (6001, 200, 1, 1, 100000, 0, 0, 0, False)]


def make(rows, dim, post, pre, gate_rows, code, pad, shift, weights, seed=0):
    g = R.gen(rows * 7 + dim + seed)
    dt = R.DT[code]
    t = dict(x=R.strided((R.randn(g, rows, dim) * 2 + 0.5).to(dt), pad, shift),
             f=R.strided((R.randn(g, rows, dim) * 0.7 - 3.0).to(dt), pad, shift),
             gate=R.strided((1 + 0.3 * R.randn(g, -(-rows // gate_rows), dim)).to(dt), pad, shift) if gate_rows else None)
    for side, kind in (("p", post), ("n", pre)):
        t[side + "w"] = 1 + 0.2 * R.randn(g, dim) if kind and weights else None
        t[side + "b"] = 0.3 * R.randn(g, dim) if kind and weights else None
    return t, g


def option(dim, post, pre, gate_rows, code, pad, alpha=0.9, beta=0.5, eps=1e-5):
    s = dim + pad
    return pkg().NormGateOption(dim=dim, postNorm=post, preNorm=pre, gateRows=gate_rows, residualScale=alpha,
                                blockScale=beta, epsilon=eps, dataType=code, strideX=s, strideF=s, strideGate=s, strideY=s,
                                strideH=s)


def reference(t, gate_rows, post, pre, alpha=0.9, beta=0.5, eps=1e-5):
    d = {n: v.double().contiguous() if v is not None else None for n, v in t.items()}
    # the option's factors are fp32 numbers
    alpha, beta, eps = (float(torch.tensor(v, dtype=torch.float32)) for v in (alpha, beta, eps))
    return d, lambda q: R.block(q["x"], q["f"], q["gate"], gate_rows, q["pw"], q["pb"], q["nw"], q["nb"], post, pre, alpha,
                                beta, eps)


@pytest.mark.parametrize("rows,dim,post,pre,gate_rows,code,pad,shift,weights", CASES)
def test_forward(rows, dim, post, pre, gate_rows, code, pad, shift, weights):
    print(f"[norm] {rows}x{dim} post={post} pre={pre} gate={gate_rows} type={code}", flush=True)
    t, _ = make(rows, dim, post, pre, gate_rows, code, pad, shift, weights)
    y, h = (R.strided(torch.full((rows, dim), 3.0, device="cuda", dtype=R.DT[code]), pad, shift) for _ in range(2))
    o = option(dim, post, pre, gate_rows, code, pad)
    args = [t[n] for n in ("x", "f", "gate", "pw", "pb", "nw", "nb")]
    d, f = reference(t, gate_rows, post, pre)
    ry, rh = f(d)
    R.launch("launchNormGateResidual", C.byref(o), *args, y, h, rows, R.stream())
    torch.cuda.synchronize()

    def close(got, want, size):
        err = (got.double() - want).abs()
        allow = REL * size + R.HALF[code] * want.abs() + R.TINY[code]
        assert (err <= allow).all(), float((err / allow).max())

    size_y = ry.abs().amax(1, keepdim=True) + d["x"].abs().amax(1, keepdim=True) + 1
    close(y, ry, size_y)
    # a norm divides by the deviation of its row: errors of y relative to that
    dev = (ry - (ry.mean(1, keepdim=True) if pre == 2 else 0)).square().mean(1, keepdim=True).add(1e-5).sqrt()
    w = d["nw"].abs().max() if d["nw"] is not None else 1.0
    close(h, rh, size_y * (w / dev if pre else 1.0) + rh.abs().amax(1, keepdim=True))
    # one output alone, and y in x's place
    h2 = torch.empty_like(h) if not pad else h.clone()
    if not pad:
        R.launch("launchNormGateResidual", C.byref(o), *args, None, h2, rows, R.stream())
        R.launch("launchNormGateResidual", C.byref(o), *args, t["x"], None, rows, R.stream())
        torch.cuda.synchronize()
        assert torch.equal(h2, h) and torch.equal(t["x"], y)


def test_norm_alone():
    """Without a block: y = alpha x, h = prenorm(y)."""
    t, _ = make(33, 320, 0, 2, 0, 2, 0, 0, True)
    y, h = torch.empty_like(t["x"]), torch.empty_like(t["x"])
    o = option(320, 0, 2, 0, 2, 0, alpha=1.0)
    R.launch("launchNormGateResidual", C.byref(o), t["x"], None, None, None, None, t["nw"], t["nb"], y, h, 33, R.stream())
    torch.cuda.synchronize()
    want = R.norm(t["x"].double(), 2, t["nw"].double(), t["nb"].double(), 1e-5)
    assert torch.equal(y, t["x"])
    assert ((h.double() - want).abs() <= 2.0 ** -8 * want.abs() + REL * 16).all()


@pytest.mark.parametrize("rows,dim,post,pre,gate_rows,code,pad,shift,weights", CASES)
def test_backward(rows, dim, post, pre, gate_rows, code, pad, shift, weights):
    print(f"[norm bwd] {rows}x{dim} post={post} pre={pre} gate={gate_rows} type={code}", flush=True)
    t, g = make(rows, dim, post, pre, gate_rows, code, pad, shift, weights)
    dt = R.DT[code]
    dy, dh = (R.strided(R.randn(g, rows, dim).to(dt), pad, shift) for _ in range(2))
    fill = lambda like: R.strided(torch.full(like.shape, 3.0, device="cuda", dtype=dt), pad, shift)  # noqa: E731
    dx, df, dg = fill(t["x"]), fill(t["f"]), fill(t["gate"]) if gate_rows else None
    par = {n: torch.full((dim,), 3.0, device="cuda") if t[n] is not None else None for n in ("pw", "pb", "nw", "nb")}
    args = [t[n] for n in ("x", "f", "gate", "pw", "pb", "nw", "nb")]
    o = option(dim, post, pre, gate_rows, code, pad)
    call = ["launchNormGateResidualBackward", C.byref(o), *args, dy, dh, dx, df, dg, par["pw"], par["pb"], par["nw"], par["nb"],
            rows, R.stream()]
    R.launch(*call)
    torch.cuda.synchronize()
    d, f = reference(t, gate_rows, post, pre)
    q = {n: v.clone().requires_grad_(True) if v is not None else None for n, v in d.items()}
    ry, rh = f(q)
    loss = (ry * dy.double()).sum() + (rh * dh.double()).sum()
    loss.backward()
    # sizes of the terms: dL/dy in full, over the rows' deviations
    y64 = ry.detach()
    dev2 = (y64 - (y64.mean(1, keepdim=True) if pre == 2 else 0)).square().mean(1, keepdim=True).add(1e-5).sqrt()
    f64 = d["f"]
    dev1 = (f64 - (f64.mean(1, keepdim=True) if post == 2 else 0)).square().mean(1, keepdim=True).add(1e-5).sqrt()
    one = torch.ones(1, dtype=torch.float64, device="cuda")
    big = lambda n: d[n].abs().max() if d[n] is not None else one  # noqa: E731
    rel2 = (1 + y64.abs().amax(1, keepdim=True) / dev2) if pre else 1.0   # a small deviation amplifies y's own errors
    rel1 = (1 + f64.abs().amax(1, keepdim=True) / dev1) if post else 1.0
    n2 = (y64.abs().amax(1, keepdim=True) / dev2) if pre else 1.0
    s2 = dy.double().abs().amax(1, keepdim=True) + dh.double().abs().amax(1, keepdim=True) * (
        big("nw") / dev2 * (1 + n2 * n2) if pre else 1.0)
    s2 = s2 * rel2
    gmax = big("gate")
    n1 = (f64.abs().amax(1, keepdim=True) / dev1) if post else f64.abs().amax(1, keepdim=True)
    s1 = s2 * gmax * (big("pw") / dev1 * (1 + n1 * n1) if post else 1.0) * rel1

    def close(got, want, size, kind=code):
        err = (got.double() - want).abs()
        allow = REL * size + R.HALF[kind] * want.abs() + R.TINY[kind]
        assert (err <= allow).all(), float((err / allow).max())

    close(dx, q["x"].grad, s2)
    close(df, q["f"].grad, s1)
    u = n1 * big("pw") + (big("pb") if d["pb"] is not None else 0)
    if gate_rows:
        per = torch.zeros(t["gate"].shape[0], 1, dtype=torch.float64, device="cuda").index_add_(
            0, torch.arange(rows, device="cuda") // gate_rows, (s2 * u * rel1).expand(rows, 1))
        close(dg, q["gate"].grad, per)
    for n, size in (("pw", s2 * gmax * n1 * rel1), ("pb", s2 * gmax), ("nw", dh.double().abs().amax(1, keepdim=True) * n2 * rel2),
                    ("nb", dh.double().abs().amax(1, keepdim=True))):
        if par[n] is not None:
            close(par[n], q[n].grad, size.expand(rows, 1).sum(), 0)
    # the same bits again
    first = [v.clone() for v in (dx, df, dg, *par.values()) if v is not None]
    R.launch(*call)
    torch.cuda.synchronize()
    for a, b in zip(first, [v for v in (dx, df, dg, *par.values()) if v is not None]):
        assert torch.equal(a, b)
    # the definition's differences along a direction of all inputs
    v = {n: torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64) if x is not None else None for n, x in d.items()}
    h = 1e-6

    def at(e):
        a, b = f({n: x + e * v[n] if x is not None else None for n, x in d.items()})
        return float((a * dy.double()).sum() + (b * dh.double()).sum())

    got = {"x": dx, "f": df, "gate": dg, **par}
    dot = sum(float((got[n].double() * v[n]).sum()) for n in d if d[n] is not None)
    sizes = sum(float((q[n].grad.abs() * v[n].abs()).sum()) for n in d if d[n] is not None)
    assert abs((at(h) - at(-h)) / (2 * h) - dot) <= sizes * (2 * R.HALF[code] + 1e-5) + 1e-6


def test_backward_parts():
    """Gradients that are not asked for, one side's gradient alone, and no rows."""
    rows, dim = 100, 256
    t, g = make(rows, dim, 1, 2, 10, 0, 0, 0, True)
    dh = R.randn(g, rows, dim)
    args = [t[n] for n in ("x", "f", "gate", "pw", "pb", "nw", "nb")]
    o = option(dim, 1, 2, 10, 0, 0)
    full = {n: torch.empty_like(t[n]) for n in ("x", "f", "gate", "pw", "pb", "nw", "nb")}
    zero = torch.zeros(rows, dim, device="cuda")
    R.launch("launchNormGateResidualBackward", C.byref(o), *args, zero, dh, *full.values(), rows, R.stream())
    for n in full:
        only = {m: torch.empty_like(t[m]) if m == n else None for m in full}
        R.launch("launchNormGateResidualBackward", C.byref(o), *args, None, dh, *only.values(), rows, R.stream())
        torch.cuda.synchronize()
        assert torch.equal(only[n], full[n]), n
    R.launch("launchNormGateResidualBackward", C.byref(o), None, t["f"], None, *args[3:], None, None, None, None, None,
             full["pw"], None, full["nw"], None, 0, R.stream())
    torch.cuda.synchronize()
    assert (full["pw"] == 0).all() and (full["nw"] == 0).all()
    dx = torch.empty_like(t["x"])
    R.launch("launchNormGateResidualBackward", C.byref(option(dim, 0, 0, 0, 0, 0)), t["x"], None, None, None, None, None, None,
             dh, None, dx, None, None, None, None, None, None, rows, R.stream())
    torch.cuda.synchronize()
    assert torch.equal(dx, 0.9 * dh)
