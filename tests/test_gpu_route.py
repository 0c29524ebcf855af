"""Routing to experts, its gradient and the plan of the experts' rows against 64-bit and plain Python references.

Weights: scores carry a few fp32 roundings (exponential, sum over at most 1,024 experts, quotient), at most 2^-20 of
their size; indices and plans are equal.  Inputs are drawn again until no decision hangs on less than 1e-5."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu
REL = 2.0 ** -20


def option(E, k, sigmoid=0, groups=1, kept=1, best=2, renorm=1, scale=1.0, code=0):
    return pkg().RouteOption(numExperts=E, topK=k, scoreType=sigmoid, numGroups=groups, topGroups=kept, groupScore=best,
                             renormalize=renorm, scale=scale, logitsType=code)


def run_route(o, z, bias, T, k):
    idx = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), -7.0, device="cuda")
    R.launch("launchRouteExperts", C.byref(o), z, z.stride(0), bias, idx, w, T, R.stream())
    torch.cuda.synchronize()
    return idx, w


def check(o, z, bias, T, k, sigmoid, groups, kept, best, renorm, scale):
    idx, w = run_route(o, z, bias, T, k)
    ri, rw, _ = R.route(z, bias, k, sigmoid, groups, kept, best, renorm, scale)
    assert torch.equal(idx.cpu(), ri)
    err = (w.cpu().double() - rw).abs()
    assert (err <= REL * rw.abs() + 1e-30).all(), float((err / rw.abs().clamp(min=1e-30)).max())


CASES = [
    # T, E, k, sigmoid, groups, kept, best, bias, renorm, scale, type, pad, shift
    (1, 1, 1, 0, 1, 1, 2, False, 1, 1.0, 0, 0, 0),
    (3, 3, 2, 0, 1, 1, 2, True, 0, 1.0, 1, 1, 1),
    (130, 8, 2, 0, 1, 1, 2, False, 1, 1.0, 0, 0, 0),
    (257, 16, 16, 1, 4, 4, 2, True, 1, 2.5, 2, 0, 0),
    (65, 60, 6, 0, 4, 2, 1, False, 1, 1.0, 2, 3, 0),
    (33, 64, 32, 1, 1, 1, 2, True, 1, 1.0, 0, 4, 4),
    (40, 160, 6, 0, 8, 3, 2, True, 1, 1.0, 1, 0, 1),
    (50, 256, 8, 1, 8, 4, 2, True, 1, 2.5, 2, 0, 0),
    (9, 333, 9, 1, 1, 1, 2, False, 0, 1.0, 0, 0, 0),
    (7, 1024, 32, 0, 64, 9, 2, True, 1, 1.0, 0, 0, 0),
    (5, 1023, 7, 1, 33, 5, 1, True, 1, 1.0, 2, 0, 0),
    (6, 512, 8, 0, 1, 1, 2, False, 1, 1.0, 1, 8, 0),
    (11, 900, 4, 1, 3, 2, 2, False, 1, 1.0, 0, 0, 0),
    (300, 4, 4, 0, 2, 1, 2, False, 1, 1.0, 0, 0, 0),
]


@pytest.mark.parametrize("T,E,k,sigmoid,groups,kept,best,bias,renorm,scale,code,pad,shift", CASES)
def test_route(T, E, k, sigmoid, groups, kept, best, bias, renorm, scale, code, pad, shift):
    print(f"[route] T={T} E={E} k={k} groups={groups} type={code}", flush=True)
    for seed in range(50):
        g = R.gen(100 + seed)
        z = (R.randn(g, T, E) * 1.5).to(R.DT[code])
        b = R.randn(g, E) * 0.1 if bias else None
        if R.route(z, b, k, sigmoid, groups, kept, best, renorm, scale)[2] > 1e-5:
            break
    else:
        pytest.fail("no input without near ties")
    check(option(E, k, sigmoid, groups, kept, best, renorm, scale, code), R.strided(z, pad, shift), b, T, k, sigmoid,
          groups, kept, best, renorm, scale)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_ties_go_to_the_lowest_index(sigmoid, groups, kept):
    T, E, k = 64, 32, 6
    g = R.gen(5)
    z = torch.randint(-1, 2, (T, E), generator=g, device="cuda").float()
    z[0] = 0.0
    z[1] = 3.0
    check(option(E, k, sigmoid, groups, kept, 1), z, None, T, k, sigmoid, groups, kept, 1, 1, 1.0)


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("sigmoid", [0, 1])
def test_experts_that_are_not_available(sigmoid, code):
    """-inf and NaN logits and biases, rows without any expert, +inf, the types' lowest values."""
    T, E, k = 12, 16, 4
    z = (R.randn(R.gen(8), T, E)).to(R.DT[code])
    low = torch.finfo(R.DT[code]).min
    z[0] = -math.inf
    z[1] = math.nan
    z[2] = -math.inf
    z[2, 5] = 1.0
    z[3, ::2] = math.nan
    z[4, 3] = math.inf
    z[5] = low
    z[6, :14] = -math.inf
    z[7] = -math.inf
    z[7, 9] = low
    z[8, 1:] = low
    bias = torch.zeros(E, device="cuda")
    bias[2], bias[4] = -math.inf, math.nan
    for b in (None, bias):
        for groups, kept in ((1, 1), (4, 2)):
            check(option(E, k, sigmoid, groups, kept, 2, 1, 1.0, code), z, b, T, k, sigmoid, groups, kept, 2, 1, 1.0)
    idx, w = run_route(option(E, k, sigmoid, code=code), z, None, T, k)
    assert (idx[0] == -1).all() and (w[0] == 0).all() and (idx[1] == -1).all()
    assert idx[2].tolist() == [5, -1, -1, -1]


@pytest.mark.parametrize("T,E,k,sigmoid,renorm,code,pad", [
    (1, 1, 1, 0, 1, 0, 0), (5, 8, 2, 0, 1, 0, 0), (130, 8, 2, 1, 1, 2, 0), (33, 60, 6, 0, 0, 1, 3), (40, 64, 6, 0, 1, 0, 0),
    (17, 256, 8, 1, 0, 2, 4), (9, 1000, 32, 0, 1, 0, 1), (3, 333, 5, 0, 1, 1, 0)])
def test_route_backward(T, E, k, sigmoid, renorm, code, pad):
    """Against the formula differentiated in 64 bits: fp32 terms of at most max |dw| / sum s, REL of the row's largest."""
    g = R.gen(31)
    z = (R.randn(g, T, E) * 1.5).to(R.DT[code])
    z[0, 0] = -math.inf if E > k else z[0, 0]
    idx = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(T)]).int().contiguous()
    if E > k:
        idx[0, idx[0] == 0] = -1
    dw = R.randn(g, T, k)
    scale = 1.7
    zs = R.strided(z, pad)
    out = R.strided(torch.full((T, E), 9.0, device="cuda", dtype=R.DT[code]), pad)
    R.launch("launchRouteExpertsBackward", C.byref(option(E, k, sigmoid, renorm=renorm, scale=scale, code=code)), zs,
             zs.stride(0), idx, dw, out, out.stride(0), T, R.stream())
    torch.cuda.synchronize()

    def loss(z64):
        s = torch.where(z > -math.inf, torch.sigmoid(z64), 0.0) if sigmoid else torch.softmax(z64, 1)
        w = torch.where(idx >= 0, s.gather(1, idx.long().clamp(min=0)), 0.0)
        if renorm:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
        return (w * dw.double()).sum() * scale

    z64 = z.double().requires_grad_(True)
    loss(z64).backward()
    ref = torch.nan_to_num(z64.grad)
    err = (out.double() - ref).abs()
    s, _ = R.scores(z, sigmoid)
    sel = torch.where(idx >= 0, s.gather(1, idx.long().clamp(min=0)), 0.0).sum(1, keepdim=True)
    top = scale * dw.double().abs().amax(1, keepdim=True) / (sel.clamp(max=1.0) if renorm else 1.0) * s
    assert (err <= 8 * REL * top + R.HALF[code] * ref.abs() + R.TINY[code]).all(), float((err / top).max())
    # and the definition's own differences along a random direction
    v = R.randn(g, T, E).double()
    z0 = z.double()
    h = 1e-6
    lo, hi = z0 - h * v, z0 + h * v
    diff = (loss(hi) - loss(lo)) / (2 * h)
    got = (out.double() * v).sum()
    size = (top * v.abs()).sum()
    assert abs(float(diff - got)) <= float(size) * (8 * REL + 2 * R.HALF[code] + 1e-6)


@pytest.mark.parametrize("sigmoid", [0, 1])
def test_one_renormalised_expert_has_no_gradient(sigmoid):
    """Its weight is s / (s + 1e-20) = 1 in fp32, whatever its logit."""
    T, E = 500, 24
    g = R.gen(6)
    z, dw = R.randn(g, T, E) * 2, R.randn(g, T, 1)
    idx = torch.randint(0, E, (T, 1), generator=g, device="cuda").int()
    out = torch.full((T, E), 9.0, device="cuda")
    R.launch("launchRouteExpertsBackward", C.byref(option(E, 1, sigmoid)), z, E, idx, dw, out, E, T, R.stream())
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("T,k,E,align", [
    (0, 2, 4, 128), (1, 1, 1, 1), (1, 8, 256, 128), (7, 2, 16, 16), (300, 3, 5, 128), (1365, 3, 1024, 1), (2048, 2, 8, 128),
    (2049, 2, 8, 128), (5000, 4, 60, 64), (9000, 8, 1024, 128), (40000, 1, 2, 7), (70000, 2, 1, 128), (70001, 2, 700, 16)])
@pytest.mark.parametrize("holes", [False, True])
def test_plan(T, k, E, align, holes):
    print(f"[plan] T={T} k={k} E={E} align={align}", flush=True)
    P = pkg()
    g = R.gen(77)
    idx = (torch.rand(T, k, generator=g, device="cuda") ** 2 * E).int().clamp(max=E - 1)
    if holes and T:
        idx[torch.rand(T, k, generator=g, device="cuda") < 0.3] = -1
        idx[0, 0] = E  # outside
        idx[T // 2:T // 2 + 1] = -1
    cap = P.lib().routePlanCapacity(T, k, E, align)
    extra = 300
    off = torch.full((E + 1,), -9, dtype=torch.int32, device="cuda")
    order = torch.full((cap + extra,), -9, dtype=torch.int32, device="cuda")
    pos = torch.full((T, k), -9, dtype=torch.int32, device="cuda")
    for capacity in (cap, cap + extra):
        R.launch("launchRoutePlan", idx, T, k, E, align, capacity, off, order, pos, R.stream())
        torch.cuda.synchronize()
        ro, rr, rp = R.plan(idx, E, align, capacity)
        assert off.tolist() == ro
        assert order[:capacity].tolist() == rr
        assert pos.reshape(-1).tolist() == rp
        assert (order[capacity:] == -9).all()


def test_zero_tokens_and_repeats():
    R.launch("launchRouteExperts", C.byref(option(8, 2)), None, 8, None, None, None, 0, R.stream())
    z = R.randn(R.gen(3), 5000, 64)
    a = run_route(option(64, 6), z, None, 5000, 6)
    b = run_route(option(64, 6), z, None, 5000, 6)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
