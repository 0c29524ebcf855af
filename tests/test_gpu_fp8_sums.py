"""What the sums of 8-bit products hold, on data that their forms tell apart: values over all of e4m3 within a block,
of one sign, and large products that cancel beside small ones.

Exact sums (fp32 results, and 16-bit ones on request): K terms of exact products added in fp32 in any order are within
K 2^-24 sum |a b| of the exact sum.  16-bit results may come from sums of eight consecutive k, each of whose products
is cut to a multiple of 2^-13 of the largest one's power of two: seven cuts of the eight's largest |a b| at most, and
the same fp32 sums of the eights.  Either is rounded once to its type."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

EXACT = 0x100


def option(m, n, k, code, act=0, experts=1, grouping=0, rows_b=1):
    return pkg().Fp8ProductOption(m=m, n=n, k=k, numExperts=experts, grouping=grouping, scaleRowsB=rows_b, activation=act,
                                  outType=code, outStride=n)


def stored(g, rows, cols, kind):
    """Bytes, scales and 64-bit values of an 8-bit matrix: scales of 2^-3 .. 2^3 for each row's block."""
    P = pkg()
    if kind == "cancel":  # of each eight 256 and -256 (against 256 twice: products that cancel) and six small values
        v = torch.randint(1, 4, (rows, cols), generator=g, device="cuda").float()
        v[:, 0::8], v[:, 1::8] = 256.0, -256.0
        q = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        q = torch.randint(0, 127, (rows, cols), generator=g, device="cuda", dtype=torch.uint8)
        if kind == "wide":
            q |= torch.randint(0, 2, (rows, cols), generator=g, device="cuda", dtype=torch.uint8) * 128
    bytes_ = torch.zeros(rows, P.fp8_pitch(cols), dtype=torch.uint8, device="cuda")
    bytes_[:, :cols] = q
    s = torch.full((rows, P.fp8_scale_pitch(cols)), 0xAA, dtype=torch.uint8, device="cuda")
    s[:, :-(-cols // 128)] = torch.randint(124, 131, (rows, -(-cols // 128)), generator=g, device="cuda", dtype=torch.uint8)
    return bytes_, s, R.values(bytes_, s, cols)


def eights_largest(a, b):
    """Sum over the eights of k of their largest |a b|."""
    pad = -a.shape[1] % 8
    a, b = (torch.nn.functional.pad(v.abs(), (0, pad)) for v in (a, b))
    out = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
    for i in range(0, a.shape[1], 8):
        top = torch.zeros_like(out)
        for j in range(8):
            top = torch.maximum(top, a[:, i + j, None] * b[None, :, i + j])
        out += top
    return out


def allowed(av, bv, want, code, exact):
    K = av.shape[1]
    allow = K * 2.0 ** -24 * (av.abs() @ bv.abs().t().contiguous()) + R.HALF[code] * want.abs() + R.TINY[code]
    return allow if exact else allow + 7 * 2.0 ** -13 * eights_largest(av, bv)


# 1024 x 512 and 1400 x 600 go to tiles, 64 x 200 to waves that share k; K 384 is the least that takes 8-bit sums
SHAPES = [(1024, 512, 384), (1024, 520, 4096), (1400, 600, 1000), (64, 200, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["wide", "positive", "cancel"])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("exact", [False, True])
def test_sums(m, n, k, code, kind, exact):
    print(f"[sums] m={m} n={n} k={k} type={code} {kind} exact={exact}", flush=True)
    g = R.gen(m + n + k)
    a, as_, av = stored(g, m, k, kind)
    b, bs, bv = stored(g, n, k, "positive" if kind == "positive" else kind)
    if kind == "cancel":  # b's pair has one sign: 256 * 256 - 256 * 256 in every eight
        bv = bv.clone()
        b[:, 1:k:8] &= 0x7F
        bv[:, 1::8] = bv[:, 1::8].abs()
        scale = 2.0 ** -6
    else:
        scale = 2.0 ** -20
    # within fp16's range, by B's scales alone
    down = int(-math.log2(scale))
    bs[:, :-(-k // 128)] -= down
    bv = bv * scale
    out = torch.empty(m, n, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, k, code | (EXACT if exact else 0))), a, as_, b, bs, None, out, R.stream())
    torch.cuda.synchronize()
    want = av @ bv.t().contiguous()
    assert float(want.abs().max()) < 60000
    err = (out.double() - want).abs()
    allow = allowed(av, bv, want, code, exact or code == 0)
    assert (err <= allow).all(), float((err / allow).max())


@pytest.mark.gpu
@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("exact", [False, True])
def test_sums_by_expert(code, exact):
    """The same with rows by expert, wide values."""
    m, n, k, E = 1300, 520, 640, 3
    g = R.gen(11)
    a, as_, av = stored(g, m, k, "wide")
    parts = [stored(g, n, k, "wide") for _ in range(E)]
    for p in parts:
        p[1][:, :k // 128] -= 20
    b, bs = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    off = [0, 700, 712, 1300]
    out = torch.empty(m, n, device="cuda", dtype=R.DT[code])
    o = option(m, n, k, code | (EXACT if exact else 0), experts=E, grouping=1)
    R.launch("launchFp8Product", C.byref(o), a, as_, b, bs, torch.tensor(off, dtype=torch.int32, device="cuda"), out, R.stream())
    torch.cuda.synchronize()
    for e in range(E):
        x, w = av[off[e]:off[e + 1]], parts[e][2] * 2.0 ** -20
        want = x @ w.t().contiguous()
        err = (out[off[e]:off[e + 1]].double() - want).abs()
        assert (err <= allowed(x, w, want, code, exact)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("act", [0, 1])
def test_nan_and_relu_in_tiles(code, exact, act):
    """A NaN makes its row or column of a 16-bit product NaN, with ReLU too, and no other; ReLU clears the rest below 0."""
    m, n, k = 1024, 512, 700
    g = R.gen(5)
    a, as_, av = stored(g, m, k, "wide")
    b, bs, bv = stored(g, n, k, "wide")
    bs[:, :-(-k // 128)] -= 20
    a[515, 300], b[77, 5] = 0x7F, 0xFF
    out = torch.empty(m, n, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, k, code | (EXACT if exact else 0), act)), a, as_, b, bs, None, out, R.stream())
    torch.cuda.synchronize()
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[515], nan[:, 77] = True, True
    assert torch.equal(out.isnan(), nan)
    av[515], bv[77] = 0.0, 0.0
    bv = bv * 2.0 ** -20
    want = av @ bv.t().contiguous()
    allow = allowed(av, bv, want, code, exact)
    got = out.double()
    if act:
        want = want.clamp(min=0)
        assert (got[~nan] >= 0).all()
    assert ((got - want).abs() <= allow)[~nan].all()


def test_exact_sums_are_an_option_of_the_results_type():
    """It goes with the types that there are, and no other."""
    def error(o):
        L = pkg().lib()
        L.launchFp8Product(C.byref(o), None, None, None, None, None, None, None)
        return L.tinymlp_last_error_message().decode() if L.tinymlp_last_error() else ""

    assert pkg().PRODUCT_EXACT == EXACT
    for code in (0, 1, 2):
        assert error(option(0, 8, 100, code | EXACT)) == ""
    assert "type" in error(option(0, 8, 100, 3 | EXACT)) and "type" in error(option(0, 8, 100, 2 * EXACT))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [0, 2])
@pytest.mark.parametrize("m,n,k", [(4, 64, 512), (1024, 512, 512)])
@pytest.mark.parametrize("low_a", [True, False])
def test_scales_at_the_ends_of_their_range(m, n, k, code, low_a):
    """Scales of 2^-110 beside 2^93 and of 2^119 beside 2^-107: every value is a bf16 number, and no bit is lost."""
    g = R.gen(21)
    a, as_, _ = stored(g, m, k, "wide")
    b, bs, _ = stored(g, n, k, "wide")
    as_.fill_(17 if low_a else 246)
    bs.fill_(220 if low_a else 20)
    av, bv = R.values(a, as_, k), R.values(b, bs, k)
    out = torch.empty(m, n, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, k, code | EXACT)), a, as_, b, bs, None, out, R.stream())
    torch.cuda.synchronize()
    want = av @ bv.t().contiguous()
    assert ((out.double() - want).abs() <= allowed(av, bv, want, code, True)).all()
