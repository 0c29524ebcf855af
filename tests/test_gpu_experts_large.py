"""Calls of more workgroups than one launch can have (2^32 threads): rows and tokens up to 2^30 are valid."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def pattern(rows, cols, dtype, period=1009):
    """[rows, cols] that repeats a random block of an odd number of rows, which does not line up with a launch."""
    p = R.randn(R.gen(period), period, cols).to(dtype)
    x = torch.empty(rows, cols, dtype=dtype, device="cuda")
    whole = rows // period * period
    x[:whole].view(-1, period, cols).copy_(p)
    x[whole:] = p[:rows - whole]
    return x


def repeats(y, period=1009):
    """Whether every block of rows has the first one's bits."""
    for r in range(0, y.shape[0], period << 10):
        part = y[r:r + (period << 10)]
        whole = part.shape[0] // period * period
        if not (bool((part[:whole].view(-1, period, *y.shape[1:]) == y[:period]).all()) and torch.equal(part[whole:], y[:part.shape[0] - whole])):
            return False
    return True


def norm_option(dim, pre):
    return pkg().NormGateOption(dim=dim, postNorm=0, preNorm=pre, gateRows=0, residualScale=0.5, blockScale=1.0, epsilon=1e-6,
                                dataType=1, strideX=dim, strideF=dim, strideGate=dim, strideY=dim, strideH=dim)


def test_norm_rows_of_a_wave():
    rows, dim = (1 << 26) + 5, 2
    x = pattern(rows, dim, torch.float16)
    h = torch.full((rows, dim), 3.0, dtype=torch.float16, device="cuda")
    R.launch("launchNormGateResidual", C.byref(norm_option(dim, 1)), x, None, None, None, None, None, None, None, h, rows, R.stream())
    torch.cuda.synchronize()
    want = R.norm(0.5 * x[:1009].double(), 1, None, None, 1e-6)
    err = (h[:1009].double() - want).abs()
    assert (err <= R.HALF[1] * want.abs() + 2.0 ** -19 * want.abs().amax(1, keepdim=True) + R.TINY[1]).all()
    assert repeats(h)


def test_norm_rows_of_a_workgroup():
    rows, dim = (1 << 24) + 3, 2056
    x = pattern(rows, dim, torch.float16)  # 69 GB: in place
    first = x[:1009].clone()
    R.launch("launchNormGateResidual", C.byref(norm_option(dim, 0)), x, None, None, None, None, None, None, x, None, rows, R.stream())
    torch.cuda.synchronize()
    assert torch.equal(x[:1009], 0.5 * first)
    assert repeats(x)


def test_combine_of_many_elements():
    """More than 2^32 elements, each a thread's: rows that are not whole 16-byte pieces."""
    T, dim, k, rows = (1 << 20) + 3, 4099, 2, 1009
    r = R.randn(R.gen(1), rows, dim).half()
    pos = torch.stack([torch.arange(T, device="cuda") % 1009, (torch.arange(T, device="cuda") % 1009 * 7 + 3) % 1009], 1).int()
    out = torch.full((T, dim), 3.0, dtype=torch.float16, device="cuda")
    R.launch("launchExpertCombine", dim, 1, r, rows, dim, pos.contiguous(), None, out, dim, T, k, R.stream())
    torch.cuda.synchronize()
    want = (r.double()[pos[:1009, 0].long()] + r.double()[pos[:1009, 1].long()])
    assert ((out[:1009].double() - want).abs() <= R.HALF[1] * want.abs() + R.TINY[1]).all()
    assert repeats(out)


@pytest.mark.parametrize("k", [1, 3])
def test_combine_backward_of_many_tokens(k):
    T, dim, rows = (1 << 26) + 5, 1, 1009
    r = R.randn(R.gen(2), rows, dim).half()
    pos = ((torch.arange(T, device="cuda") % 1009)[:, None] * (5 + torch.arange(k, device="cuda")) % 1009).int()
    dout = pattern(T, dim, torch.float16)
    dw = torch.full((T, k), 3.0, device="cuda")
    R.launch("launchExpertCombineBackward", dim, 1, r, rows, dim, pos, dout, dim, dw, T, k, R.stream())
    torch.cuda.synchronize()
    want = r.float()[pos[:1009].long(), 0] * dout[:1009].float()
    assert torch.equal(dw[:1009], want)  # one product of two 11-bit numbers each
    assert repeats(dw)


def test_routing_of_many_tokens():
    """A wave a token: 33 groups of one expert."""
    T, E, k = (1 << 26) + 5, 33, 2
    z = pattern(T, E, torch.float16)
    o = pkg().RouteOption(numExperts=E, topK=k, scoreType=0, numGroups=33, topGroups=33, groupScore=1, renormalize=1, scale=1.0,
                          logitsType=1)
    idx, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), -7.0, device="cuda")
    R.launch("launchRouteExperts", C.byref(o), z, E, None, idx, w, T, R.stream())
    torch.cuda.synchronize()
    ri, rw, _ = R.route(z[:1009], None, k, 0, 1, 1, 1, 1, 1.0)
    assert torch.equal(idx[:1009].cpu(), ri)
    assert ((w[:1009].cpu().double() - rw).abs() <= 2.0 ** -20 * rw.abs()).all()
    assert repeats(idx) and repeats(w)


def test_routing_gradient_of_many_tokens():
    T, E = (1 << 26) + 5, 129
    z = pattern(T, E, torch.float16)
    first = z[:1009].clone()
    idx = (torch.arange(T, device="cuda") % 1009 * 31 % E).int()
    dw = pattern(T, 1, torch.float32)
    o = pkg().RouteOption(numExperts=E, topK=1, scoreType=0, numGroups=1, topGroups=1, groupScore=1, renormalize=0, scale=1.0,
                          logitsType=1)
    R.launch("launchRouteExpertsBackward", C.byref(o), z, E, idx, dw, z, E, T, R.stream())  # 17 GB: in place
    torch.cuda.synchronize()
    s = torch.softmax(first.double(), 1)
    picked = s.gather(1, idx[:1009, None].long())
    hot = torch.nn.functional.one_hot(idx[:1009].long(), E)
    want = dw[:1009].double() * picked * (hot - s)
    assert ((z[:1009].double() - want).abs() <= 8 * 2.0 ** -20 * dw[:1009].double().abs() * s + R.HALF[1] * want.abs() + R.TINY[1]).all()
    assert repeats(z)


def test_quantize_many_blocks():
    """2^30 blocks of 128 and more: gathered from a small source by an order."""
    P = pkg()
    rows, cols, period = (1 << 29) + 5, 129, 1009
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 150 GB")
    x = R.randn(R.gen(7), period, cols).half()
    order = torch.arange(period, dtype=torch.int32, device="cuda").repeat(rows // period + 1)[:rows].contiguous()
    q = torch.empty(rows, P.fp8_pitch(cols), dtype=torch.uint8, device="cuda")
    s = torch.zeros(rows, P.fp8_scale_pitch(cols), dtype=torch.uint8, device="cuda")
    o = P.Fp8QuantOption(rows=rows, cols=cols, batch=1, blockRows=1, srcType=1, slotsPerRow=1, srcRows=period, srcStride=cols,
                         srcBatchStride=0, gateStride=0)
    R.launch("launchFp8Quantize", C.byref(o), x, order, None, None, q, s, None, None, R.stream())
    torch.cuda.synchronize()
    want_q, want_s = R.quantize(x)
    assert torch.equal(q[:period, :cols].contiguous().view(torch.float8_e4m3fn).double(), want_q)
    assert (q[:period, cols:] == 0).all() and torch.equal(s[:period, :2], want_s)
    assert repeats(q) and repeats(s)
