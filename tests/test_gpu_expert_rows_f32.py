"""Combining fp32 rows into tokens of any type, and the weights' gradient from them, against 64-bit sums: a sum of n
fp32 terms is within n 2^-23 of the sum of their sizes, plus the output's one rounding.  With rows of the tokens' own
16 bits the result would carry the rows' rounding too."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

ROWS_F32 = 0x100
CASES = [(1, 1, 1, 3, 1, 0, 0), (7, 2, 100, 20, 1, 0, 0), (33, 4, 64, 130, 2, 8, 0), (50, 9, 257, 500, 0, 1, 3),
         (300, 2, 1024, 640, 2, 0, 0), (5, 32, 1000, 160, 1, 0, 8), (64, 1, 2048, 64, 1, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,dim,rows,code,pad,shift", CASES)
@pytest.mark.parametrize("weighted", [False, True])
def test_combine_and_its_gradient(T, k, dim, rows, code, pad, shift, weighted):
    g = R.gen(T + dim)
    r = R.strided(R.randn(g, rows, dim), pad, shift)
    pos = torch.randint(-1, rows, (T, k), generator=g, device="cuda").int()
    pos[0] = -1
    if T > 2:
        pos[2, 0] = rows  # outside
    w = R.randn(g, T, k) if weighted else None
    out = R.strided(torch.full((T, dim), 5.0, device="cuda", dtype=R.DT[code]), pad, shift)
    type_ = code | ROWS_F32
    R.launch("launchExpertCombine", dim, type_, r, rows, r.stride(0), pos, w, out, out.stride(0), T, k, R.stream())
    dout = R.strided(R.randn(g, T, dim).to(R.DT[code]), pad, shift)
    dw = torch.full((T, k), 5.0, device="cuda")
    R.launch("launchExpertCombineBackward", dim, type_, r, rows, r.stride(0), pos, dout, dout.stride(0), dw, T, k, R.stream())
    torch.cuda.synchronize()
    fine = (pos >= 0) & (pos < rows)
    picked = r.double()[torch.where(fine, pos, 0).long()] * fine[:, :, None]
    terms = picked * (w.double()[:, :, None] if weighted else 1.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    assert ((out.double() - want).abs() <= k * 2.0 ** -23 * size + R.HALF[code] * want.abs() + R.TINY[code]).all()
    terms = picked * dout.double()[:, None, :]
    assert ((dw.double() - terms.sum(2)).abs() <= dim * 2.0 ** -23 * terms.abs().sum(2) + 1e-40).all()
    assert (dw[0] == 0).all() and (out[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", [1, 2])
def test_experts_forward_is_rounded_once(code):
    """Product of each expert's rows in fp32, combined: the tokens are within their own rounding of the exact sums."""
    P = pkg()
    T, k, E, N, K = 90, 2, 4, 264, 640
    g = R.gen(31)
    idx = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(T)]).int().contiguous()
    w = torch.rand(T, k, generator=g, device="cuda")
    cap = P.lib().routePlanCapacity(T, k, E, 16)
    off, order = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(cap, dtype=torch.int32, device="cuda")
    pos = torch.empty(T, k, dtype=torch.int32, device="cuda")
    R.launch("launchRoutePlan", idx, T, k, E, 16, cap, off, order, pos, R.stream())
    x = R.randn(g, T, K).to(R.DT[code])
    a, as_, _, _ = R.run_quantize(x, order=order, slots=k, rows=cap)
    parts = [R.make_fp8(g, N, K, 128) for _ in range(E)]
    b, bs = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    rows = torch.empty(cap, N, device="cuda")
    o = P.Fp8ProductOption(m=cap, n=N, k=K, numExperts=E, grouping=1, scaleRowsB=128, activation=0, outType=0, outStride=N)
    R.launch("launchFp8Product", C.byref(o), a, as_, b, bs, off, rows, R.stream())
    out = torch.empty(T, N, device="cuda", dtype=R.DT[code])
    R.launch("launchExpertCombine", N, code | ROWS_F32, rows, cap, N, pos, w, out, N, T, k, R.stream())
    torch.cuda.synchronize()
    q, s, _, _ = R.run_quantize(x)
    xv = R.values(q, s, K)
    want = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        by = w[t, j].double()[:, None]
        want.index_add_(0, t, xv[t] @ parts[e][2].t().contiguous() * by)
        size.index_add_(0, t, xv[t].abs() @ parts[e][2].abs().t().contiguous() * by)
    allow = (K * 2.0 ** -24 + k * 2.0 ** -23) * size + R.HALF[code] * want.abs() + R.TINY[code]
    assert ((out.double() - want).abs() <= allow).all()


def test_the_rows_type_goes_with_the_types_that_there_are():
    fake = 1 << 20  # never dereferenced

    def error(name, *args):
        L = pkg().lib()
        getattr(L, name)(*args)
        return L.tinymlp_last_error_message().decode() if L.tinymlp_last_error() else ""

    assert pkg().COMBINE_ROWS_F32 == ROWS_F32
    for type_, text in ((3 | ROWS_F32, "type"), (2 * ROWS_F32, "type"), (1 | ROWS_F32, "")):
        assert text in error("launchExpertCombine", 8, type_, fake, 4, 8, fake, None, fake, 8, 0, 2, None)
        assert text in error("launchExpertCombineBackward", 8, type_, fake, 4, 8, fake, fake, 8, fake, 0, 2, None)
    assert error("launchExpertCombine", 8, 1 | ROWS_F32, None, 0, 8, None, None, None, 8, 0, 2, None) == ""
