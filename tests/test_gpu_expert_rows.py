"""Combining the experts' rows and the weights' gradient against 64-bit sums: a sum of n fp32 terms is within
n 2^-23 of the sum of their sizes, plus the output's rounding."""
import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu

CASES = [(1, 1, 1, 3, 0, 0, 0), (7, 2, 100, 20, 1, 0, 0), (33, 4, 64, 130, 2, 8, 0), (50, 9, 257, 500, 0, 1, 3),
         (300, 2, 1024, 640, 2, 0, 0), (5, 32, 1000, 160, 1, 0, 4)]


@pytest.mark.parametrize("T,k,dim,rows,code,pad,shift", CASES)
@pytest.mark.parametrize("weighted", [False, True])
def test_combine_and_its_gradient(T, k, dim, rows, code, pad, shift, weighted):
    g = R.gen(T + dim)
    r = R.strided(R.randn(g, rows, dim).to(R.DT[code]), pad, shift)
    pos = torch.randint(-1, rows, (T, k), generator=g, device="cuda").int()
    pos[0] = -1
    if T > 2:
        pos[2, 0] = rows  # outside
    w = R.randn(g, T, k) if weighted else None
    out = R.strided(torch.full((T, dim), 5.0, device="cuda", dtype=R.DT[code]), pad, shift)
    R.launch("launchExpertCombine", dim, code, r, rows, r.stride(0), pos, w, out, out.stride(0), T, k, R.stream())
    dout = R.strided(R.randn(g, T, dim).to(R.DT[code]), pad, shift)
    dw = torch.full((T, k), 5.0, device="cuda")
    R.launch("launchExpertCombineBackward", dim, code, r, rows, r.stride(0), pos, dout, dout.stride(0), dw, T, k, R.stream())
    torch.cuda.synchronize()
    fine = (pos >= 0) & (pos < rows)
    picked = r.double()[torch.where(fine, pos, 0).long()] * fine[:, :, None]
    terms = picked * (w.double()[:, :, None] if weighted else 1.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    err = (out.double() - want).abs()
    assert (err <= k * 2.0 ** -23 * size + R.HALF[code] * want.abs() + R.TINY[code]).all()
    terms = picked * dout.double()[:, None, :]
    err = (dw.double() - terms.sum(2)).abs()
    assert (err <= dim * 2.0 ** -23 * terms.abs().sum(2) + 1e-40).all()
    assert (dw[0] == 0).all() and (out[0] == 0).all()


def test_zero_tokens():
    R.launch("launchExpertCombine", 8, 0, None, 0, 8, None, None, None, 8, 0, 2, R.stream())
    R.launch("launchExpertCombineBackward", 8, 0, None, 0, 8, None, None, 8, None, 0, 2, R.stream())
