"""Gather and quantise, products by expert and combine in 4 bits (include/experts_abi.h), their rows in between in fp32 or in
the tokens' type, against 64 bits of the whole chain."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("T,E,k,n,K", [(1, 4, 2, 33, 100), (50, 5, 2, 257, 300), (700, 8, 3, 512, 1024), (5000, 8, 2, 1025, 260)])
def test_rows_between(T, E, k, n, K, code, f32):
    P, g = pkg(), R.gen(T + n)
    x = R.randn(g, T, K).to(S.DT[code])
    index = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k].int().contiguous()
    weight = torch.softmax(R.randn(g, T, k), 1).contiguous()
    parts = [S.make_fp4(g, n, K) for _ in range(E)]
    w, ws, b = (torch.stack(p).contiguous() for p in zip(*parts))
    cap = P.lib().routePlanCapacity(T, k, E, 1)
    offsets, order = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(cap, dtype=torch.int32, device="cuda")
    position = torch.empty(T, k, dtype=torch.int32, device="cuda")
    R.launch("launchRoutePlan", index, T, k, E, 1, cap, offsets, order, position, R.stream())
    q, s = S.run_quantize4(x, 1, order, k, cap)
    between = 0 if f32 else code
    rows = torch.full((cap, n), -7.0, dtype=S.DT[between], device="cuda")
    o = P.Fp4ProductOption(m=cap, n=n, k=K, numExperts=E, grouping=P.PRODUCT_ROWS, activation=0, outType=between, outStride=n)
    R.launch("launchFp4Product", C.byref(o), q, s, w, ws, offsets, rows, R.stream())
    out = torch.empty(T, n, dtype=S.DT[code], device="cuda")
    R.launch("launchExpertCombine", n, code | (P.COMBINE_ROWS_F32 if f32 else 0), rows, cap, n, position, weight, out, n, T, k, R.stream())
    qx, byte = S.quantize4(x, 1)
    a = qx * torch.exp2(byte.double() - 127).repeat_interleave(32, 1)[:, :K]
    want, off = torch.zeros(T, n, dtype=torch.float64, device="cuda"), torch.zeros(T, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for e in range(E):
        t, j = torch.nonzero(index == e, as_tuple=True)
        ref, mag = a[t] @ b[e].t(), a[t].abs() @ b[e].abs().t()
        by = weight[t, j].double()[:, None]
        bound = S.product_bound(K, mag, ref, between)  # each row in fp32 or rounded to the tokens' type
        want.index_add_(0, t, ref * by)
        off.index_add_(0, t, bound * by)
        size.index_add_(0, t, (ref.abs() + bound) * by)
    off = off + (k + 1) * 2.0 ** -24 * size  # a product and an addition each
    bound = off + S.HALF[code] * (want.abs() + off) + S.TINY[code]
    fine = (size < 60000) | (code != 1)
    assert bool(((out.double() - want).abs().le(bound) | ~fine).all())
