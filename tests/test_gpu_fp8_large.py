"""8-bit matrices at the sizes where other forms take over: rows by expert in tiles of 128 and of 256 with more experts
than lanes, sums of more experts than are sorted by length, quantising of 2^17 blocks and more, batches of row-scaled
matrices.  Sums and roundings as in test_gpu_fp8_sums.py; quantised values bit for bit."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402
from test_gpu_fp8 import same_q, zero_blocks  # noqa: E402
from test_gpu_fp8_sums import EXACT, allowed, option, stored  # noqa: E402

pytestmark = pytest.mark.gpu


def ragged(g, experts, rows):
    """Starts of `experts` segments of `rows` in all, a few of them of 0 or 1 row."""
    w = torch.rand(experts, generator=g, device="cuda") + 0.2
    n = (w / w.sum() * rows).int()
    n[::17] = 0
    n[5::23] = 1
    n[-1] += rows - n.sum()
    return [0] + torch.cumsum(n, 0).tolist()


# 16-bit results with k of more than two blocks: tiles of 128 (the last three: of 256) by the rounds of tiles
ROWS = [(65, 13000, 300, 384, 2), (200, 12900, 1030, 300, 1), (300, 12000, 520, 640, 2), (1024, 9000, 130, 384, 1),
        (8, 36000, 2048, 384, 2), (8, 36100, 2041, 300, 1), (66, 147000, 2048, 300, 2)]


@pytest.mark.parametrize("E,rows,n,k,code", ROWS)
@pytest.mark.parametrize("exact", [False, True])
def test_rows_by_many_experts(E, rows, n, k, code, exact):
    print(f"[rows] E={E} rows={rows} n={n} k={k} type={code} exact={exact}", flush=True)
    g = R.gen(E + n)
    off = ragged(g, E, rows)
    m = off[-1] + 50
    a, as_, av = R.make_fp8(g, m, k)
    w = R.randn(g, E * n, k)  # all experts' rows in one: 1 row a scale
    b, bs, _, _ = R.run_quantize(w)
    out = torch.full((m, n), 7.0, device="cuda", dtype=R.DT[code])
    o = option(m, n, k, code | (EXACT if exact else 0), experts=E, grouping=1)
    o32 = torch.tensor(off, dtype=torch.int32, device="cuda")
    for _ in range(2):
        out.fill_(7.0)
        R.launch("launchFp8Product", C.byref(o), a, as_, b, bs, o32, out, R.stream())
        again = out.clone()
    R.launch("launchFp8Product", C.byref(o), a, as_, b, bs, o32, out, R.stream())
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    assert (out[off[-1]:] == 7.0).all()
    for e in range(E):
        r = slice(off[e], off[e + 1])
        if off[e] == off[e + 1] or (E > 100 and 3 < e < E - 40 and e % 5 and off[e + 1] - off[e] > 1):
            continue  # a part of many experts' references
        x, y = av[r], R.values(b[e * n:(e + 1) * n], bs[e * n:(e + 1) * n], k)
        want = x @ y.t().contiguous()
        # the eights' largest |a b| add up to at most sum |a b|
        size = x.abs() @ y.abs().t().contiguous()
        allow = k * 2.0 ** -24 * size + R.HALF[code] * want.abs() + R.TINY[code] + (0 if exact else 7 * 2.0 ** -13 * size)
        assert ((out[r].double() - want).abs() <= allow).all(), e


@pytest.mark.parametrize("E,m,n,code,longest", [(129, 130, 200, 0, 3), (300, 70, 136, 0, 2), (1024, 40, 60, 2, 1)])
def test_sums_of_many_experts(E, m, n, code, longest):
    print(f"[sums] E={E} m={m} n={n}", flush=True)
    g = R.gen(E)
    blocks = torch.randint(0, longest + 1, (E,), generator=g, device="cuda")
    off = [0] + (torch.cumsum(blocks, 0) * 128).tolist()
    K = off[-1] + 128
    a, as_, av = R.make_fp8(g, m, K)
    b, bs, bv = R.make_fp8(g, n, K)
    out = torch.full((E, m, n), 7.0, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, K, code, experts=E, grouping=2)), a, as_, b, bs,
             torch.tensor(off, dtype=torch.int32, device="cuda"), out, R.stream())
    torch.cuda.synchronize()
    for e in range(E):
        x, y = av[:, off[e]:off[e + 1]].contiguous(), bv[:, off[e]:off[e + 1]].contiguous()
        if x.shape[1] == 0:
            assert (out[e] == 0).all()
            continue
        want = x @ y.t().contiguous()
        assert ((out[e].double() - want).abs() <= allowed(x, y, want, code, True)).all(), e


@pytest.mark.parametrize("m,n,k,code", [(4090, 4093, 640, 1), (4090, 4093, 640, 2)])
@pytest.mark.parametrize("kind", ["wide", "cancel"])
def test_dense_in_the_largest_tiles(m, n, k, code, kind):
    """16 x 16 tiles of 256 with ragged ends; the bound of the 8-bit sums on data that cancels."""
    g = R.gen(m)
    a, as_, av = stored(g, m, k, kind)
    b, bs, bv = stored(g, n, k, kind)
    down = 20
    bs[:, :k // 128] -= down
    bv = bv * 2.0 ** -down
    out = torch.empty(m, n, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, k, code)), a, as_, b, bs, None, out, R.stream())
    torch.cuda.synchronize()
    for r in list(range(0, 700, 128)) + [3840, 4000]:  # rows of several tiles, the last ones among them
        x = av[r:r + 100]
        want = x @ bv.t().contiguous()
        allow = allowed(x, bv, want, code, False)
        assert ((out[r:r + 100].double() - want).abs() <= allow).all(), r


@pytest.mark.parametrize("rows,cols,code", [(45000, 384, 1), (33001, 385, 2), (140001, 128, 0), (17, 1 << 20, 2)])
@pytest.mark.parametrize("gathered", [False, True])
def test_quantize_many_blocks(rows, cols, code, gathered):
    print(f"[quantize] {rows}x{cols} type={code} gathered={gathered}", flush=True)
    g = R.gen(rows)
    src = 16 if cols > 1000 else 1003
    if not gathered:
        x = (R.randn(g, rows, cols) * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g, device="cuda").float())).to(R.DT[code])
        x[rows // 2, cols // 2] = float("inf")
        q, s, _, _ = R.run_quantize(x)
        want = x
    else:
        x = R.randn(g, src, cols).to(R.DT[code])
        order = torch.randint(-1, 2 * src, (rows,), generator=g, device="cuda").int()
        w = torch.rand(2 * src, generator=g, device="cuda")
        q, s, _, _ = R.run_quantize(x, order=order, weights=w, slots=2, rows=rows)
        slot = order.clamp(min=0).long()
        want = x.float()[slot // 2] * w[slot][:, None] * (order >= 0)[:, None]
    torch.cuda.synchronize()
    for r in range(0, rows, 8192):
        part = slice(r, min(r + 8192, rows))
        same_q(q[part], s[part], *R.quantize(want[part]), part.stop - part.start, cols, zero_blocks(want[part], 1))


@pytest.mark.parametrize("rows,cols,code", [(130, 200, 0), (5, 640, 1), (300, 128, 2)])
@pytest.mark.parametrize("t_side", [False, True])
def test_batches_with_a_scale_a_row(rows, cols, code, t_side):
    P = pkg()
    g = R.gen(rows)
    B, gap = 3, 40
    x = torch.zeros(B, rows * cols + gap, device="cuda", dtype=R.DT[code])
    v = x[:, :rows * cols].view(B, rows, cols)
    v.copy_(R.randn(g, B, rows, cols) * torch.tensor([1.0, 30.0, 0.01], device="cuda")[:, None, None])
    q, s = R.q_buffers(B * rows, cols)
    qt, st = R.q_buffers(B * cols, rows) if t_side else (None, None)
    o = P.Fp8QuantOption(rows=rows, cols=cols, batch=B, blockRows=1, srcType=code, slotsPerRow=1, srcRows=rows, srcStride=cols,
                         srcBatchStride=rows * cols + gap, gateStride=0)
    R.launch("launchFp8Quantize", C.byref(o), x, None, None, None, q, s, qt, st, R.stream())
    torch.cuda.synchronize()
    for i in range(B):
        r = slice(i * rows, (i + 1) * rows)
        same_q(q[r], s[r], *R.quantize(v[i]), rows, cols, zero_blocks(v[i], 1))
        if t_side:
            t, c = v[i].t().contiguous(), slice(i * cols, (i + 1) * cols)
            same_q(qt[c], st[c], *R.quantize(t), cols, rows, zero_blocks(t, 1))
