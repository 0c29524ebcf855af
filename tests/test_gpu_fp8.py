"""8-bit matrices with a scale for each block of 128: quantising bit for bit against 64-bit arithmetic, products
against 64-bit sums of the stored values.

A product's fp32 sum of K terms is within K 2^-24 sum |a b| of the exact one whatever the order of its additions, and
its output within half a spacing of its type."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


def same_q(q, s, want_q, want_s, rows, cols, zero_blocks):
    got = q[:, :cols].contiguous().view(torch.float8_e4m3fn).double()
    assert torch.equal(got.isnan(), want_q.isnan())
    assert torch.equal(got.nan_to_num(), want_q.nan_to_num())
    assert (q[:, cols:] == 0).all()
    b = want_s.shape[1]
    same = (s[:, :b] == want_s) | zero_blocks
    assert same.all()


def zero_blocks(x, block_rows):
    q, _ = R.quantize(x.nan_to_num(0.0, 0.0, 0.0), block_rows)
    R_, Cc = x.shape
    p = torch.zeros(-(-R_ // block_rows) * block_rows, -(-Cc // 128) * 128, device=x.device)
    p[:R_, :Cc] = (x.double().nan_to_num(0.0, 0.0, 0.0) != 0).float()
    return p.view(-(-R_ // block_rows), block_rows, -1, 128).amax((1, 3)) == 0


def wild(g, rows, cols, dtype):
    x = R.randn(g, rows, cols) * torch.exp2(torch.randint(-12, 8, (rows, 1), generator=g, device="cuda").float())
    x = x.to(dtype)
    if rows > 2 and cols > 2:
        x[0] = 0.0
        x[1, cols // 2] = math.nan
        x[2, 0] = math.inf
        x[2, -1] = -math.inf
    if rows > 4:
        x[3] = 448.0 * 2.0 ** -3
        x[4] = torch.tensor(449.0, dtype=dtype)
        x[4, ::2] = 17.0
    return x


@pytest.mark.parametrize("rows,cols,code,pad,shift", [
    (1, 1, 0, 0, 0), (5, 127, 1, 0, 1), (7, 128, 2, 0, 0), (33, 129, 0, 3, 0), (130, 640, 1, 8, 0), (257, 1000, 2, 0, 0),
    (3, 4096, 0, 0, 4), (128, 384, 2, 0, 8)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(rows, cols, code, pad, shift, block_rows):
    x = R.strided(wild(R.gen(rows + cols), rows, cols, R.DT[code]), pad, shift)
    for row_side, t_side in ((True, False), (False, True), (True, True)):
        q, s, qt, st = R.run_quantize(x, block_rows, row_side=row_side, t_side=t_side)
        torch.cuda.synchronize()
        if row_side:
            same_q(q, s, *R.quantize(x, block_rows), rows, cols, zero_blocks(x, block_rows))
        if t_side:
            xt = x.t().contiguous()
            same_q(qt, st, *R.quantize(xt, block_rows), cols, rows, zero_blocks(xt, block_rows))


def test_every_e4m3_rounding():
    """Values between neighbours of e4m3 and at their halves, both signs, at the scale 1 (the row's 448 sets it)."""
    b = torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).float()
    halves = (b[:-1] + b[1:]) / 2
    near = torch.cat([b, halves, halves * (1 + 2.0 ** -20), halves * (1 - 2.0 ** -20)])
    x = torch.cat([near, -near])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 127)).view(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), 448.0, device="cuda")], 1).contiguous()
    q, s, _, _ = R.run_quantize(x)
    torch.cuda.synchronize()
    assert (s[:, 0] == 127).all()
    assert torch.equal(q.view(torch.float8_e4m3fn).float(), x.to(torch.float8_e4m3fn).float())


def test_smallest_and_largest_scales():
    x = torch.zeros(4, 128, device="cuda")
    x[0] = 1e-44
    x[1] = 3e38
    x[2] = 2.0 ** -126
    x[3, 5] = 2.0 ** -110
    q, s, _, _ = R.run_quantize(x)
    torch.cuda.synchronize()
    rq, rs = R.quantize(x)
    assert torch.equal(s[:, :1], rs)
    assert torch.equal(q.view(torch.float8_e4m3fn).double(), rq)


@pytest.mark.parametrize("code", [0, 2])
def test_quantize_gathered_weighted_gated(code):
    """Rows by an order with holes, slots of a row, weights of the slots, and the gradient behind a ReLU."""
    g = R.gen(12)
    T, k, cols, rows = 50, 2, 200, 270
    x = R.randn(g, T, cols).to(R.DT[code])
    order = torch.randint(-1, T * k, (rows,), generator=g, device="cuda").int()
    order[5] = T * k + 3  # behind the source's rows: zero
    w = torch.rand(T * k + 8, generator=g, device="cuda")
    gate = R.randn(g, rows, cols).to(R.DT[code])
    gate[0, :10] = 0.0
    fine = (order >= 0) & (order < T * k)
    slot = torch.where(fine, order, 0).long()
    v = x.float()[slot // k] * fine[:, None]
    for weights, gt in ((None, None), (w, None), (None, gate), (w, gate)):
        want = v * w[slot][:, None] if weights is not None else v
        want = torch.where(gate.float() > 0, want, 0.0) if gt is not None else want
        for t_side in (False, True):
            q, s, qt, st = R.run_quantize(x, order=order, weights=weights, gate=gt, slots=k, rows=rows, t_side=t_side)
            torch.cuda.synchronize()
            same_q(q, s, *R.quantize(want), rows, cols, zero_blocks(want, 1))
            if t_side:
                t = want.t().contiguous()
                same_q(qt, st, *R.quantize(t), cols, rows, zero_blocks(t, 1))


def test_quantize_batches():
    P = pkg()
    g = R.gen(3)
    B, rows, cols = 3, 130, 200
    x = R.randn(g, B, rows, cols) * torch.tensor([1.0, 30.0, 0.01], device="cuda")[:, None, None]
    q = torch.empty(B, rows, P.fp8_pitch(cols), dtype=torch.uint8, device="cuda")
    s = torch.empty(B, 2, P.fp8_scale_pitch(cols), dtype=torch.uint8, device="cuda")
    qt = torch.empty(B, cols, P.fp8_pitch(rows), dtype=torch.uint8, device="cuda")
    st = torch.empty(B, 2, P.fp8_scale_pitch(rows), dtype=torch.uint8, device="cuda")
    o = P.Fp8QuantOption(rows=rows, cols=cols, batch=B, blockRows=128, srcType=0, slotsPerRow=1, srcRows=rows,
                         srcStride=cols, srcBatchStride=rows * cols, gateStride=0)
    P.launch("launchFp8Quantize", C.byref(o), x, None, None, None, q, s, qt, st, R.stream())
    torch.cuda.synchronize()
    for b in range(B):
        same_q(q[b], s[b], *R.quantize(x[b], 128), rows, cols, zero_blocks(x[b], 128))
        t = x[b].t().contiguous()
        same_q(qt[b], st[b], *R.quantize(t, 128), cols, rows, zero_blocks(t, 128))


def check_product(out, want, size, K, code, relu=False):
    """want: exact, size: sum |a b|."""
    if relu:
        want = want.clamp(min=0)
    err = (out.double() - want).abs()
    allow = K * 2.0 ** -24 * size + R.HALF[code] * want.abs() + R.TINY[code]
    assert (err <= allow).all(), float((err / allow.clamp(min=1e-300)).max())


def option(m, n, k, experts=1, grouping=0, rows_b=128, act=0, code=0, stride=None):
    return pkg().Fp8ProductOption(m=m, n=n, k=k, numExperts=experts, grouping=grouping, scaleRowsB=rows_b, activation=act,
                                  outType=code, outStride=stride or n)


@pytest.mark.parametrize("m,n,k,code,rows_b,act,pad,shift", [
    (1, 1, 1, 0, 128, 0, 0, 0), (1, 4096, 512, 2, 128, 0, 0, 0), (1, 100, 4000, 1, 1, 0, 0, 0), (2, 129, 128, 0, 1, 1, 3, 1),
    (5, 640, 1280, 1, 128, 0, 0, 0), (16, 257, 2000, 0, 128, 0, 0, 0), (17, 512, 130, 2, 1, 0, 0, 0),
    (31, 96, 5000, 0, 1, 0, 0, 0), (33, 64, 640, 1, 128, 1, 4, 0), (64, 1000, 1024, 2, 128, 0, 0, 0),
    (65, 31, 384, 0, 128, 0, 1, 0), (100, 300, 900, 0, 1, 0, 0, 0), (128, 128, 256, 1, 128, 0, 0, 0),
    (129, 1290, 127, 0, 128, 0, 0, 0), (257, 513, 1000, 2, 1, 1, 0, 2), (300, 2048, 512, 1, 128, 0, 8, 0),
    (1000, 700, 700, 0, 128, 0, 0, 0), (4096, 4090, 700, 2, 128, 0, 0, 0), (4090, 4096, 4300, 1, 1, 1, 8, 0), (2049, 1025, 260, 2, 128, 0, 0, 0), (4100, 2100, 128, 1, 1, 0, 0, 0)])
def test_dense_product(m, n, k, code, rows_b, act, pad, shift):
    print(f"[product] m={m} n={n} k={k} type={code}", flush=True)
    g = R.gen(m + n + k)
    a, as_, av = R.make_fp8(g, m, k)
    b, bs, bv = R.make_fp8(g, n, k, rows_b)
    out = R.strided(torch.full((m, n), 7.0, device="cuda", dtype=R.DT[code]), pad, shift)
    whole = out.as_strided((m * (n + pad),), (1,), shift)
    guard = whole.clone()
    R.launch("launchFp8Product", C.byref(option(m, n, k, rows_b=rows_b, act=act, code=code, stride=out.stride(0))), a, as_, b,
             bs, None, out, R.stream())
    torch.cuda.synchronize()
    check_product(out, av @ bv.t().contiguous(), av.abs() @ bv.abs().t().contiguous(), k, code, act == 1)
    if pad:
        assert torch.equal(whole.view(m, n + pad)[:, n:], guard.view(m, n + pad)[:, n:])


@pytest.mark.parametrize("m,n,k,code,rows_b,act,pad,shift", [
    (65, 64, 4096, 0, 128, 0, 0, 0), (300, 511, 4000, 1, 1, 1, 1, 1), (1025, 64, 2000, 2, 128, 0, 0, 0), (130, 2048, 1024, 2, 1, 0, 8, 0),
    (4099, 40, 900, 0, 128, 0, 0, 0), (129, 5121, 1300, 0, 128, 0, 0, 0), (64, 20480, 700, 2, 128, 0, 0, 0),
    (17, 30001, 1030, 0, 128, 1, 0, 0), (1, 65537, 600, 1, 128, 0, 0, 0), (33, 40000, 200, 1, 1, 0, 0, 0)])
def test_dense_product_either_form(m, n, k, code, rows_b, act, pad, shift):
    """Many rows by few columns with a long k, whose waves share k, and few rows by many columns, in tiles."""
    test_dense_product(m, n, k, code, rows_b, act, pad, shift)


def segments(lengths, align):
    off = [0]
    for n in lengths:
        off.append(off[-1] + -(-n // align) * align)
    return off


@pytest.mark.parametrize("lengths,align,n,k,code,rows_b", [
    ([5], 1, 40, 100, 0, 128), ([0, 3, 0, 0, 130, 1], 1, 200, 300, 1, 128), ([128, 0, 300, 77], 128, 640, 512, 2, 128),
    ([0, 0, 0], 128, 64, 64, 0, 1), ([1] * 20 + [0] * 60 + [7] * 5, 1, 136, 260, 0, 1), ([700, 10, 513], 128, 300, 384, 2, 128),
    ([4000, 60, 1, 0, 3000], 128, 2050, 300, 2, 128), ([2, 1, 3, 0, 2], 16, 1030, 1000, 1, 128), ([20, 40, 60, 17], 16, 256, 640, 0, 128), ([1500, 2000], 128, 520, 130, 1, 1)])
def test_rows_product(lengths, align, n, k, code, rows_b):
    print(f"[rows product] {lengths} n={n} k={k}", flush=True)
    E = len(lengths)
    off = segments(lengths, align)
    m = off[-1] + 37
    g = R.gen(n + k)
    a, as_, av = R.make_fp8(g, m, k)
    parts = [R.make_fp8(g, n, k, rows_b) for _ in range(E)]
    b, bs = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    o32 = torch.tensor(off, dtype=torch.int32, device="cuda")
    out = torch.full((m, n), 7.0, device="cuda", dtype=R.DT[code])
    R.launch("launchFp8Product", C.byref(option(m, n, k, E, 1, rows_b, code=code)), a, as_, b, bs, o32, out, R.stream())
    torch.cuda.synchronize()
    for e in range(E):
        r = slice(off[e], off[e + 1])
        check_product(out[r], av[r] @ parts[e][2].t().contiguous(), av[r].abs() @ parts[e][2].abs().t().contiguous(), k, code)
    assert (out[off[-1]:] == 7.0).all()


@pytest.mark.parametrize("lengths,align,n,k,code,rows_b", [
    ([200, 0, 90, 17], 1, 64, 2000, 0, 1), ([300, 129], 128, 100, 4100, 1, 128), ([70, 1, 0, 64], 16, 33, 1500, 2, 128),
    ([3, 0, 1, 5, 2, 0, 9, 4], 1, 8193, 384, 2, 128), ([40, 2, 0, 130], 1, 16384, 300, 0, 128)])
def test_rows_product_either_form(lengths, align, n, k, code, rows_b):
    """The same with experts: segments that end inside a tile, an empty one, and one much longer than the others."""
    test_rows_product(lengths, align, n, k, code, rows_b)


@pytest.mark.parametrize("lengths,m,n,code,rows_b", [
    ([100], 40, 60, 0, 1), ([0, 128, 0, 300, 1], 130, 257, 0, 1), ([1000, 0, 129], 300, 200, 2, 1), ([0, 0], 33, 20, 1, 128),
    ([5, 6, 7, 8], 512, 640, 0, 1), ([5, 4300, 7, 8], 512, 640, 0, 1), ([0, 700, 384, 5], 2050, 2100, 1, 1), ([], 8, 8, 0, 1), ([2500, 130], 64, 1000, 1, 1)])
def test_sum_product(lengths, m, n, code, rows_b):
    print(f"[sum product] {lengths} m={m} n={n}", flush=True)
    lengths = lengths or [0]
    E = len(lengths)
    off = segments(lengths, 128)
    K = off[-1] + (256 if off[-1] else 0)
    out = torch.full((E, m, n), 7.0, device="cuda", dtype=R.DT[code])
    o32 = torch.tensor(off, dtype=torch.int32, device="cuda")
    if K:
        g = R.gen(m + n)
        a, as_, av = R.make_fp8(g, m, K)
        b, bs, bv = R.make_fp8(g, n, K, rows_b)
    else:
        a = as_ = b = bs = None
    R.launch("launchFp8Product", C.byref(option(m, n, K, E, 2, rows_b, code=code)), a, as_, b, bs, o32, out, R.stream())
    torch.cuda.synchronize()
    for e in range(E):
        if off[e] == off[e + 1]:
            assert (out[e] == 0).all()
            continue
        x, y = av[:, off[e]:off[e + 1]].contiguous(), bv[:, off[e]:off[e + 1]].contiguous()
        check_product(out[e], x @ y.t().contiguous(), x.abs() @ y.abs().t().contiguous(), off[e + 1] - off[e], code)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_nan_rows_stay_their_own(m):
    """A NaN in a row of A or B makes that row or column of the product NaN, with ReLU too, and no other."""
    g = R.gen(9)
    n, k = 200, 700
    x, w = R.randn(g, m, k), R.randn(g, n, k)
    x[m // 2, 300] = math.inf
    w[77, 5] = math.nan
    a, as_, _, _ = R.run_quantize(x)
    b, bs, _, _ = R.run_quantize(w)
    out = torch.empty(m, n, device="cuda")
    R.launch("launchFp8Product", C.byref(option(m, n, k, rows_b=1, act=1)), a, as_, b, bs, None, out, R.stream())
    torch.cuda.synchronize()
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[m // 2], want[:, 77] = True, True
    assert torch.equal(out.isnan(), want)


@pytest.mark.parametrize("m,n,k", [(1, 640, 4000), (40, 200, 3000), (500, 700, 600)])
def test_repeats_and_other_streams(m, n, k):
    """The same bits from every call, also on a stream of its own behind the inputs' stream."""
    g = R.gen(2)
    a, as_, _ = R.make_fp8(g, m, k)
    b, bs, _ = R.make_fp8(g, n, k, 128)
    outs = []
    side = torch.cuda.Stream()
    for i in range(4):
        out = torch.full((m, n), 3.0, device="cuda")
        s = side if i % 2 else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        R.launch("launchFp8Product", C.byref(option(m, n, k)), a, as_, b, bs, None, out, s.cuda_stream)
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
