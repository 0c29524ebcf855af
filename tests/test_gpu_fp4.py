"""4-bit matrices (include/experts_abi.h): quantising bit for bit against 64-bit arithmetic, products against 64-bit sums."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


def check_quantized(x, q, s, rule, want_rows=None):
    x = x if want_rows is None else want_rows
    cols = x.shape[1]
    want, byte = S.quantize4(x, rule)
    assert torch.equal(s, byte)
    got = S.codes4(q, q.shape[1] * 2)
    assert torch.equal(got[:, :cols], want)
    assert not bool(q.view(x.shape[0], -1)[:, (cols + 1) // 2:].any())
    assert not bool(got[:, cols:].any())


@pytest.mark.parametrize("rule", [0, 1])
@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("rows,cols,pad,shift", [(1, 1, 0, 0), (3, 31, 2, 1), (5, 32, 0, 0), (2, 33, 7, 3), (7, 128, 8, 0),
                                                (4, 136, 0, 0), (33, 300, 4, 0), (130, 1000, 24, 8), (257, 257, 0, 0)])
def test_quantize(rows, cols, pad, shift, code, rule):
    g = R.gen(rows * 1000 + cols)
    x = R.randn(g, rows, cols) * torch.exp2(torch.randint(-20, 13, (rows, 1), generator=g, device="cuda").float())
    x = R.strided(x.to(S.DT[code]), pad, shift)
    check_quantized(x, *S.run_quantize4(x, rule), rule)


@pytest.mark.parametrize("rule", [0, 1])
def test_quantize_borders(rule):
    """Every tie and its neighbours at scales from the least to the largest, blocks of zeros, subnormal numbers, the largest
    magnitudes at and around the borders of a scale."""
    v = [0.0, -0.0]
    for a, b in zip(S.GRID, S.GRID[1:]):
        m = (a + b) / 2
        v += [m, -m, m * (1 + 2.0 ** -23), m * (1 - 2.0 ** -24), a, b]
    v += [7.0, 7.9]
    block = torch.tensor(v[:31] + [6.0], dtype=torch.float64)
    rest = torch.tensor((v[31:] + [0.0] * 32)[:31] + [4.0], dtype=torch.float64)
    rows = []
    for e in (-126, -125, -30, 0, 1, 50, 119):
        for top in (4.0, 5.0, 6.0, 6.0 * (1 + 2.0 ** -23), 7.75, 8.0 * (1 - 2.0 ** -24), 8.0):
            r = torch.cat([block, rest]) * 2.0 ** e
            r[31] = r[63] = top * 2.0 ** e
            rows.append(r)
    rows.append(torch.zeros(64, dtype=torch.float64))
    rows.append(torch.full((64,), 2.0 ** -149, dtype=torch.float64))
    rows.append(torch.full((64,), 2.0 ** -127, dtype=torch.float64))
    rows.append(torch.full((64,), torch.finfo(torch.float32).max, dtype=torch.float64))
    x = torch.stack(rows).float().cuda()
    check_quantized(x, *S.run_quantize4(x, rule), rule)


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("rule", [0, 1])
def test_quantize_not_finite(code, rule):
    """A block with an infinity or a NaN is one of NaN, its neighbours are not."""
    x = R.randn(R.gen(3), 6, 200).to(S.DT[code])
    x[1, 40], x[2, 64], x[3, 199], x[4, 0] = math.inf, -math.inf, math.nan, math.nan
    q, s = S.run_quantize4(x, rule)
    check_quantized(x, q, s, rule)
    assert [(int(r), int(c)) for r, c in (s == 255).nonzero()] == [(1, 1), (2, 2), (3, 6), (4, 0)]


@pytest.mark.parametrize("code", [0, 2])
def test_gather(code):
    g = R.gen(8)
    x = R.strided(R.randn(g, 40, 264).to(S.DT[code]), 8)
    order = torch.randint(-1, 130, (300,), generator=g, device="cuda").int()  # slots of rows beyond the last among them
    q, s = S.run_quantize4(x, 0, order, 3, 300)
    row = (order // 3).long()
    there = (order >= 0) & (row < 40)
    want = torch.where(there[:, None], x[row.clamp(0, 39)].float(), 0.0)
    check_quantized(x, q, s, 0, want)


def test_batches():
    P, g = pkg(), R.gen(9)
    x = R.randn(g, 3, 5, 96).bfloat16()
    o = P.Fp4QuantOption(rows=5, cols=90, batch=3, scaleRule=1, srcType=2, slotsPerRow=1, srcRows=5, srcStride=96,
                         srcBatchStride=480)
    q = torch.full((3, 5, P.fp4_pitch(90)), 0xAA, dtype=torch.uint8, device="cuda")
    s = torch.full((3, 5, P.fp4_scale_pitch(90)), 0xAA, dtype=torch.uint8, device="cuda")
    R.launch("launchFp4Quantize", C.byref(o), x, None, q, s, R.stream())
    for b in range(3):
        check_quantized(x[b, :, :90].contiguous(), q[b], s[b], 1)


def test_beyond_one_launch():
    """More blocks than a launch of 2^32 threads has: rows of 128 columns, 16 threads each."""
    rows = (1 << 28) + 5
    x = torch.zeros(2, 128, device="cuda", dtype=torch.bfloat16)
    x[1] = 3.0
    order = torch.zeros(rows, dtype=torch.int32, device="cuda")
    order[-3:] = 1
    order[(1 << 28) - 2:(1 << 28) + 1] = 1
    P = pkg()
    q = torch.empty(rows, 64, dtype=torch.uint8, device="cuda")
    s = torch.empty(rows, 4, dtype=torch.uint8, device="cuda")
    o = P.Fp4QuantOption(rows=rows, cols=128, batch=1, scaleRule=0, srcType=2, slotsPerRow=1, srcRows=2, srcStride=128,
                         srcBatchStride=0)
    R.launch("launchFp4Quantize", C.byref(o), x, order, q, s, R.stream())
    want = order != 0
    for lo in range(0, rows, 1 << 26):
        w, b = want[lo:lo + (1 << 26)], q[lo:lo + (1 << 26)]
        assert bool(((b == 0x77).all(1) == w).all()) and bool(((b == 0).all(1) != w).all())
        assert bool((s[lo:lo + (1 << 26), 0] == torch.where(w, 126, 1)).all())


def product(q, s, w, ws, m, n, k, code, experts=1, offsets=None, relu=False, stride=None, out=None):
    P = pkg()
    stride = stride or n
    out = torch.full((max(m, 1), stride), -7.0, dtype=S.DT[code], device="cuda") if out is None else out
    o = P.Fp4ProductOption(m=m, n=n, k=k, numExperts=experts, grouping=0 if offsets is None else 1, activation=int(relu),
                           outType=code, outStride=stride)
    R.launch("launchFp4Product", C.byref(o), q, s, w, ws, offsets, out, R.stream())
    return out


SIZES = [(1, 1, 1), (1, 17, 33), (2, 64, 128), (5, 100, 200), (16, 16, 384), (17, 130, 640), (33, 257, 1000), (64, 300, 129),
         (65, 128, 256), (128, 128, 4096), (130, 520, 896), (257, 255, 513), (300, 1000, 2100), (1000, 384, 160), (513, 2049, 777)]


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_dense(m, n, k, code):
    g = R.gen(m * 7 + n * 3 + k)
    q, s, a = S.make_fp4(g, m, k)
    w, ws, b = S.make_fp4(g, n, k)
    out = product(q, s, w, ws, m, n, k, code)
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    fine = (ref.abs() < 60000) | (code != 1)  # beyond, fp16 has no number
    assert bool((out.double() - ref).abs()[fine].le(S.product_bound(k, mag, ref, code)[fine]).all())
    assert torch.equal(out, product(q, s, w, ws, m, n, k, code))  # the same bits again


@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (70, 200, 300), (700, 700, 1024)])
def test_large_products_that_cancel(m, n, k):
    """Blocks of 2^12 beside blocks of 2^-12, the large ones in pairs that cancel: what is small is left, to fp32's last bits
    of the largest."""
    g = R.gen(5)
    x = R.randn(g, m, k)
    x[:, 0:32] = 4096.0 * torch.sign(x[:, 0:32])
    x[:, 32:64] = -x[:, 0:32]
    x[:, 64:] *= 2.0 ** -12
    y = R.randn(g, n, k)
    y[:, 32:64] = y[:, 0:32]
    q, s = S.run_quantize4(x, 1)
    w, ws = S.run_quantize4(y, 1)
    a, b = S.values4(q, s, k), S.values4(w, ws, k)
    assert torch.equal(a[:, 0:32], -a[:, 32:64]) and torch.equal(b[:, 0:32], b[:, 32:64])
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    out = product(q, s, w, ws, m, n, k, 0)
    assert bool((out.double() - ref).abs().le(S.product_bound(k, mag, ref, 0)).all())


@pytest.mark.parametrize("stride,shift", [(130, 0), (131, 0), (136, 1), (136, 8), (2048, 0)])
@pytest.mark.parametrize("m,n", [(9, 129), (300, 129)])
def test_strided_results_and_relu(m, n, stride, shift):
    g = R.gen(12)
    q, s, a = S.make_fp4(g, m, 192)
    w, ws, b = S.make_fp4(g, n, 192)
    for code in (0, 2):
        buf = torch.full((shift + m * stride,), -7.0, dtype=S.DT[code], device="cuda")
        out = buf[shift:].view(m, stride)
        product(q, s, w, ws, m, n, 192, code, relu=True, stride=stride, out=out)
        ref, mag = a @ b.t(), a.abs() @ b.abs().t()
        bound = S.product_bound(192, mag, ref, code)
        assert bool((out[:, :n].double() - ref.clamp(min=0)).abs().le(bound).all())
        assert bool((out[:, n:] == -7).all()) and bool((buf[:shift] == -7).all())


def test_not_finite():
    """A block of NaN makes its row's, or its column's, results NaN and no others; ReLU keeps them."""
    g = R.gen(13)
    for m, n, k in ((4, 40, 300), (400, 300, 700)):
        x, y = R.randn(g, m, k), R.randn(g, n, k)
        x[1, 5], y[7, k - 1] = math.nan, math.inf
        out = product(*S.run_quantize4(x), *S.run_quantize4(y), m, n, k, 2, relu=True)
        want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        want[1], want[:, 7] = True, True
        assert torch.equal(out.isnan(), want)


def test_scales_at_the_ends():
    """Products beyond fp32 are infinite, tiny ones as exact as fp32 is."""
    k = 128
    big, small = torch.full((2, k), 3.0 * 2.0 ** 120), torch.full((2, k), 2.0 ** -126)
    for x, y, want in ((big, big, math.inf), (small, torch.full((2, k), 2.0 ** -20), k * 2.0 ** -146),
                       (small, torch.full((2, k), 3.0 * 2.0 ** 120), 3 * k * 2.0 ** -6)):
        out = product(*S.run_quantize4(x.cuda(), 1), *S.run_quantize4(y.cuda(), 1), 2, 2, k, 0)
        assert out.tolist() == [[want] * 2] * 2


ROWS = [  # rows of each expert, rows behind the last
    ([1], 0), ([0, 3, 0], 2), ([16, 1, 17, 0, 31], 0), ([128, 128], 128), ([5, 200, 0, 300], 1),
    ([1] * 40, 3), ([3, 0] * 50, 0), ([600, 1, 259], 5), ([0, 0], 4)]


@pytest.mark.parametrize("n,k", [(33, 100), (300, 1300)])
@pytest.mark.parametrize("rows,behind", ROWS)
def test_rows_by_expert(rows, behind, n, k):
    """Segments of any length; rows outside all of them stay as they are."""
    g = R.gen(sum(rows) + n)
    E, front = len(rows), 2
    m = front + sum(rows) + behind
    offsets = torch.tensor([front + sum(rows[:i]) for i in range(E + 1)], dtype=torch.int32, device="cuda")
    q, s, a = S.make_fp4(g, m, k)
    parts = [S.make_fp4(g, n, k) for _ in range(E)]
    w, ws, b = (torch.stack(p).contiguous() for p in zip(*parts))
    for code in (0, 1, 2):
        out = product(q, s, w, ws, m, n, k, code, E, offsets)
        for e in range(E):
            lo, hi = int(offsets[e]), int(offsets[e + 1])
            ref, mag = a[lo:hi] @ b[e].t(), a[lo:hi].abs() @ b[e].abs().t()
            fine = ref.abs() < 60000
            bound = S.product_bound(k, mag, ref, code)
            assert bool((out[lo:hi].double() - ref).abs()[fine].le(bound[fine]).all()), (code, e)
        assert bool((out[:front] == -7).all()) and bool((out[front + sum(rows):] == -7).all())


def test_offsets_out_of_range():
    """Offsets are held within the rows: nothing outside is read or written."""
    g = R.gen(77)
    q, s, a = S.make_fp4(g, 20, 256)
    w, ws, _ = S.make_fp4(g, 3 * 32, 256)
    offsets = torch.tensor([-5, 7, 3, 400], dtype=torch.int32, device="cuda")
    buf = torch.full((60, 32), -7.0, device="cuda")
    product(q, s, w, ws, 20, 32, 256, 0, 3, offsets, out=buf[20:40])
    assert bool((buf[:20] == -7).all()) and bool((buf[40:] == -7).all())
    # the first expert's rows are 0..6, the second's 7 has none (7..3), the third's 3..19: rows 3..6 are two experts'
    b = S.values4(w, ws, 256).view(3, 32, 256)
    for lo, hi, e in ((0, 3, 0), (7, 20, 2)):
        ref, mag = a[lo:hi] @ b[e].t(), a[lo:hi].abs() @ b[e].abs().t()
        assert bool((buf[20 + lo:20 + hi].double() - ref).abs().le(S.product_bound(256, mag, ref, 0)).all())


def test_another_stream_and_graph():
    g = R.gen(21)
    x = R.randn(g, 300, 512).half()
    w, ws, b = S.make_fp4(g, 256, 512)
    P = pkg()
    st = torch.cuda.Stream()
    q = torch.empty(300, P.fp4_pitch(512), dtype=torch.uint8, device="cuda")
    s = torch.empty(300, P.fp4_scale_pitch(512), dtype=torch.uint8, device="cuda")
    out = torch.zeros(300, 256, dtype=torch.float16, device="cuda")
    qo = P.Fp4QuantOption(rows=300, cols=512, batch=1, scaleRule=0, srcType=1, slotsPerRow=1, srcRows=300, srcStride=512,
                          srcBatchStride=0)
    po = P.Fp4ProductOption(m=300, n=256, k=512, numExperts=1, grouping=0, activation=0, outType=1, outStride=256)

    def call():
        h = torch.cuda.current_stream().cuda_stream
        R.launch("launchFp4Quantize", C.byref(qo), x, None, q, s, h)
        R.launch("launchFp4Product", C.byref(po), q, s, w, ws, None, out, h)

    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        call()
        st.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        st.synchronize()
        with torch.cuda.graph(graph, stream=st):
            call()
    for i in range(4):
        x.copy_(x.roll(1, 0))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want.roll(i + 1, 0))
