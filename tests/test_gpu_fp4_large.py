"""4-bit products of sizes that go into persistent tiles of 256 x 256, or into more tiles of 128 x 128 than are worked on at
once, against 64-bit sums (include/experts_abi.h).  What form a call takes goes by its sizes; those here are well within
the range of the form that they are named for."""
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from test_gpu_fp4 import product  # noqa: E402

pytestmark = pytest.mark.gpu

# tiles of 256: several rounds of them, or one; tiles of 128 in several rounds.  Whole and ragged rows, columns and blocks of k
T256 = [(8191, 5120, 300), (8192, 5120, 512), (5000, 5000, 700), (9000, 1025, 129), (3000, 3100, 2100)]
T128 = [(6900, 2550, 513), (4099, 8200, 160), (2500, 9000, 1000)]


def check(out, a, b, k, code, relu=False):
    """Some rows at a time."""
    for lo in range(0, a.shape[0], 4096):
        x = a[lo:lo + 4096]
        ref, mag = x @ b.t(), x.abs() @ b.abs().t()
        bound = S.product_bound(k, mag, ref, code)
        fine = (ref.abs() < 60000) | (code != 1)  # beyond, fp16 has no number
        ref = ref.clamp(min=0) if relu else ref
        off = (out[lo:lo + 4096].double() - ref).abs()
        assert bool((off.le(bound) | ~fine).all()), (code, lo, float((off / bound)[fine].max()))


@pytest.mark.parametrize("m,n,k", T256 + T128)
def test_dense(m, n, k):
    g = R.gen(m + n + k)
    q, s, a = S.make_fp4(g, m, k)
    w, ws, b = S.make_fp4(g, n, k)
    for code in (0, 1, 2):
        out = product(q, s, w, ws, m, n, k, code)
        check(out, a, b, k, code)
        assert torch.equal(out, product(q, s, w, ws, m, n, k, code))  # the same bits again


@pytest.mark.parametrize("m,n,k,stride,shift", [
    (8191, 5120, 300, 5136, 8), (9000, 1025, 129, 1025, 0), (9000, 1025, 129, 1031, 3), (5000, 5000, 260, 5001, 0),
    (6900, 2550, 513, 2560, 16), (4099, 8200, 160, 8203, 1)])
def test_strided_results_and_relu(m, n, k, stride, shift):
    """Rows that 16-byte stores can reach and others; what lies between them and around stays."""
    g = R.gen(m + stride)
    q, s, a = S.make_fp4(g, m, k)
    w, ws, b = S.make_fp4(g, n, k)
    for code in (0, 2):
        buf = torch.full((shift + m * stride + 9,), -7.0, dtype=S.DT[code], device="cuda")
        out = buf[shift:shift + m * stride].view(m, stride)
        product(q, s, w, ws, m, n, k, code, relu=True, stride=stride, out=out)
        check(out[:, :n], a, b, k, code, relu=True)
        assert bool((out[:, n:] == -7).all()) and bool((buf[:shift] == -7).all()) and bool((buf[-9:] == -7).all())


@pytest.mark.parametrize("m,n,k", [T256[0], T256[2], T128[0]])
def test_not_finite(m, n, k):
    """Blocks of NaN in the first, a middle and the last row, column and block of k: theirs and no other results."""
    g = R.gen(7)
    x, y = R.randn(g, m, k), R.randn(g, n, k)
    rows, cols = [0, m // 2 + 1, m - 1], [0, n // 2 + 3, n - 1]
    for r, c, at in zip(rows, cols, (0, k // 2, k - 1)):
        x[r, at], y[c, k - 1 - at] = math.nan, math.inf
    out = product(*S.run_quantize4(x), *S.run_quantize4(y), m, n, k, 2, relu=True)
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[rows], want[:, cols] = True, True
    assert torch.equal(out.isnan(), want)


def spread(total, experts, seed):
    """Rows of each expert: some none, some few, some many; `total` in all."""
    g = torch.Generator()
    g.manual_seed(seed)
    share = torch.rand(experts, generator=g, dtype=torch.float64) ** 2 + 1e-3
    share[torch.randperm(experts, generator=g)[:experts // 8]] = 0
    rows = (share / share.sum() * total).long()
    rows[int(rows.argmax())] += total - int(rows.sum())
    return rows.tolist()


ROWS = {  # rows of each expert, n, k
    "256 of 8": ([16384, 0, 20000, 1, 9001, 255, 257, 15000], 2050, 300),
    "256 of 5": ([8000, 8192, 7999, 8001, 8200], 1000, 640),
    "256 of 64": (spread(96000, 64, 1), 1270, 150),
    "256 of 66": (spread(60000, 66, 2), 700, 290),
    "256 of 80": (spread(120000, 80, 3), 1030, 128),
    "128 of 16": (spread(50000, 16, 4), 520, 520),
    "128 of 65": (spread(20000, 65, 5), 1300, 260),
    "128 of 100": (spread(70000, 100, 6), 777, 140),
}


@pytest.mark.parametrize("name", ROWS)
def test_rows_by_expert(name):
    """Segments that end inside tiles, one behind the other; rows outside all of them stay as they are."""
    rows, n, k = ROWS[name]
    front, behind = 3, 100
    E, m = len(rows), front + sum(rows) + behind
    g = R.gen(E * 10 + n)
    offsets = torch.tensor([front + sum(rows[:i]) for i in range(E + 1)], dtype=torch.int32, device="cuda")
    q, s, a = S.make_fp4(g, m, k)
    parts = [S.make_fp4(g, n, k) for _ in range(E)]
    w, ws, b = (torch.stack(p).contiguous() for p in zip(*parts))
    at = offsets.tolist()
    for code in (0, 1, 2):
        out = product(q, s, w, ws, m, n, k, code, E, offsets)
        for e in range(E):
            check(out[at[e]:at[e + 1]], a[at[e]:at[e + 1]], b[e], k, code)
        assert bool((out[:front] == -7).all()) and bool((out[at[E]:] == -7).all())


@pytest.mark.parametrize("E,m,n", [(8, 60000, 2050), (66, 60000, 700)])
def test_offsets_out_of_range(E, m, n):
    """Offsets are held within the rows: nothing outside is read or written."""
    k = 200
    g = R.gen(E)
    q, s, a = S.make_fp4(g, m, k)
    parts = [S.make_fp4(g, n, k) for _ in range(E)]
    w, ws, b = (torch.stack(p).contiguous() for p in zip(*parts))
    lo = [m * e // E for e in range(E)]
    offsets = torch.tensor([-9] + lo[1:] + [1 << 30], dtype=torch.int32, device="cuda")
    offsets[3] = lo[4] + 700  # the third expert's go on into the fifth's, the fourth has none
    buf = torch.full((m + 40, n), -7.0, device="cuda")
    product(q, s, w, ws, m, n, k, 0, E, offsets, out=buf[20:20 + m])
    assert bool((buf[:20] == -7).all()) and bool((buf[20 + m:] == -7).all())
    for e in range(E):
        begin, end = (lo[4] + 700 if e == 4 else lo[e]), (lo[e + 1] if e + 1 < E else m)  # without the rows that are two experts'
        expert = 2 if e == 3 else e
        check(buf[20 + begin:20 + end], a[begin:end], b[expert], k, 0)
