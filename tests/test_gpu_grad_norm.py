"""The gradients' norm and its clipping (include/grad_abi.h) against 64-bit arithmetic."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def norm(data, kind=0, scale=1.0):
    out = torch.full((1,), -1.0, device="cuda")
    R.launch("launchGradNorm", S.tensors(data), len(data), kind, scale, out, R.stream())
    return out


def make(sizes, codes, seed=0, shift=0):
    """Tensors of these sizes, types in turn, each of another magnitude, `shift` elements off an allocation's start."""
    g = R.gen(seed)
    out = []
    for i, n in enumerate(sizes):
        t = torch.zeros(n + shift, device="cuda", dtype=S.DT[codes[i % len(codes)]])[shift:]
        t.copy_(R.randn(g, n) * 2.0 ** (i % 7 - 3))
        out.append(t)
    return out


LISTS = [[1], [0, 5, 0], [7, 1, 64], [4096, 4097, 8191], [100000, 3, 65537, 1, 12345], [(i * 37) % 301 for i in range(700)],
         [2_000_003, 1, 1 << 20]]


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("codes", [[0], [1], [2], [0, 1, 2]])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: str(len(s)) + "x" + str(max(s)))
def test_norms(sizes, codes, shift):
    data = make(sizes, codes, len(sizes), shift)
    for kind in (0, 1):
        want = S.norm64(data, kind, 128.0)
        got = float(norm(data, kind, 128.0))
        # one rounding to fp32 of a 64-bit result
        assert abs(got - want) <= (UNIT + 1e-12) * want, kind


def clip(data, out, max_norm, kind=0, scale=1.0, zero=False, given=None):
    """The norm, after clipping (out None: in place)."""
    t = S.tensors(data, out)
    if given is not None:
        R.launch("launchGradClip", t, len(data), max_norm, int(zero), given, R.stream())
        return given
    n = torch.full((1,), -1.0, device="cuda")
    R.launch("launchGradNormClip", t, len(data), kind, scale, max_norm, int(zero), n, R.stream())
    return n


def check_clipped(before, after, n, max_norm):
    """g times the fp32 factor: that is off by 2^-24, the product by as much, its rounding by the type's."""
    factor = min(1.0, max_norm / n) if n > 0 else 1.0
    for a, b in zip(before, after):
        if factor == 1.0:
            assert torch.equal(a, b)
            continue
        want = a.double() * factor
        bound = (3 * UNIT + S.HALF[S.CODE[a.dtype]]) * want.abs() + S.TINY[S.CODE[a.dtype]]
        assert bool((b.double() - want).abs().le(bound).all())


@pytest.mark.parametrize("over", [0.5, 1.0, 1.5, 1000.0])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: str(len(s)) + "x" + str(max(s)))
def test_clip(sizes, kind, over):
    for place in ("in", "out", "shifted"):
        data = make(sizes, [0, 2, 1], 5, 2 if place == "shifted" else 0)
        before = [t.clone() for t in data]
        n = float(norm(data, kind, 64.0))
        max_norm = float(torch.tensor(n / over, dtype=torch.float32))
        out = None
        if place != "in":
            out = [torch.full((t.numel() + 9,), -3.0, dtype=t.dtype, device="cuda") for t in data]
        views = None if out is None else [o[(1 if place == "shifted" else 0):][:t.numel()] for o, t in zip(out, data)]
        got = clip(data, views, max_norm, kind, 64.0)
        assert float(got) == n
        if n > 0:
            check_clipped(before, data if out is None else views, n, max_norm)
        if out is not None:  # inputs and what lies around the outputs are as they were
            assert all(torch.equal(a, b) for a, b in zip(before, data))
            for o, v in zip(out, views):
                first = v.storage_offset()
                assert bool((o[:first] == -3).all()) and bool((o[first + v.numel():] == -3).all())


def test_parts_of_a_buffer_side_by_side():
    """Tensors that follow each other without a gap, of odd lengths, each clipped within its own elements."""
    for code in (0, 1, 2):
        sizes = [1, 3, 5, 16, 7, 4099, 2, 8190, 31]
        flat = R.randn(R.gen(1), sum(sizes) + 6).to(S.DT[code])
        before = flat.clone()
        views, at = [], 3
        for s in sizes:
            views.append(flat[at:at + s])
            at += s
        n = float(clip(views, None, 0.25))
        assert abs(n - S.norm64([before[3:at]], 0, 1.0)) <= 2 * UNIT * n
        check_clipped([before[3:at]], [flat[3:at]], n, 0.25)
        assert torch.equal(flat[:3], before[:3]) and torch.equal(flat[at:], before[at:])


@pytest.mark.parametrize("big", [1e30, 3e38, 1e-30, 2.0 ** -149])
def test_squares_neither_overflow_nor_vanish(big):
    data = [torch.full((1000,), big, device="cuda"), torch.full((24,), -big, device="cuda")]
    want = S.norm64(data, 0, 1.0)
    got = float(norm(data))
    if want > torch.finfo(torch.float32).max:
        assert got == math.inf
    else:
        assert abs(got - want) <= UNIT * want + 2.0 ** -150
    assert abs(float(norm(data, 0, 1e6)) - want / 1e6) <= UNIT * want / 1e6 + 2.0 ** -150


def test_nothing():
    assert float(norm([])) == 0.0
    empty = [torch.empty(0, device="cuda")] * 3
    for kind in (0, 1):
        assert float(norm(empty, kind)) == 0.0
    assert float(clip(empty, None, 1.0)) == 0.0
    zeros = [torch.zeros(100, device="cuda")]
    for m in (0.0, 1.0):
        assert float(clip(zeros, None, m)) == 0.0 and not bool(zeros[0].any())
    data = make([50, 9], [0, 2])
    clip(data, None, 0.0)
    assert not any(bool(t.any()) for t in data)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("size", [40, 200_000])
def test_not_finite(bad, kind, size):
    for code in (0, 1, 2):
        data = make([5, size, 300], [code])
        data[1][size // 2] = bad
        before = [t.clone() for t in data]
        n = float(norm(data, kind))
        assert math.isnan(n) if math.isnan(bad) else n == math.inf
        out = [torch.full_like(t, 9) for t in data]
        for where in (None, out):
            clip(data, where, 1.0, kind)
            for a, b in zip(before, where or data):
                assert torch.equal(a.nan_to_num(7), b.nan_to_num(7)) and torch.equal(a.isnan(), b.isnan())
        clip(data, out, 1.0, kind, zero=True)
        assert not any(bool(t.any()) for t in out)
        clip(data, None, 1.0, kind, zero=True)
        assert not any(bool(t.any()) for t in data)


def test_a_given_norm():
    """As ranks use it that hold parts of the gradients: the norm of all comes from theirs."""
    parts = [make([1000, 77], [0, 2], s) for s in (1, 2)]
    norms = torch.cat([norm(p) for p in parts])
    whole = torch.sqrt(norms.square().sum()).view(1)
    assert abs(float(whole) - S.norm64(parts[0] + parts[1], 0, 1.0)) <= 4 * UNIT * float(whole)
    for p in parts:
        before = [t.clone() for t in p]
        clip(p, None, 0.5, given=whole)
        check_clipped(before, p, float(whole), 0.5)
    for bad in (math.inf, math.nan):
        data = make([30], [0])
        before = data[0].clone()
        clip(data, None, 0.5, given=torch.tensor([bad], device="cuda"))
        assert torch.equal(before, data[0])


def test_same_bits_and_same_input_twice():
    data = make([300_001, 5, 70_000], [2, 0, 1])
    first = norm(data)
    assert all(torch.equal(first, norm(data)) for _ in range(3))
    twice = [data[0], data[0]]  # read twice, written apart
    out = [torch.empty_like(data[0]) for _ in range(2)]
    n = float(clip(twice, out, 1.0))
    assert abs(n - S.norm64(twice, 0, 1.0)) <= 2 * UNIT * n
    assert torch.equal(out[0], out[1])


def test_graph():
    """Captured, replayed on new gradients; an eager call of another list between the replays."""
    s = torch.cuda.Stream()
    for sizes in ([100, 7], [300_000, 11]):
        data = make(sizes, [0, 1])
        other = make([5000] * 200, [2])
        n = torch.zeros(1, device="cuda")
        t, keep = S.tensors(data), [d.clone() for d in data]
        torch.cuda.synchronize()

        def call():
            R.launch("launchGradNormClip", t, len(data), 0, 1.0, 2.0, 0, n, torch.cuda.current_stream().cuda_stream)

        with torch.cuda.stream(s):
            call()
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call()
        for i in range(4):
            for d, k in zip(data, keep):
                d.copy_(k * 2.0 ** i)
            torch.cuda.synchronize()
            want = S.norm64(data, 0, 1.0)
            before = [d.clone() for d in data]
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                graph.replay()
                R.launch("launchGradNorm", S.tensors(other), len(other), 0, 1.0, torch.empty(1, device="cuda"), s.cuda_stream)
            s.synchronize()
            assert abs(float(n) - want) <= 2 * UNIT * want
            check_clipped(before, data, float(n), 2.0)


def test_far_elements():
    """A tensor beyond 2^32 bytes and 2^31 elements of 16 bits."""
    t = torch.zeros((1 << 31) + 77, dtype=torch.bfloat16, device="cuda")
    t[-1], t[1 << 31], t[5] = 3.0, 4.0, 12.0
    assert float(norm([t])) == 13.0
    n = clip([t], None, 6.5)
    assert float(n) == 13.0 and [float(t[i]) for i in (-1, 1 << 31, 5, 0)] == [1.5, 2.0, 6.0, 0.0]
