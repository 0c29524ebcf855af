"""The layer of experts for few tokens (include/experts_abi.h) against 64-bit arithmetic, expert by expert."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


class Layer:
    """Weights, tokens and the call; routes that do not hang on a score's last bits."""

    def __init__(self, T, E, k, D, H, act=1, gated=False, fmt=0, scale_rows=128, code=0, router=0, bias=False, seed=0, pad_x=0,
                 pad_o=0, shift=0, **route):
        g = R.gen(seed * 131 + T * 7 + D)
        self.size = (T, E, k, D, H, act, gated, code)
        make = S.weights4 if fmt else S.weights8
        scale_rows = 1 if fmt else scale_rows
        self.w1 = make(g, E, H * (2 if gated else 1), D, scale_rows)
        self.w2 = make(g, E, D, H, scale_rows)
        self.router = (R.randn(g, E, D) * 1.5 / math.sqrt(D)).to(S.DT[router])
        self.bias = R.randn(g, E) * 0.1 if bias else None
        self.route = dict(sigmoid=route.get("scoreType", 0) == 1, groups=route.get("numGroups", 1),
                          kept=route.get("topGroups", 1), group_best=route.get("groupScore", 2),
                          renorm=bool(route.get("renormalize", 1)), scale=route.get("scale", 1.0))
        x = R.randn(g, T, D).to(S.DT[code])
        for _ in range(20):
            self.indices, self.weights, gap = self.routes(x)
            if gap > 1e-4:
                break
            x = R.randn(g, T, D).to(S.DT[code])
        else:
            self.indices, self.weights, _ = self.routes(x)
        self.x = R.strided(x, pad_x, shift)
        self.buf = torch.full((shift + T * (D + pad_o) + 5,), -7.0, dtype=S.DT[code], device="cuda")
        self.out = self.buf[shift:shift + T * (D + pad_o)].view(T, D + pad_o)
        self.o = S.layer_option(E, k, D, H, act, gated, fmt, scale_rows, code, router, D + pad_x, D + pad_o, **route)

    def routes(self, x):
        z = x.double() @ self.router.double().t()
        r = self.route
        return R.route(z, self.bias, self.size[2], r["sigmoid"], r["groups"], r["kept"], r["group_best"], r["renorm"], r["scale"])

    def run(self, stream=None, tokens=None):
        R.launch("launchExpertLayer", C.byref(self.o), self.x, self.router, self.bias, self.w1[0], self.w1[1], self.w2[0],
                 self.w2[1], self.out, self.size[0] if tokens is None else tokens, R.stream() if stream is None else stream)
        return self.out[:, :self.size[3]]

    def check(self, got=None):
        T, E, k, D, H, act, gated, code = self.size
        want, bound = S.layer(self.x, self.indices, self.weights, self.w1[2], self.w2[2], H, act, gated, code)
        # the routing weights come from fp32 logits: their errors, a few units of their sums of D products, count for the whole
        dz = float(((D / 8 + 16) * 2.0 ** -24 * (self.x.double().abs() @ self.router.double().abs().t())).max())
        got = self.run() if got is None else got
        off = (got.double() - want).abs()
        share = (4 * dz + 16 * 2.0 ** -24) * self.magnitude()
        assert bool(off.le(bound + share).all()), float((off / (bound + share)).max())

    def magnitude(self):
        """sum_j |w_j W2 a_j|, by which an error of the routing weights counts."""
        T, E, k, D, H, act, gated, code = self.size
        parts = [S.layer(self.x, self.indices[:, j:j + 1], self.weights[:, j:j + 1], self.w1[2], self.w2[2], H, act, gated,
                         code)[0].abs() for j in range(k)]
        return sum(parts)


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("fmt,scale_rows", [(0, 128), (0, 1), (1, 1)])
@pytest.mark.parametrize("T,E,k,D,H", [(1, 1, 1, 1, 1), (1, 8, 2, 64, 96), (2, 4, 4, 129, 33), (5, 6, 1, 300, 200),
                                       (16, 3, 2, 128, 256), (17, 8, 3, 200, 130), (33, 5, 2, 260, 72), (64, 4, 2, 136, 140)])
def test_sizes_and_types(T, E, k, D, H, fmt, scale_rows, code):
    Layer(T, E, k, D, H, act=T % 4, gated=T % 2 == 0, fmt=fmt, scale_rows=scale_rows, code=code, router=(code + T) % 3).check()


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fmt", [0, 1])
def test_activations(act, gated, fmt):
    Layer(6, 5, 2, 192, 256, act=act, gated=gated, fmt=fmt, code=act % 3, seed=2).check()


@pytest.mark.parametrize("T,E,k,route", [
    (9, 60, 6, dict(scoreType=1, scale=2.5)), (9, 64, 8, dict(numGroups=8, topGroups=4, scoreType=1)),
    (7, 32, 4, dict(numGroups=4, topGroups=2, groupScore=1, renormalize=0)), (3, 200, 32, dict(renormalize=0, scale=0.5)),
    (64, 96, 4, {}), (20, 1024, 2, dict(scoreType=1))])
def test_routes(T, E, k, route):
    for bias in (False, True):
        Layer(T, E, k, 64, 40, act=2, gated=True, fmt=1, code=2, bias=bias, seed=3, **route).check()


@pytest.mark.parametrize("T,E,k,route", [
    (16, 1024, 4, dict(numGroups=8, topGroups=4, scoreType=1)), (64, 1024, 32, dict(numGroups=64, topGroups=9, groupScore=1)),
    (40, 512, 20, dict(numGroups=64, topGroups=32)), (64, 300, 2, {}), (64, 1024, 1, dict(scoreType=1)),
    (6, 64, 24, {}), (11, 64, 3, dict(numGroups=32, topGroups=7)), (13, 128, 6, dict(numGroups=64, topGroups=20, groupScore=1)),
    (64, 8, 8, {}), (1, 1024, 32, dict(numGroups=2, topGroups=1))])
def test_routes_of_many_experts_groups_and_picks(T, E, k, route):
    """Every width of a token's lanes; logits that have room beside scores and keys in LDS, and such as have not."""
    Layer(T, E, k, 160, 24, fmt=1, code=1, router=1, seed=12, **route).check()


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("pad_x,pad_o,shift", [(1, 3, 0), (8, 8, 8), (0, 0, 1), (24, 5, 3)])
def test_strides(pad_x, pad_o, shift, code):
    """Rows of any distance and start; nothing between and around them is written."""
    L = Layer(11, 4, 2, 200, 64, code=code, pad_x=pad_x, pad_o=pad_o, shift=shift)
    L.check()
    assert bool((L.out[:, 200:] == -7).all()) and bool((L.buf[:shift] == -7).all()) and bool((L.buf[-5:] == -7).all())


@pytest.mark.parametrize("T", [1, 16, 40])
def test_a_longer_layer(T):
    """Sizes at which the experts' k is shared out among many waves and workgroups."""
    for fmt, code in ((0, 2), (1, 0), (1, 1)):
        Layer(T, 8, 2, 2048, 768, act=2, gated=True, fmt=fmt, code=code, seed=4).check()


def test_all_tokens_one_expert():
    """A bias sends every token to the same two experts."""
    for T in (8, 16, 48, 64):
        L = Layer(T, 16, 2, 96, 160, code=2, seed=5)
        L.bias = torch.zeros(16, device="cuda")
        L.bias[3], L.bias[9] = 10.0, 9.0
        L.indices, L.weights, _ = L.routes(L.x)
        assert set(L.indices.flatten().tolist()) == {3, 9}
        L.check()


def test_tokens_without_experts():
    """NaN or minus infinity among a token's logits or in the bias: its experts are those that are left, zeros if none is."""
    L = Layer(5, 4, 3, 64, 64, code=0)
    L.bias = torch.tensor([0.0, -math.inf, math.nan, 0.0], device="cuda")
    L.indices, L.weights, _ = L.routes(L.x)
    assert (L.indices[:, 2] == -1).all()
    L.check()
    L.bias = None
    L.x[2, 5] = math.nan
    L.indices, L.weights, _ = L.routes(L.x)
    got = L.run()
    assert not bool(got[2].any()) and bool(got.isfinite().all())
    L.x[2, 5] = 0.0
    L.indices, L.weights, _ = L.routes(L.x)
    L.check()


def test_nan_weights_reach_their_own_tokens_alone():
    for fmt in (0, 1):
        L = Layer(12, 4, 1, 130, 130, code=2, fmt=fmt, seed=6)
        clean = L.run().clone()
        e = int(L.indices[0, 0])
        hit = (L.indices[:, 0] == e).cuda()
        assert bool(hit.any()) and not bool(hit.all())
        for w in (L.w1, L.w2):
            keep = (w[0].clone(), w[1].clone())
            if fmt:
                w[1][e, 0, 0] = 255
            else:
                w[0][e, 0, 0] = 0x7f
            got = L.run().clone()
            assert bool(got[hit].isnan().any(1).all()) and torch.equal(got[~hit], clean[~hit])
            w[0].copy_(keep[0])
            w[1].copy_(keep[1])
        assert torch.equal(L.run(), clean)


def test_large_hidden_values():
    """Hidden activations beyond fp16's and near bf16's largest numbers."""
    for code in (0, 2):
        L = Layer(4, 2, 1, 64, 64, act=1, code=code, seed=7)
        L.w1[1].copy_((L.w1[1].int() + 100).clamp(max=246).to(torch.uint8))
        L.w2[1].copy_((L.w2[1].int() - 100).clamp(min=17).to(torch.uint8))
        for w, (rows, cols) in ((L.w1, (64, 64)), (L.w2, (64, 64))):
            w[2].copy_(torch.stack([R.values(q, s, cols, 128) for q, s in zip(w[0], w[1])]))
        L.check()


def test_nothing_and_fewer_tokens():
    L = Layer(9, 4, 2, 64, 64, code=1)
    whole = L.run().clone()
    L.out.fill_(-7)
    L.run(tokens=0)
    assert bool((L.out == -7).all())
    L.check(whole)
    for n in (1, 4):  # rows behind the last token stay
        L.out.fill_(-7)
        L.run(tokens=n)
        assert bool((L.out[n:] == -7).all())
        whole[:n] = L.out[:n]
        L.check(whole)


def test_same_bits():
    L = Layer(40, 16, 4, 520, 300, act=2, gated=True, fmt=1, code=2, seed=8)
    first = L.run().clone()
    for _ in range(5):
        assert torch.equal(first, L.run())


def test_streams_and_graphs():
    """Two layers on streams of their own, captured and replayed on new tokens, with larger eager calls between."""
    jobs = [Layer(8, 8, 2, 256, 192, code=2, seed=20), Layer(30, 12, 3, 320, 128, fmt=1, code=1, seed=21)]
    big = Layer(64, 16, 4, 640, 512, code=2, seed=22)
    streams = [torch.cuda.Stream() for _ in jobs]
    tokens = [[j.x.clone(), torch.roll(j.x, 1, 0), torch.roll(j.x, 3, 0)] for j in jobs]
    want = []
    for j, xs in zip(jobs, tokens):
        w = []
        for x in xs:
            j.x.copy_(x)
            w.append(j.run().clone())
        want.append(w)
    torch.cuda.synchronize()
    graphs = []
    for j, s in zip(jobs, streams):
        with torch.cuda.stream(s):
            j.run(s.cuda_stream)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                j.run(s.cuda_stream)
            graphs.append(g)
    for rep in range(6):
        for j, xs in zip(jobs, tokens):
            j.x.copy_(xs[rep % 3])
            j.out.fill_(-7)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                if rep == 2:
                    big.run(s.cuda_stream)
        torch.cuda.synchronize()
        for j, w in zip(jobs, want):
            assert torch.equal(j.out, w[rep % 3]), rep


def test_beside_the_blocks_other_operators():
    """The same weights through routing, gather, 8-bit products and combine: the layer differs by the quantising of the
    tokens and of the hidden values alone (e4m3: 2^-4 of each value at most, 2^-5 in the middle)."""
    P = pkg()
    T, E, k, D, H = 24, 4, 2, 256, 384
    L = Layer(T, E, k, D, H, act=1, code=2, router=0, seed=9)
    z = (L.x.float() @ L.router.t()).contiguous()
    ro = L.o.route
    idx = torch.empty(T, k, dtype=torch.int32, device="cuda")
    wts = torch.empty(T, k, device="cuda")
    R.launch("launchRouteExperts", C.byref(ro), z, E, None, idx, wts, T, R.stream())
    cap = P.lib().routePlanCapacity(T, k, E, 128)
    offsets, order = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(cap, dtype=torch.int32, device="cuda")
    position = torch.empty(T, k, dtype=torch.int32, device="cuda")
    R.launch("launchRoutePlan", idx, T, k, E, 128, cap, offsets, order, position, R.stream())

    def product(x, w, n, kk, relu, order=None, slots=1):
        q, s, _, _ = R.run_quantize(x, 1, order=order, slots=slots, rows=cap)
        out = torch.zeros(cap, n, dtype=torch.bfloat16, device="cuda")
        o = P.Fp8ProductOption(m=cap, n=n, k=kk, numExperts=E, grouping=1, scaleRowsB=128, activation=int(relu), outType=2,
                               outStride=n)
        R.launch("launchFp8Product", C.byref(o), q, s, w[0], w[1], offsets, out, R.stream())
        return out

    hidden = product(L.x, L.w1, H, D, True, order, k)
    rows = product(hidden, L.w2, D, H, False)
    out = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    R.launch("launchExpertCombine", D, 2, rows, cap, D, position, wts, out, D, T, k, R.stream())
    got = L.run()
    assert torch.equal(idx.cpu(), L.indices)
    rel = float((got.double() - out.double()).norm() / out.double().norm())
    assert 1e-3 < rel < 2.0 ** -4 * 2  # two quantisings, each within 2^-4 of a value


def test_most_slots():
    """64 tokens that all take 32 of 64 experts (the most LDS that the outputs need), and all of 32."""
    for E, fmt, code in ((64, 0, 0), (32, 0, 2), (32, 1, 1)):
        Layer(64, E, 32, 140, 136, act=2, gated=True, fmt=fmt, code=code, seed=80 + E).check()


@pytest.mark.parametrize("T,E,gated", [(2, 9, False), (64, 9, False), (64, 8, True)])
def test_weights_beyond_2_gib(T, E, gated):
    """The last expert's matrices begin 2 GiB behind the first's (the gated form's first matrix does); dim and hidden are the
    largest."""
    D, H, code, last = 16384, 16384, 2, E - 1
    P = pkg()
    g = R.gen(90)
    w = []
    for rows in (2 * H if gated else H, D):
        q = torch.zeros(E, rows, P.fp8_pitch(D), dtype=torch.uint8, device="cuda")
        s = torch.full((E, rows // 128, P.fp8_scale_pitch(D)), 127, dtype=torch.uint8, device="cuda")
        q[last], s[last], _, _ = R.run_quantize(R.randn(g, rows, D) / 128, 128)
        w.append((q, s, {last: R.values(q[last], s[last], D, 128)}))
    x = R.randn(g, T, D).to(S.DT[code])
    router, bias = torch.zeros(E, D, device="cuda"), torch.zeros(E, device="cuda")
    bias[last] = 1.0
    out = torch.full((T, D), -7.0, dtype=S.DT[code], device="cuda")
    o = S.layer_option(E, 1, D, H, 1, gated, 0, 128, code, 0)
    R.launch("launchExpertLayer", C.byref(o), x, router, bias, w[0][0], w[0][1], w[1][0], w[1][1], out, T, R.stream())
    # one expert, renormalised: its weight is 1 to a rounding
    for t in range(0, T, 21):
        want, bound = S.layer(x[t:t + 1], torch.full((1, 1), last), torch.ones(1, 1), w[0][2], w[1][2], H, 1, gated, code)
        assert bool((out[t].double() - want[0]).abs().le(bound[0] + 2.0 ** -23 * want[0].abs()).all())


@pytest.mark.parametrize("T,E,k,code,fmt", [(64, 8, 2, 0, 0), (64, 1024, 4, 2, 1), (64, 64, 32, 1, 0)])
def test_captured_with_much_lds(T, E, k, code, fmt):
    """Kernels that ask for more than 64 KB of LDS, many slots an expert and many experts, replayed on other tokens."""
    L = Layer(T, E, k, 192, 136, act=3, code=code, fmt=fmt, seed=95)
    tokens = [L.x.clone(), torch.roll(L.x, 5, 0)]
    want = []
    for x in tokens:
        L.x.copy_(x)
        want.append(L.run().clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        L.run(s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            L.run(s.cuda_stream)
        for rep in range(5):
            L.x.copy_(tokens[rep % 2])
            L.out.fill_(-7)
            graph.replay()
            s.synchronize()
            assert torch.equal(L.out, want[rep % 2]), rep
