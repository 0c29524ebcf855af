"""Gradients' clipping, 4-bit matrices and the layer of experts as they are used together: a training step of the block of
examples/expert_field.py, its weights made ready and its answers; the same in a graph, on threads' own streams and in place."""
import ctypes as C
import threading

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from helpers import pkg  # noqa: E402
from test_gpu_expert_field import example  # noqa: E402
from test_gpu_expert_layer import Layer  # noqa: E402

pytestmark = pytest.mark.gpu


def trained(D, H, E, k, seed):
    """A block after a step of gradient descent on clipped gradients, each part checked on the way."""
    M = example()
    block = M.ExpertBlock(D, H, E, k, seed=seed)
    g = R.gen(seed + 1)
    x = R.randn(g, 256, D).half()
    block.forward(x)
    _, grad = block.backward(R.randn(g, 256, D).half())
    names = list(grad)
    before = [grad[n].clone() for n in names]
    want = S.norm64(before, 0, 64.0)
    n = float(M.clip([grad[i] for i in names], want / 8, 64.0))
    assert abs(n - want) <= (2.0 ** -24 + 1e-12) * want
    # maxNorm and the factor are fp32, three roundings with the element's own
    for b, i in zip(before, names):
        off = (grad[i].double() - b.double() / 8).abs()
        assert bool(off.le(4 * 2.0 ** -24 * b.double().abs() / 8 + 2.0 ** -149).all()), i
    for i in names:
        block.p[i] -= 0.1 * grad[i] / 64.0
    block.prepare()
    return M, block, g


def routed(block, h):
    z = h.double() @ block.p["router"].double().t()
    return R.route(z, None, block.topk, False, 1, 1, 2, True, 1.0)


@pytest.mark.parametrize("T", [1, 7, 64])
@pytest.mark.parametrize("D,H,E,k", [(64, 128, 4, 2), (192, 320, 5, 2), (256, 512, 8, 1)])
def test_a_step_and_its_answers(D, H, E, k, T):
    M, block, g = trained(D, H, E, k, T)
    x = R.randn(g, T, D).half()
    y = block.answer(x)
    assert torch.equal(y, block.answer(x))
    p = {n: v.double() for n, v in block.p.items()}
    h = R.norm(x.double(), 1, p["norm_in"], None, 1e-6).half()
    index, weight, gap = routed(block, h)
    w1 = torch.stack([R.values(q, s, D, 128) for q, s in zip(block.w1.q, block.w1.s)])
    w2 = torch.stack([R.values(q, s, H, 128) for q, s in zip(block.w2.q, block.w2.s)])
    f, bound = S.layer(h, index, weight, w1, w2, H, 1, False, 1)
    want = x.double() + block.p["gate"].half().double() * R.norm(f, 1, p["norm_out"], None, 1e-6)
    rms = f.square().mean(1).sqrt()
    # A row's error: h may differ by a rounding to fp16 here and there, 2^-10 of f's norm with the layer's Lipschitz constant
    # of about 2; f's bound; both through the norm (at most 2 / rms of a change); y's rounding.
    share = (bound.norm(dim=1) + 2 * 2.0 ** -10 * f.norm(dim=1)) * 2 / rms * float(p["gate"].abs().max()) + 2.0 ** -10 * want.norm(dim=1)
    if gap > 1e-2:  # no route that a rounding of h turns
        assert bool((y.double() - want).norm(dim=1).le(share).all())
    # and the block's own chain, which quantises tokens and hidden values to e4m3 (2^-4 at most, 2^-5 in the middle)
    other = block.forward(x)
    rel = float((y.double() - other.double()).norm() / (other.double() - x.double()).norm())
    assert rel < 2 * 2.0 ** -4


def quantized4(w):
    """launchFp4Quantize of all experts' matrices at once: (q, s, 64-bit values)."""
    P = pkg()
    E, rows, cols = w.shape
    q = torch.empty(E, rows, P.fp4_pitch(cols), dtype=torch.uint8, device="cuda")
    s = torch.empty(E, rows, P.fp4_scale_pitch(cols), dtype=torch.uint8, device="cuda")
    o = P.Fp4QuantOption(rows=rows, cols=cols, batch=E, scaleRule=P.FP4_SCALE_COVER, srcType=0, slotsPerRow=0, srcRows=rows,
                         srcStride=cols, srcBatchStride=rows * cols)
    P.launch("launchFp4Quantize", C.byref(o), w, None, q, s, R.stream())
    return q, s, torch.stack([S.values4(a, b, cols) for a, b in zip(q, s)])


@pytest.mark.parametrize("T", [3, 50])
def test_four_bits_both_ways(T):
    """The trained experts in 4 bits: the layer, and routing, gather, 4-bit products and combine, which quantise the tokens and
    the hidden values too."""
    P = pkg()
    D, H, E, k = 192, 320, 5, 2
    M, block, g = trained(D, H, E, k, 3)
    L = Layer(T, E, k, D, H, act=1, fmt=1, code=1, router=0, seed=30)
    L.router = block.p["router"]
    L.w1, L.w2 = quantized4(block.p["w1"]), quantized4(block.p["w2"])
    L.indices, L.weights, _ = L.routes(L.x)
    L.check()
    z = (L.x.float() @ L.router.t()).contiguous()
    idx, wts = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
    R.launch("launchRouteExperts", C.byref(L.o.route), z, E, None, idx, wts, T, R.stream())
    cap = P.lib().routePlanCapacity(T, k, E, 1)
    offsets, order = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(cap, dtype=torch.int32, device="cuda")
    position = torch.empty(T, k, dtype=torch.int32, device="cuda")
    R.launch("launchRoutePlan", idx, T, k, E, 1, cap, offsets, order, position, R.stream())

    def product(x, w, n, kk, relu, order=None, slots=1):
        q, s = S.run_quantize4(x, 1, order, slots, cap)
        out = torch.full((cap, n), -7.0, dtype=torch.float16, device="cuda")
        o = P.Fp4ProductOption(m=cap, n=n, k=kk, numExperts=E, grouping=P.PRODUCT_ROWS, activation=int(relu), outType=1, outStride=n)
        R.launch("launchFp4Product", C.byref(o), q, s, w[0], w[1], offsets, out, R.stream())
        return out, S.values4(q, s, kk)

    hidden, a = product(L.x, L.w1, H, D, True, order, k)
    rows, b = product(hidden, L.w2, D, H, False)
    out = torch.empty(T, D, dtype=torch.float16, device="cuda")
    R.launch("launchExpertCombine", D, 1, rows, cap, D, position, wts, out, D, T, k, R.stream())
    assert torch.equal(idx.cpu(), L.indices)
    bounds = offsets.tolist()
    for e in range(E):
        mine = slice(bounds[e], bounds[e + 1])
        for x, w, n, got, relu in ((a, L.w1, D, hidden, True), (b, L.w2, H, rows, False)):
            want = x[mine] @ w[2][e].t()
            bound = S.product_bound(n, x[mine].abs() @ w[2][e].abs().t(), want, 1)
            want = want.clamp(min=0) if relu else want
            assert bool((got[mine].double() - want).abs().le(bound).all())
    rel = float((L.run().double() - out.double()).norm() / out.double().norm())
    assert 1e-2 < rel < 2 * 2.0 ** -2  # two quantisings to e2m1, each within a quarter of a value


def test_clip_quantise_and_layer_in_one_graph():
    """Captured once, replayed on other gradients, weights and tokens, with eager calls on the stream between the replays."""
    M = example()
    D, H, E, k, T = 160, 256, 6, 2, 12
    L = Layer(T, E, k, D, H, act=2, gated=True, fmt=1, code=2, seed=40)
    big = Layer(64, 8, 2, 512, 512, code=0, seed=41)
    g = R.gen(42)
    sets = [(R.randn(g, E, 2 * H, D) / 12, R.randn(g, E, D, H) / 16, R.randn(g, T, D).bfloat16()) for _ in range(3)]
    w1, w2 = torch.empty_like(sets[0][0]), torch.empty_like(sets[0][1])
    P = pkg()

    def run(handle):
        n = M.clip([w1, w2], 5.0, 1.0)
        for w, to in ((w1, L.w1), (w2, L.w2)):
            o = P.Fp4QuantOption(rows=w.shape[1], cols=w.shape[2], batch=E, scaleRule=0, srcType=0, slotsPerRow=0, srcRows=w.shape[1],
                                 srcStride=w.shape[2], srcBatchStride=w[0].numel())
            P.launch("launchFp4Quantize", C.byref(o), w, None, to[0], to[1], handle)
        L.run(handle)
        return n

    def put(i):
        w1.copy_(sets[i][0])
        w2.copy_(sets[i][1])
        L.x.copy_(sets[i][2])
        L.out.fill_(-7)

    want = []
    for i in range(3):
        put(i)
        n = run(R.stream())
        want.append((n.clone(), w1.clone(), L.w2[0].clone(), L.out.clone()))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        put(0)
        run(s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            n = run(s.cuda_stream)
        for rep in range(7):
            put(rep % 3)
            graph.replay()
            s.synchronize()
            for a, b in zip((n, w1, L.w2[0], L.out), want[rep % 3]):
                assert torch.equal(a, b), rep
            if rep % 2:
                big.run(s.cuda_stream)
                s.synchronize()


def test_a_first_call_under_capture_is_refused():
    """On a stream that has had none; the same call captures after one that was not captured."""
    hip = C.CDLL("libamdhip64.so")
    handle = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(handle)) == 0
    s = torch.cuda.ExternalStream(handle.value)
    L = Layer(5, 4, 2, 64, 64, code=2, seed=50)
    want = L.run().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        with pytest.raises(RuntimeError, match="first call"):
            L.run(handle.value)
        L.out.zero_()
    with torch.cuda.stream(s):
        L.run(handle.value)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            L.run(handle.value)
        for _ in range(3):
            L.out.fill_(-7)
            graph.replay()
            s.synchronize()
            assert torch.equal(L.out, want)


def test_threads_on_their_own_streams():
    """hipStreamPerThread: each thread's calls have counters and scratch of their own."""
    jobs = [Layer(7 * i + 3, 8, 2, 256, 192, fmt=i % 2, code=i % 3, seed=60 + i) for i in range(4)]
    want = [j.run().clone() for j in jobs]
    torch.cuda.synchronize()
    bad = []

    def work(j, w):
        for _ in range(20):
            j.run(2)
        if C.CDLL("libamdhip64.so").hipStreamSynchronize(C.c_void_p(2)) or not torch.equal(j.out, w):
            bad.append(j.size)

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (9, 6, 3), (64, 4, 2)])
@pytest.mark.parametrize("code", [0, 1, 2])
def test_in_place(T, E, k, code):
    """Tokens are read before anything is written: out may be x."""
    L = Layer(T, E, k, 200, 136, act=3, code=code, seed=70)
    want = L.run().clone()
    L.out = L.x
    L.o.strideOut = L.o.strideX
    assert torch.equal(L.run(), want)


def test_a_training_with_and_without_clipping():
    """A bound that no norm reaches changes nothing; one that is reached changes the course."""
    M = example()
    kind = dict(steps=3, tokens=256, dim=64, hidden=128, experts=4, verbose=False)
    plain = M.train(**kind)
    assert M.train(max_norm=1e30, **kind) == plain
    assert M.train(max_norm=1e-3, **kind) != plain
