"""How many bits the layer of experts (include/experts_abi.h) keeps between tokens and results: hidden activations whose
large parts cancel in the second product, logits whose large parts cancel in the router's."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from helpers import pkg  # noqa: E402
from test_gpu_expert_layer import Layer  # noqa: E402

pytestmark = pytest.mark.gpu
EXACT = pkg().EXPERT_HIDDEN_F32


def quantized(w):
    """One expert's matrix [rows, cols] of numbers that e4m3 holds: (q, scales) as the layer takes them."""
    q, s, _, _ = R.run_quantize(w, 128)
    assert torch.equal(R.values(q, s, w.shape[1], 128), w.double())
    return q[None].contiguous(), s[None].contiguous()


def run(x, router, w1, w2, o):
    out = torch.full(x.shape, -7.0, dtype=x.dtype, device="cuda")
    (q1, s1), (q2, s2) = quantized(w1), quantized(w2)
    R.launch("launchExpertLayer", C.byref(o), x, router, None, q1, s1, q2, s2, out, x.shape[0], R.stream())
    return out


def hidden_values(T, n, code):
    """(x, w1, w2, the outputs in 64 bits): hidden value i is w_0 + w_1 / 16 + .. + w_5 / 16^5 with w in 1 .. 1.875, all 24
    bits of an fp32 number below 2, and hidden value n + i the first four of them, 16 bits; output i is their difference."""
    w = 1 + torch.randint(0, 8, (n, 6), generator=R.gen(T + n), device="cuda").double() / 8
    w[:, 0] = w[:, 0].clamp(max=1.75)
    x = torch.zeros(T, n, dtype=S.DT[code], device="cuda")
    x[:, :6] = torch.tensor([16.0 ** -i for i in range(6)])
    w1 = torch.zeros(2 * n, n, dtype=torch.float64, device="cuda")
    w1[:n, :6], w1[n:, :4] = w, w[:, :4]
    w2 = torch.cat([torch.eye(n), -torch.eye(n)], 1).cuda()
    want = (w[:, 4:] * torch.tensor([16.0 ** -4, 16.0 ** -5], dtype=torch.float64, device="cuda")).sum(1)
    return x, w1.float(), w2, want


@pytest.mark.parametrize("T", [1, 7, 40])
@pytest.mark.parametrize("code", [0, 1, 2])
def test_hidden_values(T, code):
    """Two bf16 terms, each the nearest: of a value h in 1 .. 2 the first leaves at most 2^-8, of which the second is off by at
    most half of 2^-16.  Three terms hold all of it.  All sums are of multiples of 2^-24 below 2: exact."""
    n = 96
    x, w1, w2, want = hidden_values(T, n, code)
    o = S.layer_option(1, 1, n, 2 * n, act=0, code=code)
    got = run(x, torch.zeros(1, n, device="cuda"), w1, w2, o).double()
    off = 0.0 if code == 0 else 2.0 ** -17
    bound = off + S.HALF[code] * (want + off) + S.TINY[code]
    assert bool((got - want).abs().le(bound).all()), float((got - want).abs().max() * 2 ** 17)


@pytest.mark.parametrize("T", [1, 7, 40])
@pytest.mark.parametrize("code", [0, 1, 2])
def test_hidden_values_in_fp32(T, code):
    """On request nothing of them is lost, and no other result changes."""
    n = 96
    x, w1, w2, want = hidden_values(T, n, code)
    o = S.layer_option(1, 1, n, 2 * n, act=0, code=code | EXACT)
    got = run(x, torch.zeros(1, n, device="cuda"), w1, w2, o)
    assert torch.equal(got, want.to(got.dtype).expand(T, n))


@pytest.mark.parametrize("T,E,k,D,H,act,gated,fmt", [
    (1, 8, 2, 64, 96, 1, False, 0), (7, 16, 4, 300, 200, 2, True, 1), (11, 4, 2, 136, 140, 3, False, 0),
    (33, 5, 2, 260, 72, 2, True, 1), (64, 4, 2, 136, 264, 0, True, 0), (64, 16, 1, 384, 130, 3, False, 1)])
@pytest.mark.parametrize("code", [1, 2])
def test_layers_in_fp32(T, E, k, D, H, act, gated, fmt, code):
    """Against 64 bits with hidden values of 24 bits: tokens widened to fp32 are the same tokens, whose bound counts that."""
    L = Layer(T, E, k, D, H, act=act, gated=gated, fmt=fmt, code=code, seed=11)
    L.o.dataType |= EXACT
    got = L.run()
    want, bound = S.layer(L.x, L.indices, L.weights, L.w1[2], L.w2[2], H, act, gated, 0)
    dz = float(((D / 8 + 16) * 2.0 ** -24 * (L.x.double().abs() @ L.router.double().abs().t())).max())
    bound = bound + (4 * dz + 16 * 2.0 ** -24) * L.magnitude()
    assert bool((got.double() - want).abs().le(bound + S.HALF[code] * (want.abs() + bound) + S.TINY[code]).all())
    assert torch.equal(got, L.run())


def test_layers_in_fp32_captured():
    """Many slots an expert and few, on a stream of its own, replayed on other tokens."""
    for T, E in ((40, 4), (9, 16)):
        L = Layer(T, E, 2, 264, 136, act=2, gated=True, code=2, seed=12)
        L.o.dataType |= EXACT
        tokens = [L.x.clone(), torch.roll(L.x, 3, 0)]
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
            for rep in range(4):
                L.x.copy_(tokens[rep % 2])
                L.out.fill_(-7)
                graph.replay()
                s.synchronize()
                assert torch.equal(L.out, want[rep % 2]), rep


def test_logits():
    """a b - c in the router, where c is a b rounded to fp32, times 2^15: what the products of the third terms that are left
    out may change.  Of a and b in 1 .. 2 the second term is at most 2^-8 and the third 2^-17, so both such products are
    within 2^-24, and the ninth, of both third terms, 2^-34.  The other products add up within 2^-5 behind the first, on a
    grid of 2^-31 at least: at most a rounding of 2^-30 for each of 14."""
    T, n = 64, 8
    g = R.gen(77)
    a = 1 + torch.rand(T, generator=g, device="cuda")
    b = 1 + torch.rand(T, generator=g, device="cuda")
    a[0] = b[0] = a[1] = float.fromhex("0x1.01fffep+0")
    a[2] = b[2] = float.fromhex("0x1.fffffep+0")
    for t in range(T):  # each with its own router
        x = torch.zeros(1, n, device="cuda")
        x[0, 0], x[0, 1] = a[t] * 2.0 ** 15, 2.0 ** 15
        router = torch.zeros(1, n, device="cuda")
        c = (a[t].double() * b[t].double()).float()
        router[0, 0], router[0, 1] = b[t], -c
        z = 2.0 ** 15 * (float(a[t]) * float(b[t]) - float(c))
        w1 = torch.zeros(n, n, device="cuda")
        w1[:, 1] = 2.0 ** -15
        o = S.layer_option(1, 1, n, n, act=0, scoreType=1, renormalize=0)
        got = float(run(x, router, w1, torch.eye(n, device="cuda"), o)[0, 0])
        want = float(torch.sigmoid(torch.tensor(z, dtype=torch.float64)))
        # a quarter of the logit's error, and the score's own few roundings
        assert abs(got - want) <= 2.0 ** 15 * (2.0 ** -24 + 2.0 ** -34 + 14 * 2.0 ** -30) / 4 + 8 * 2.0 ** -24, t
