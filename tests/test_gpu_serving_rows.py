"""The answers of examples/expert_field.py's block against 64 bits, row by row and element by element."""
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from test_gpu_serving import trained  # noqa: E402

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def inner(block, x):
    """The layer's tokens as answer() makes them: the first norm's fp16 results."""
    P = R.pkg()
    h = torch.empty_like(x)
    o = block.norm_option(P.NORM_NONE, P.NORM_RMS, 0, 1.0)
    R.launch("launchNormGateResidual", R.byref(o), x, None, None, None, None, block.p["norm_in"], None, None, h, x.shape[0], R.stream())
    return h


def check_answers(block, x, y, w1, w2):
    T, D, H = x.shape[0], block.dim, block.hidden
    p = {n: v.double() for n, v in block.p.items()}
    h = inner(block, x)
    want_h = R.norm(x.double(), 1, p["norm_in"], None, 1e-6)
    # statistics in fp32: their sums of D squares, the root and the quotient
    assert bool((h.double() - want_h).abs().le((S.HALF[1] + (D / 8 + 32) * UNIT) * want_h.abs() + S.TINY[1]).all())
    # logits: sums of D products in fp32, twice the off of which a score's relative error is, and so a weight's
    z = h.double() @ p["router"].t()
    dz = (D / 8 + 16) * UNIT * (h.double().abs() @ p["router"].abs().t()).amax(1)
    done = 0
    for t in range(T):
        index, weight, gap = R.route(z[t:t + 1], None, block.topk, False, 1, 1, 2, True, 1.0)
        if gap <= 4 * float(dz[t]) + 16 * UNIT:
            continue  # a score's last bits decide
        done += 1
        f, off = S.layer(h[t:t + 1], index, weight, w1, w2, H, 1, False, 1)
        for j in range(block.topk):
            part, _ = S.layer(h[t:t + 1], index[:, j:j + 1], weight[:, j:j + 1], w1, w2, H, 1, False, 1)
            off = off + (4 * float(dz[t]) + 16 * UNIT) * part.abs()
        rms = float(torch.sqrt(f.square().mean() + 1e-6))
        n = f * p["norm_out"] / rms
        # n = f w / rms, and rms changes by at most |off| / sqrt(D); the products of two such changes and fp32's own steps
        dn = p["norm_out"].abs() * (off + f.abs() * off.norm() / (math.sqrt(D) * rms)) / rms
        assert float(off.norm()) / (math.sqrt(D) * rms) < 2.0 ** -8
        dn = dn * (1 + 2.0 ** -6) + (D / 8 + 40) * UNIT * n.abs()
        gate = p["gate"][0].half().double()
        want = x[t].double() + gate * n[0]
        bound = gate.abs() * dn[0] + 4 * UNIT * (x[t].double().abs() + (gate * n[0]).abs())
        bound = bound + S.HALF[1] * (want.abs() + bound) + S.TINY[1]
        assert bool((y[t].double() - want).abs().le(bound).all()), t
    assert done >= max(1, 0.9 * T)


@pytest.mark.parametrize("T", [1, 7, 64])
@pytest.mark.parametrize("D,H,E,k", [(64, 128, 4, 2), (192, 320, 5, 2), (256, 512, 8, 1)])
def test_answers(D, H, E, k, T):
    _, block, g = trained(D, H, E, k, T)
    x = R.randn(g, T, D).half()
    w1 = torch.stack([R.values(q, s, D, 128) for q, s in zip(block.w1.q, block.w1.s)])
    w2 = torch.stack([R.values(q, s, H, 128) for q, s in zip(block.w2.q, block.w2.s)])
    check_answers(block, x, block.answer(x), w1, w2)


@pytest.mark.parametrize("T", [1, 33])
def test_answers_from_four_bits(T):
    D, H, E, k = 192, 320, 5, 2
    M, block, g = trained(D, H, E, k, T)
    block.prepare(4)
    (w1, w2), x = block.served, R.randn(g, T, D).half()
    v1 = torch.stack([S.values4(q, s, D) for q, s in zip(w1.q, w1.s)])
    v2 = torch.stack([S.values4(q, s, H) for q, s in zip(w2.q, w2.s)])
    for w, v in ((block.p["w1"], v1), (block.p["w2"], v2)):  # as quantised to 64 bits
        assert all(torch.equal(S.quantize4(a, 1)[0] * torch.exp2(S.quantize4(a, 1)[1].double() - 127).repeat_interleave(32, 1)
                               [:, :a.shape[1]], b) for a, b in zip(w, v))
    y = block.answer(x)
    check_answers(block, x, y, v1, v2)
    points = torch.rand(T, 3, generator=g, device="cuda")
    head = R.randn(g, 3, D)
    assert torch.equal(M.colours(block, head, points), block.answer(M.embed(points, D).half()).float() @ head.t())


@pytest.mark.parametrize("bits", [4, 8])
def test_a_training_that_ends_with_answers(bits):
    from test_gpu_expert_field import example
    kind = dict(steps=2, tokens=256, dim=64, hidden=128, experts=4, verbose=False)
    M = example()
    plain, losses = M.train(**kind), M.train(answer_bits=bits, **kind)
    assert losses[:-1] == plain and len(losses) == 3 and math.isfinite(losses[-1])
