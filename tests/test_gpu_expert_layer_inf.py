"""Infinite tokens and router weights in the layer of experts (include/experts_abi.h): their logits are infinite, not NaN,
whatever bits the other operand has, and route as launchRouteExperts routes such logits."""
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from test_gpu_expert_layer import Layer  # noqa: E402

pytestmark = pytest.mark.gpu


def in_eight_bits(t):
    """The nearest bf16 numbers, in t's type: fp16 holds those of the router's and tokens' size."""
    return t.bfloat16().to(t.dtype)


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("router", [0, 1, 2])
@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("T", [1, 9, 40])
def test_infinite_tokens(T, code, router, short):
    """Every other token has one: the experts whose router weight has its sign are available, all with the largest score, and
    the first of them is taken.  That one's outputs are +infinity, all others' -infinity or NaN."""
    E, D, H = 8, 136, 64
    L = Layer(T, E, 1, D, H, act=0, code=code, router=router, scoreType=1, renormalize=0, seed=7)
    if short:  # no second terms
        L.router.copy_(in_eight_bits(L.router))
        L.x.copy_(in_eight_bits(L.x))
    clean = L.run().clone()
    col, hit = 37, torch.arange(0, T, 2)
    sign = [1.0 if i % 4 == 0 else -1.0 for i in hit.tolist()]
    L.x[hit, col] = torch.tensor(sign, device="cuda").to(L.x.dtype) * math.inf
    # every hidden value takes that column with a positive weight, every output hidden value 0 alone
    w1, w2 = L.w1[0].view(E, H, -1), L.w2[0].view(E, D, -1)
    w1[:, :, col] = 0x38  # 1 times the block's scale
    w2.zero_()
    z = L.x.double() @ L.router.double().t()
    assert bool(z[hit].isinf().all())
    idx, weight, _ = R.route(z, None, 1, True, 1, 1, 2, False, 1.0)
    assert bool((weight[hit] == 1.0).all())
    for s in (1.0, -1.0):
        mine = hit[[i for i, v in enumerate(sign) if v == s]]
        if len(mine) == 0:
            continue
        first = set(idx[mine, 0].tolist())
        assert len(first) == 1
        e = first.pop()
        # 1 or -1 times the scale, so that the right expert's products are +infinity and another's -infinity
        w2[:, :, :H] = 0xB8 if s > 0 else 0x38
        w2[e, :, :H] = 0x38 if s > 0 else 0xB8
        got = L.run()
        assert bool((got[mine] == math.inf).all())
        if s > 0:
            w2.zero_()
    # the others take the experts that they took
    other = torch.arange(1, T, 2)
    assert bool(clean.isfinite().all()) and bool(L.run()[other].isfinite().all())


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("router", [0, 1, 2])
@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("sigmoid", [0, 1])
def test_infinite_router_weights(code, router, short, sigmoid):
    """Two experts have one: their logits are +infinity or -infinity by the sign of the token's element."""
    T, E, k, D, H = 23, 8, 3, 136, 64
    L = Layer(T, E, k, D, H, act=1, code=code, router=router, scoreType=sigmoid, seed=8)
    if short:
        L.x.copy_(in_eight_bits(L.x))
        L.router.copy_(in_eight_bits(L.router))
    finite = L.router.clone()
    L.router[2, 11], L.router[5, 90] = math.inf, -math.inf
    assert bool((L.x[:, [11, 90]] != 0).all())
    L.indices, L.weights, gap = L.routes(L.x)
    assert gap > 1e-5 and (L.indices == 2).any() and (L.indices == 5).any() and not (L.indices == 2).any(1).all()
    want, bound = S.layer(L.x, L.indices, L.weights, L.w1[2], L.w2[2], H, 1, False, code)
    # logits without infinities are off by a few units of their sums, which count for the weights (see Layer.check)
    dz = float(((D / 8 + 16) * 2.0 ** -24 * (L.x.double().abs() @ finite.double().abs().t())).max())
    off = (L.run().double() - want).abs()
    assert bool(off.le(bound + (4 * dz + 16 * 2.0 ** -24) * L.magnitude()).all())
