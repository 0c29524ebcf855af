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
@pytest.mark.parametrize("T,E", [(1, 8), (9, 8), (40, 8), (64, 4)])
def test_infinite_tokens(T, E, code, router, short):
    """Every other token has one: the experts whose router weight has its sign are available, all with the largest score, and
    the first of them is taken.  That one's outputs are +infinity, all others' -infinity or NaN."""
    D, H = 136, 64
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


@pytest.mark.parametrize("T,E,k", [(9, 8, 2), (64, 4, 2)])
@pytest.mark.parametrize("router", [0, 1, 2])
def test_largest_tokens(T, E, k, router):
    """fp32 numbers that would round to an infinity in bf16, in tokens that also have ordinary ones; the router's weights for
    them are bf16 numbers, so that no bits of the products are below 2^-133."""
    D, H, col = 200, 64, 17
    L = Layer(T, E, k, D, H, act=1, code=0, router=router, seed=9)
    big = torch.tensor([3.4028234e38, -3.4e38, 3.3962e38, 1.0], device="cuda")
    g = R.gen(T)
    sign = torch.where(torch.rand(E, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    if router != 1:  # fp16 has none that small
        L.router[:, col] = (sign * (1 + torch.arange(E, device="cuda") / 16) * 2.0 ** -126).to(L.router.dtype)
    else:
        L.router[:, col] = 0
    L.w1[0][:, :, col] = 0
    L.w1[0][:, 0, col] = 1  # the least number of the block's
    L.w1[2].copy_(torch.stack([R.values(q, s, D, 128) for q, s in zip(L.w1[0], L.w1[1])]))
    for shift in range(50):  # tokens whose routes do not hang on a score's last bits
        L.x[:, col] = big[(torch.arange(T, device="cuda") + shift) % 4]
        L.indices, L.weights, gap = L.routes(L.x)
        if gap > 1e-4:
            break
        L.x.copy_(R.randn(g, T, D))
    assert gap > 1e-4
    L.check()


@pytest.mark.parametrize("T,E,k", [(3, 8, 2), (33, 300, 3), (64, 4, 2)])
@pytest.mark.parametrize("code", [0, 2])
def test_tokens_of_nan(T, E, k, code):
    """Some, or all, tokens have no expert: zeros; the others' results are theirs, within what their sums may be off by (how
    the outputs' sums are shared out goes by the number of experts that are taken)."""
    D, H = 136, 72
    L = Layer(T, E, k, D, H, act=2, gated=True, code=code, fmt=1, seed=10)
    want, bound = S.layer(L.x, L.indices, L.weights, L.w1[2], L.w2[2], H, 2, True, code)
    dz = float(((D / 8 + 16) * 2.0 ** -24 * (L.x.double().abs() @ L.router.double().abs().t())).max())
    bound = bound + (4 * dz + 16 * 2.0 ** -24) * L.magnitude()  # as in Layer.check
    lost = torch.arange(T, device="cuda") % 3 == 0
    for hit in (lost, lost | True):
        L.x[hit, 5] = math.nan
        got = L.run()
        assert not bool(got[hit].any()) and bool((got.double() - want).abs().le(bound)[~hit].all())
