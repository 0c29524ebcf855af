"""Experts whose scores are subnormal numbers (their logits 87 to 103 behind the first one's) are ordered by them, as
any others; indices equal the 64-bit definition's.  Logits are at least half apart: a score's steps are 2^-149 there,
which at e^-100 is 4 % of it."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,k,groups,kept", [(32, 32, 1, 1), (64, 20, 1, 1), (64, 12, 4, 2), (200, 32, 1, 1), (512, 32, 1, 1)])
@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("code", [0, 1])
def test_far_experts_in_order(E, k, groups, kept, sigmoid, code):
    print(f"[far] E={E} k={k} groups={groups} sigmoid={sigmoid} type={code}", flush=True)
    T = 40
    g = R.gen(E + k)
    z = torch.full((T, E), -150.0, device="cuda")  # scores of 0: equal, lowest index first
    for t in range(T):
        n = min(31, E)
        at = torch.randperm(E, generator=g, device="cuda")[:n]
        z[t, at] = -85.0 - 0.5 * torch.arange(n, device="cuda")
        if t % 2 == 0:
            z[t, at[0]] = 0.0
        else:
            z[t, at[0]] = -84.0
    if not sigmoid:  # behind the first one, wherever that is
        z -= z.amax(1, keepdim=True) - 1.5
    z = z.to(R.DT[code])
    o = pkg().RouteOption(numExperts=E, topK=k, scoreType=sigmoid, numGroups=groups, topGroups=kept, groupScore=1, renormalize=0,
                          scale=1.0, logitsType=code)
    idx, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), -7.0, device="cuda")
    R.launch("launchRouteExperts", C.byref(o), z, E, None, idx, w, T, R.stream())
    torch.cuda.synchronize()
    # the definition in 64 bits, with scores that fp32 has not as 0
    s, live = R.scores(z, sigmoid)
    s = torch.where(s < 2.0 ** -150, 0.0, s)
    order = []
    for row in s.cpu().tolist():
        pool = range(E)
        if groups > 1:
            per = E // groups
            best = sorted(range(groups), key=lambda q: (-max(row[q * per:(q + 1) * per]), q))[:kept]
            pool = [e for e in pool if e // per in best]
        order.append(sorted(pool, key=lambda e: (-row[e], e))[:k])
    want = torch.tensor(order, dtype=torch.int32)
    assert torch.equal(idx.cpu(), want)
    rw = s.cpu().gather(1, want.long())
    assert ((w.cpu().double() - rw).abs() <= 2.0 ** -20 * rw + 2.0 ** -148).all()
