"""Clipping gradients that are far above the norm they are scaled to (include/grad_abi.h), against 64-bit arithmetic."""
import math

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from test_gpu_grad_norm import clip, norm  # noqa: E402

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


@pytest.mark.parametrize("max_norm", [0.0, 2.0 ** -149, 1e-40, 1e-30, 1e-3, 1.0, 3.0])
@pytest.mark.parametrize("place", ["in", "out", "given"])
@pytest.mark.parametrize("code", [0, 2])
@pytest.mark.parametrize("size", [9, 300_001])
def test_factors_below_the_normal_numbers(size, code, place, max_norm):
    """maxNorm / n is below 2^-126: it counts with all of fp32's bits (2^-24), as do the product and, of results above the
    subnormal numbers, the rounding.  Below those: a step of 2^-149 for each of two roundings, and the type's."""
    g = R.gen(size)
    data = [R.randn(g, size).clamp(-3, 3) * 2.0 ** 100, R.randn(g, 33).clamp(-3, 3) * 2.0 ** 10, torch.zeros(7, device="cuda")]
    data = [t.to(S.DT[code]) for t in data]
    data[0][size // 2], data[0][0] = 2.9e38, -1.7e38
    before = [t.clone() for t in data]
    n = float(norm(data))
    assert abs(n - S.norm64(data, 0, 1.0)) <= UNIT * n and max_norm / n < 2.0 ** -126
    max_norm = float(torch.tensor(max_norm, dtype=torch.float32))
    out = [torch.full_like(t, 5.0) for t in data] if place == "out" else None
    got = clip(data, out, max_norm, given=torch.tensor([n], device="cuda") if place == "given" else None)
    assert float(got) == n and math.isfinite(n)
    for a, b in zip(before, out or data):
        want = a.double() * (max_norm / n)
        bound = (3 * UNIT + S.HALF[code]) * want.abs() + 2 * 2.0 ** -149 + S.TINY[code]
        assert bool((b.double() - want).abs().le(bound).all())
