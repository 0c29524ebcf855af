"""64-bit references of the 4-bit matrices, the expert layer for few tokens (include/experts_abi.h) and the gradients'
norm (include/grad_abi.h), plain torch, and their inputs."""
from __future__ import annotations

import ctypes as C
import math

import torch

import experts_ref as R
from helpers import pkg

DT, HALF, TINY, DEV = R.DT, R.HALF, R.TINY, "cuda"
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---- 4-bit matrices ---------------------------------------------------------------

def quantize4(x, rule):
    """x [R, C] (any float type): e2m1 values and the scales' bytes in 64-bit arithmetic, [R, C] and [R, scale pitch]."""
    rows, cols = x.shape
    blocks = pkg().fp4_scale_pitch(cols)
    p = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    p[:, :cols] = x.double()
    p = p.view(rows, blocks, 32)
    top = p.abs().amax(2)
    fine = p.isfinite().all(2)
    top = torch.where(fine, top, 0.0)
    e = torch.full_like(top, -126.0)
    for n in range(-126, 126):  # a step for every border that the largest has passed
        border = 2.0 ** (n + 3) if rule == 0 else math.nextafter(6.0 * 2.0 ** n, math.inf)
        e = torch.where(top >= border, float(n + 1), e)
    v = torch.where(fine[:, :, None], p, 0.0) / torch.exp2(e)[:, :, None]
    a, count = v.abs(), torch.zeros_like(v, dtype=torch.int64)
    for i in range(7):
        half = (GRID[i] + GRID[i + 1]) / 2
        count += (a > half) if i % 2 == 0 else (a >= half)
    q = torch.tensor(GRID, dtype=torch.float64, device=x.device)[count] * torch.where(torch.signbit(v), -1.0, 1.0)
    byte = torch.where(fine, e + 127, 255.0).to(torch.uint8)
    return q.view(rows, -1)[:, :cols], byte


def codes4(q, cols):
    """64-bit values of the stored halves of bytes [R, pitch]: [R, cols]."""
    c = torch.stack([q & 15, q >> 4], 2).view(q.shape[0], -1).long()[:, :cols]
    return torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=q.device)[c]


def values4(q, s, cols):
    """64-bit values of a stored matrix."""
    scale = torch.exp2(s.double() - 127)
    scale = torch.where(s == 255, math.nan, scale)
    return codes4(q, cols) * scale.repeat_interleave(32, 1)[:, :cols]


def run_quantize4(x, rule=0, order=None, slots=1, rows=None):
    """Through the entry point: (q, s); x [R, C] of any row stride."""
    P = pkg()
    n, cols = x.shape
    rows = n if rows is None else rows
    o = P.Fp4QuantOption(rows=rows, cols=cols, batch=1, scaleRule=rule, srcType=CODE[x.dtype], slotsPerRow=slots, srcRows=n,
                         srcStride=x.stride(0), srcBatchStride=0)
    q = torch.full((rows, P.fp4_pitch(cols)), 0xAA, dtype=torch.uint8, device=DEV)
    s = torch.full((rows, P.fp4_scale_pitch(cols)), 0xAA, dtype=torch.uint8, device=DEV)
    P.launch("launchFp4Quantize", C.byref(o), x, order, q, s, R.stream())
    return q, s


def make_fp4(g, rows, cols):
    """A stored random matrix, its blocks' scales over several powers of two, and its 64-bit values."""
    spread = torch.exp2(torch.randint(-4, 5, (rows, -(-cols // 32)), generator=g, device=DEV).float())
    x = R.randn(g, rows, cols) * spread.repeat_interleave(32, 1)[:, :cols]
    q, s = run_quantize4(x, 1)
    return q, s, values4(q, s, cols)


def product_bound(k, magnitude, ref, code):
    """What an fp32 sum of k exact products may be off by (each of the at most k / 8 + 16 additions that follow one another
    rounds to 2^-24 of at most the sum of all magnitudes), and the result's own rounding."""
    sums = (k / 8 + 16) * 2.0 ** -24 * magnitude
    return sums + HALF[code] * (ref.abs() + sums) + TINY[code]


# ---- the layer of experts -----------------------------------------------------------

def weights8(g, experts, rows, cols, block_rows):
    """Stored e4m3 matrices of all experts (q, scales) and their 64-bit values [E, rows, cols]."""
    parts = []
    for _ in range(experts):
        q, s, _, _ = R.run_quantize(R.randn(g, rows, cols) / math.sqrt(cols), block_rows)
        parts.append((q, s, R.values(q, s, cols, block_rows)))
    return tuple(torch.stack(p).contiguous() for p in zip(*parts))


def weights4(g, experts, rows, cols, _=1):
    parts = []
    for _ in range(experts):
        q, s = run_quantize4(R.randn(g, rows, cols) / math.sqrt(cols), 1)
        parts.append((q, s, values4(q, s, cols)))
    return tuple(torch.stack(p).contiguous() for p in zip(*parts))


ACT = [lambda v: v, lambda v: torch.where(v < 0, 0.0, v), lambda v: v / (1 + torch.exp(-v)),
       lambda v: 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))]


def layer(x, indices, weights, w1, w2, hidden, act, gated, code):
    """(out, bound) in 64 bits of given routes: indices [T, k], weights [T, k], w1 [E, rows, D], w2 [E, D, H].

    The bound counts, in this order: hidden sums in fp32 (at most D / 8 + 16 additions in a row); the activation, whose slope
    is at most 1.13, in 8 units of 2^-24 of its argument and result; the product with the up rows; the hidden value in 16 bits
    (24 under fp32 tokens), 2^-16 (2^-23); the output's sums over H and over the experts; its rounding."""
    T, D = x.shape
    x = x.double()
    out = torch.zeros(T, D, dtype=torch.float64, device=x.device)
    off = torch.zeros_like(out)
    total = torch.zeros_like(out)
    unit = 2.0 ** -24
    n1, n2 = D / 8 + 16, hidden / 8 + 16
    for t in range(T):
        for j in range(indices.shape[1]):
            e = int(indices[t, j])
            if e < 0:
                continue
            w = float(weights[t, j])
            h = w1[e] @ x[t]
            dh = n1 * unit * (w1[e].abs() @ x[t].abs())
            v, dv = h[:hidden], dh[:hidden]
            a = ACT[act](v)
            da = 1.13 * dv + 8 * unit * (a.abs() + v.abs())
            if gated:
                u, du = h[hidden:], dh[hidden:]
                da = da * u.abs() + a.abs() * du + da * du + unit * (a * u).abs()
                a = a * u
            da = da + (2.0 ** -23 if code == 0 else 2.0 ** -16) * (a.abs() + da) + 2.0 ** -126
            y = w2[e] @ a
            mag = w2[e].abs() @ (a.abs() + da)
            out[t] += w * y
            off[t] += abs(w) * (w2[e].abs() @ da + n2 * unit * mag)
            total[t] += abs(w) * mag
    off = off + (indices.shape[1] + 10) * unit * total
    return out, off + HALF[code] * (out.abs() + off) + TINY[code]


def layer_option(experts, topk, dim, hidden, act=1, gated=False, fmt=0, scale_rows=128, code=0, router=0, sx=None, so=None,
                 **route):
    P = pkg()
    r = dict(numExperts=experts, topK=topk, scoreType=0, numGroups=1, topGroups=1, groupScore=2, renormalize=1, scale=1.0,
             logitsType=0)
    r.update(route)
    return P.ExpertLayerOption(route=P.RouteOption(**r), dim=dim, hidden=hidden, activation=act, gated=int(gated),
                               weightFormat=fmt, scaleRows=scale_rows, dataType=code, routerType=router, strideX=sx or dim,
                               strideOut=so or dim)


# ---- gradients ------------------------------------------------------------------------

def tensors(data, out=None):
    P = pkg()
    out = out or [None] * len(data)
    return (P.GradTensor * len(data))(*(
        P.GradTensor(data=t.data_ptr() if t.numel() else None, out=o.data_ptr() if o is not None and o.numel() else None,
                     n=t.numel(), dataType=CODE[t.dtype]) for t, o in zip(data, out)))


def norm64(data, kind, scale):
    if kind == 1:
        tops = [float(t.double().abs().amax()) for t in data if t.numel()]
        return (math.nan if any(math.isnan(v) for v in tops) else max(tops, default=0.0)) / scale
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in data)) / scale
