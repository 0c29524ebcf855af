"""64-bit references of the mixture-of-experts operators (include/experts_abi.h), plain torch, and their inputs."""
from __future__ import annotations

import ctypes as C
import math

import torch

from helpers import pkg

DT = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
# half of the relative spacing of a type (its rounding), and the smallest spacing
HALF = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}
TINY = {0: 2.0 ** -149, 1: 2.0 ** -24, 2: 2.0 ** -133}
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def strided(t, pad, shift=0):
    """t [R, C] with rows C + pad apart, `shift` elements off an allocation's start."""
    R, Cc = t.shape
    buf = torch.zeros(shift + R * (Cc + pad), dtype=t.dtype, device=t.device)
    v = buf[shift:].view(R, Cc + pad)[:, :Cc]
    v.copy_(t)
    return v


def launch(name, *args):
    pkg().launch(name, *args)


def byref(o):
    return C.byref(o)


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- routing -------------------------------------------------------------------

def scores(z, sigmoid):
    """[T, E] scores in 64 bits; experts whose logit is -inf or NaN have none (0)."""
    z = z.double()
    live = z > -math.inf
    z = torch.where(live, z.clamp(max=3.402823466e38), 0.0)
    if sigmoid:
        s = torch.sigmoid(z)
    else:
        m = torch.where(live, z, -math.inf).amax(1, keepdim=True)
        m = torch.where(m > -math.inf, m, 0.0)
        e = torch.where(live, torch.exp(z - m), 0.0)
        t = e.sum(1, keepdim=True)
        s = e / torch.where(t > 0, t, 1.0)
    return torch.where(live, s, 0.0), live


def route(z, bias, k, sigmoid, groups, kept, group_best, renorm, scale):
    """(indices, weights, least gap of a decision), row by row in plain Python."""
    s, live = scores(z, sigmoid)
    c = s + bias.double() if bias is not None else s.clone()
    live = live & (c > -math.inf)
    s_, c_, l_ = s.cpu().tolist(), c.cpu().tolist(), live.cpu().tolist()
    T, E = z.shape
    per = E // groups
    idx, wts, gap = [], [], math.inf

    def decide(order, n):
        nonlocal gap
        for a, b in zip(order[:n], order[1:n + 1]):
            if a[0] != b[0]:
                gap = min(gap, abs(a[0] - b[0]) / max(abs(a[0]), abs(b[0])))

    for t in range(T):
        ok = [e for e in range(E) if l_[t][e]]
        if groups > 1:
            best = []
            for g in range(groups):
                own = sorted((c_[t][e] for e in ok if e // per == g), reverse=True)[:group_best]
                if own:
                    best.append((sum(own), g))
            best.sort(key=lambda v: (-v[0], v[1]))
            decide(best, kept)
            keep = {g for _, g in best[:kept]}
            ok = [e for e in ok if e // per in keep]
        order = sorted(((c_[t][e], e) for e in ok), key=lambda v: (-v[0], v[1]))
        decide(order, k)
        pick = [e for _, e in order[:k]]
        w = [s_[t][e] for e in pick]
        total = sum(w) + 1e-20
        idx.append(pick + [-1] * (k - len(pick)))
        wts.append([v * scale / (total if renorm else 1.0) for v in w] + [0.0] * (k - len(pick)))
    return torch.tensor(idx, dtype=torch.int32), torch.tensor(wts, dtype=torch.float64), gap


def plan(indices, experts, align, capacity):
    """(offsets, order, position) as lists."""
    flat = indices.reshape(-1).cpu().tolist()
    rows = [[i for i, e in enumerate(flat) if e == x] for x in range(experts)]
    offsets, order, position = [0], [-1] * capacity, [-1] * len(flat)
    for r in rows:
        for n, slot in enumerate(r):
            order[offsets[-1] + n] = slot
            position[slot] = offsets[-1] + n
        offsets.append(offsets[-1] + -(-len(r) // align) * align)
    return offsets, order, position


# ---- 8-bit matrices ---------------------------------------------------------------

def quantize(x, block_rows=1):
    """x [R, C] (any float type): e4m3 values and scales' bytes in 64-bit arithmetic."""
    R, Cc = x.shape
    rb, cb = -(-R // block_rows), -(-Cc // 128)
    p = torch.zeros(rb * block_rows, cb * 128, dtype=torch.float64, device=x.device)
    p[:R, :Cc] = x.double()
    b = p.view(rb, block_rows, cb, 128)
    top = torch.where(b.isfinite(), b.abs(), 0.0).amax((1, 3))
    e = torch.full_like(top, -126.0)
    for n in range(-126, 121):  # the smallest power of two that brings the block within 448
        e = torch.where(top > 448.0 * 2.0 ** n, float(n + 1), e)
    v = torch.where(p.isfinite(), p, math.nan).view_as(b) / torch.exp2(e)[:, None, :, None]
    a = v.abs()
    lead = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    lead = torch.where(a < torch.exp2(lead), lead - 1, lead).clamp(min=-6)
    step = torch.exp2(lead - 3)
    q = torch.where(a.isnan(), v, torch.round(v / step) * step)
    return q.view(rb * block_rows, cb * 128)[:R, :Cc], (e + 127).to(torch.uint8)


def values(q, s, cols, block_rows=1):
    """64-bit values of stored bytes [R, pitch] and scale bytes [R', scale pitch]."""
    v = q[:, :cols].contiguous().view(torch.float8_e4m3fn).double()
    e = torch.exp2(s.double() - 127)
    return v * e[torch.arange(v.shape[0], device=v.device) // block_rows][:, torch.arange(cols, device=v.device) // 128]


def q_buffers(rows, cols, block_rows=1):
    P = pkg()
    q = torch.full((rows, P.fp8_pitch(cols)), 0xAA, dtype=torch.uint8, device=DEV)
    s = torch.full((-(-rows // block_rows), P.fp8_scale_pitch(cols)), 0xAA, dtype=torch.uint8, device=DEV)
    return q, s


def run_quantize(x, block_rows=1, order=None, weights=None, gate=None, slots=1, rows=None, row_side=True, t_side=False,
                 type_=None):
    """Through the entry point: (q, s, qt, st); x [R, C] of any row stride."""
    P = pkg()
    R, Cc = x.shape
    rows = R if rows is None else rows
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
    o = P.Fp8QuantOption(rows=rows, cols=Cc, batch=1, blockRows=block_rows, srcType=code, slotsPerRow=slots, srcRows=R,
                         srcStride=x.stride(0), srcBatchStride=0, gateStride=gate.stride(0) if gate is not None else 0)
    q, s = q_buffers(rows, Cc, block_rows) if row_side else (None, None)
    qt, st = q_buffers(Cc, rows, block_rows) if t_side else (None, None)
    P.launch("launchFp8Quantize", C.byref(o), x, order, weights, gate, q, s, qt, st, stream())
    return q, s, qt, st


def make_fp8(g, rows, cols, block_rows=1, spread=3.0):
    """A stored random matrix of this many rows, its scales over several powers of two, and its 64-bit values."""
    x = randn(g, rows, cols) * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g, device=DEV).float() * spread / 3)
    q, s, _, _ = run_quantize(x, block_rows)
    return q, s, values(q, s, cols, block_rows)


# ---- norms ------------------------------------------------------------------------

def norm(v, kind, w, b, eps):
    if kind == 0:
        return v
    if kind == 2:
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def block(x, f, gate, gate_rows, pw, pb, nw, nb, post, pre, alpha, beta, eps):
    y = alpha * x
    if f is not None:
        u = norm(f, post, pw, pb, eps)
        if gate is not None:
            u = u * gate[torch.arange(x.shape[0], device=x.device) // gate_rows]
        y = y + beta * u
    return y, norm(y, pre, nw, nb, eps)
