"""A field over 3D points whose capacity is a mixture of experts, trained with the block's operators.

    python examples/expert_field.py [--steps 200] [--tokens 8192]

Points are embedded as sines and cosines (D features); one residual block

    h = rmsnorm(x),  (experts, weights) = route(h Wr),  e = relu(h W1_e) W2_e,  f = sum_j weights_j e_j,
    y = x + gate * rmsnorm(f)

and a linear map to colours follow; the loss is the mean squared error against a synthetic scene of boxes.  The block's
products run in 8 bits with a scale for each block of 128, forward and backward; master weights and Adam are fp32.
Everything but the embedding, the colour map and Adam goes through the launchers of include/experts_abi.h.
"""
from __future__ import annotations

import argparse
import ctypes as C
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
P = importlib.import_module("3dmaker_amd")

TYPE, DT = P.DATA_F16, torch.float16


def stream():
    return torch.cuda.current_stream().cuda_stream


def empty(*shape, dtype=DT):
    return torch.empty(*shape, dtype=dtype, device="cuda")


class Fp8:
    """An 8-bit matrix and, on request, its transpose (include/experts_abi.h)."""

    def __init__(self, rows, cols, batch=1, block_rows=1, row_side=True, transposed=False):
        def side(r, c):
            blocks = -(-r // block_rows)
            return empty(batch, r, P.fp8_pitch(c), dtype=torch.uint8), empty(batch, blocks, P.fp8_scale_pitch(c), dtype=torch.uint8)

        self.rows, self.cols, self.batch, self.block_rows = rows, cols, batch, block_rows
        self.q, self.s = side(rows, cols) if row_side else (None, None)
        self.qt, self.st = side(cols, rows) if transposed else (None, None)

    def quantize(self, x, order=None, slots=1, weights=None, gate=None):
        code = {torch.float32: P.DATA_F32, torch.float16: P.DATA_F16, torch.bfloat16: P.DATA_BF16}[x.dtype]
        o = P.Fp8QuantOption(rows=self.rows, cols=self.cols, batch=self.batch, blockRows=self.block_rows, srcType=code,
                             slotsPerRow=slots, srcRows=x.shape[-2], srcStride=x.stride(-2),
                             srcBatchStride=x.stride(0) if x.dim() == 3 else 0, gateStride=gate.stride(0) if gate is not None else 0)
        P.launch("launchFp8Quantize", C.byref(o), x, order, weights, gate, self.q, self.s, self.qt, self.st, stream())
        return self


def product(a, a_scales, b, b_scales, out, m, n, k, experts, grouping, scale_rows, offsets, relu=False):
    o = P.Fp8ProductOption(m=m, n=n, k=k, numExperts=experts, grouping=grouping, scaleRowsB=scale_rows, activation=int(relu),
                           outType=P.DATA_F32 if out.dtype == torch.float32 else TYPE, outStride=out.stride(-2))
    P.launch("launchFp8Product", C.byref(o), a, a_scales, b, b_scales, offsets, out, stream())
    return out


class ExpertBlock:
    """y = x + gate * rmsnorm(sum_j w_j relu(h W1_e(j)) W2_e(j)),  h = rmsnorm(x): forward and backward."""

    def __init__(self, dim, hidden, experts, topk, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.dim, self.hidden, self.experts, self.topk = dim, hidden, experts, topk
        self.p = dict(router=rand(experts, dim) * dim ** -0.5, w1=rand(experts, hidden, dim) * dim ** -0.5,
                      w2=rand(experts, dim, hidden) * hidden ** -0.5, norm_in=torch.ones(dim, device="cuda"),
                      norm_out=torch.ones(dim, device="cuda"), gate=torch.full((1, dim), 0.5, device="cuda"))
        self.w1 = Fp8(hidden, dim, experts, 128, transposed=True)
        self.w2 = Fp8(dim, hidden, experts, 128, transposed=True)

    def route_option(self):
        return P.RouteOption(numExperts=self.experts, topK=self.topk, scoreType=P.ROUTE_SOFTMAX, numGroups=1, topGroups=1,
                             groupScore=2, renormalize=1, scale=1.0, logitsType=P.DATA_F32)

    def norm_option(self, post, pre, gate_rows, alpha):
        D = self.dim
        return P.NormGateOption(dim=D, postNorm=post, preNorm=pre, gateRows=gate_rows, residualScale=alpha, blockScale=1.0,
                                epsilon=1e-6, dataType=TYPE, strideX=D, strideF=D, strideGate=D, strideY=D, strideH=D)

    def forward(self, x):
        p, T, D, H, E, k = self.p, x.shape[0], self.dim, self.hidden, self.experts, self.topk
        L = P.lib()
        self.x, self.h = x, torch.empty_like(x)
        o = self.norm_option(P.NORM_NONE, P.NORM_RMS, 0, 1.0)
        P.launch("launchNormGateResidual", C.byref(o), x, None, None, None, None, p["norm_in"], None, None, self.h, T, stream())
        self.logits = self.h.float() @ p["router"].t()
        self.index, self.weight = empty(T, k, dtype=torch.int32), empty(T, k, dtype=torch.float32)
        P.launch("launchRouteExperts", C.byref(self.route_option()), self.logits, E, None, self.index, self.weight, T, stream())
        cap = self.cap = L.routePlanCapacity(T, k, E, 128)
        self.offsets, self.order = empty(E + 1, dtype=torch.int32), empty(cap, dtype=torch.int32)
        self.position = empty(T, k, dtype=torch.int32)
        P.launch("launchRoutePlan", self.index, T, k, E, 128, cap, self.offsets, self.order, self.position, stream())
        self.w1.quantize(p["w1"])
        self.w2.quantize(p["w2"])
        rows = Fp8(cap, D).quantize(self.h, self.order, k)
        # rows outside all segments are neither written by the products nor read by the next ones
        self.hidden_rows = product(rows.q, rows.s, self.w1.q, self.w1.s, empty(cap, H), cap, H, D, E, P.PRODUCT_ROWS, 128,
                                   self.offsets, relu=True)
        act = Fp8(cap, H).quantize(self.hidden_rows)
        self.rows = product(act.q, act.s, self.w2.q, self.w2.s, empty(cap, D), cap, D, H, E, P.PRODUCT_ROWS, 128, self.offsets)
        self.f = empty(T, D)
        P.launch("launchExpertCombine", D, TYPE, self.rows, cap, D, self.position, self.weight, self.f, D, T, k, stream())
        self.gate = p["gate"].to(DT)
        y = torch.empty_like(x)
        o = self.norm_option(P.NORM_RMS, P.NORM_NONE, T, 1.0)
        P.launch("launchNormGateResidual", C.byref(o), x, self.f, self.gate, p["norm_out"], None, None, None, y, None, T, stream())
        return y

    def backward(self, dy):
        """dL/dx and the parameters' gradients (fp32)."""
        p, T, D, H, E, k, cap = self.p, dy.shape[0], self.dim, self.hidden, self.experts, self.topk, self.cap
        grad = {n: torch.empty_like(v) for n, v in p.items()}
        dx, df, dgate = torch.empty_like(dy), torch.empty_like(dy), empty(1, D)
        o = self.norm_option(P.NORM_RMS, P.NORM_NONE, T, 1.0)
        P.launch("launchNormGateResidualBackward", C.byref(o), self.x, self.f, self.gate, p["norm_out"], None, None, None, dy, None,
                 dx, df, dgate, grad["norm_out"], None, None, None, T, stream())
        grad["gate"] = dgate.float()
        dweight = empty(T, k, dtype=torch.float32)
        P.launch("launchExpertCombineBackward", D, TYPE, self.rows, cap, D, self.position, df, D, dweight, T, k, stream())
        # second product: rows' gradient weight * df, gathered by the order; both its sides are needed
        g2 = Fp8(cap, D, transposed=True).quantize(df, self.order, k, self.weight)
        act = Fp8(cap, H, row_side=False, transposed=True).quantize(self.hidden_rows)
        product(g2.qt, g2.st, act.qt, act.st, grad["w2"], D, H, cap, E, P.PRODUCT_SUM, 1, self.offsets)
        dhid = product(g2.q, g2.s, self.w2.qt, self.w2.st, empty(cap, H), cap, H, D, E, P.PRODUCT_ROWS, 128, self.offsets)
        # first product: behind the ReLU
        g1 = Fp8(cap, H, transposed=True).quantize(dhid, gate=self.hidden_rows)
        rows = Fp8(cap, D, row_side=False, transposed=True).quantize(self.h, self.order, k)
        product(g1.qt, g1.st, rows.qt, rows.st, grad["w1"], H, D, cap, E, P.PRODUCT_SUM, 1, self.offsets)
        drows = product(g1.q, g1.s, self.w1.qt, self.w1.st, empty(cap, D), cap, D, H, E, P.PRODUCT_ROWS, 128, self.offsets)
        dh = empty(T, D)
        P.launch("launchExpertCombine", D, TYPE, drows, cap, D, self.position, None, dh, D, T, k, stream())
        dlogits = torch.empty_like(self.logits)
        P.launch("launchRouteExpertsBackward", C.byref(self.route_option()), self.logits, E, self.index, dweight, dlogits, E, T,
                 stream())
        grad["router"] = dlogits.t().contiguous() @ self.h.float()
        dh += (dlogits @ p["router"]).to(DT)
        o = self.norm_option(P.NORM_NONE, P.NORM_RMS, 0, 1.0)
        dx_in = torch.empty_like(dx)
        P.launch("launchNormGateResidualBackward", C.byref(o), self.x, None, None, None, None, p["norm_in"], None, dx, dh, dx_in,
                 None, None, None, None, grad["norm_in"], None, T, stream())
        return dx_in, grad


def scene(points):
    """Colours of a synthetic scene: a checker of boxes, each octant with its own tint."""
    cell = torch.floor(points * 4).long()
    on = (cell.sum(1) % 2).float()[:, None]
    octant = (points > 0.5).float()
    return 0.1 + 0.8 * on * octant + 0.1 * torch.sin(6 * points)


def embed(points, dim):
    n = dim // 6
    f = 2.0 ** torch.linspace(0, 5, n, device=points.device) * torch.pi
    a = points[:, :, None] * f
    e = torch.cat([torch.sin(a), torch.cos(a)], 1).reshape(points.shape[0], -1)
    return torch.nn.functional.pad(e, (0, dim - e.shape[1]))


def train(steps=200, tokens=8192, dim=256, hidden=512, experts=8, topk=2, lr=2e-3, loss_scale=1024.0, verbose=True):
    """The losses of the steps."""
    block = ExpertBlock(dim, hidden, experts, topk)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    params = dict(block.p, head=torch.randn(3, dim, generator=g, device="cuda") * dim ** -0.5)
    m, v = ({n: torch.zeros_like(t) for n, t in params.items()} for _ in range(2))
    losses = []
    for step in range(1, steps + 1):
        points = torch.rand(tokens, 3, generator=g, device="cuda")
        y = block.forward(embed(points, dim).to(DT))
        err = y.float() @ params["head"].t() - scene(points)
        losses.append(err.square().mean())
        dout = err * (2.0 / err.numel()) * loss_scale
        _, grad = block.backward((dout @ params["head"]).to(DT))
        grad["head"] = dout.t() @ y.float()
        for n, t in params.items():
            d = grad[n] / loss_scale
            m[n].mul_(0.9).add_(d, alpha=0.1)
            v[n].mul_(0.99).addcmul_(d, d, value=0.01)
            t.addcdiv_(m[n] / (1 - 0.9 ** step), (v[n] / (1 - 0.99 ** step)).sqrt() + 1e-8, value=-lr)
        if verbose and (step == 1 or step % 50 == 0):
            print(f"step {step} loss {float(losses[-1]):.5f}", flush=True)
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--tokens", type=int, default=8192)
    a = ap.parse_args()
    train(a.steps, a.tokens)
