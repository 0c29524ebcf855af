"""A field over 3D points whose capacity is a mixture of experts, trained with the block's operators.

    python examples/expert_field.py [--steps 200] [--tokens 8192] [--max-norm 1.0] [--answer-bits 4]

Points are embedded as sines and cosines (D features); one residual block

    h = rmsnorm(x),  (experts, weights) = route(h Wr),  e = relu(h W1_e) W2_e,  f = sum_j weights_j e_j,
    y = x + gate * rmsnorm(f)

and a linear map to colours follow; the loss is the mean squared error against a synthetic scene of boxes.  The block's
products run in 8 bits with a scale for each block of 128, forward and backward; master weights and Adam are fp32.
Everything but the embedding, the colour map and Adam goes through the launchers of include/experts_abi.h; with a largest
norm the gradients are clipped by those of include/grad_abi.h.  A few points at a time are answered by the whole layer in
one call (ExpertBlock.answer), from weights in 8 bits or in 4, which the run ends with.
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
CODES = {torch.float32: P.DATA_F32, torch.float16: P.DATA_F16, torch.bfloat16: P.DATA_BF16}


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
        o = P.Fp8QuantOption(rows=self.rows, cols=self.cols, batch=self.batch, blockRows=self.block_rows, srcType=CODES[x.dtype],
                             slotsPerRow=slots, srcRows=x.shape[-2], srcStride=x.stride(-2),
                             srcBatchStride=x.stride(0) if x.dim() == 3 else 0, gateStride=gate.stride(0) if gate is not None else 0)
        P.launch("launchFp8Quantize", C.byref(o), x, order, weights, gate, self.q, self.s, self.qt, self.st, stream())
        return self


def product(a, a_scales, b, b_scales, out, m, n, k, experts, grouping, scale_rows, offsets, relu=False):
    o = P.Fp8ProductOption(m=m, n=n, k=k, numExperts=experts, grouping=grouping, scaleRowsB=scale_rows, activation=int(relu),
                           outType=P.DATA_F32 if out.dtype == torch.float32 else TYPE, outStride=out.stride(-2))
    P.launch("launchFp8Product", C.byref(o), a, a_scales, b, b_scales, offsets, out, stream())
    return out


class Fp4:
    """All experts' matrices [experts, rows, cols] as e2m1 values with a scale for each 32 columns."""

    def __init__(self, w):
        E, rows, cols = w.shape
        self.q = empty(E, rows, P.fp4_pitch(cols), dtype=torch.uint8)
        self.s = empty(E, rows, P.fp4_scale_pitch(cols), dtype=torch.uint8)
        o = P.Fp4QuantOption(rows=rows, cols=cols, batch=E, scaleRule=P.FP4_SCALE_COVER, srcType=CODES[w.dtype], slotsPerRow=0,
                             srcRows=rows, srcStride=w.stride(1), srcBatchStride=w.stride(0))
        P.launch("launchFp4Quantize", C.byref(o), w, None, self.q, self.s, stream())


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

    def prepare(self, bits=8):
        """The weights' form for answer(), in 8 bits or 4, once after training."""
        self.bits = bits
        if bits == 4:
            self.served = Fp4(self.p["w1"]), Fp4(self.p["w2"])
        else:
            self.served = self.w1.quantize(self.p["w1"]), self.w2.quantize(self.p["w2"])

    def answer(self, x):
        """forward() for up to 64 rows: the layer of experts in one call, neither tokens nor hidden activations quantised."""
        p, T, D = self.p, x.shape[0], self.dim
        h, f, y = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        o = self.norm_option(P.NORM_NONE, P.NORM_RMS, 0, 1.0)
        P.launch("launchNormGateResidual", C.byref(o), x, None, None, None, None, p["norm_in"], None, None, h, T, stream())
        o = P.ExpertLayerOption(route=self.route_option(), dim=D, hidden=self.hidden, activation=P.EXPERT_RELU, gated=0,
                                weightFormat=P.EXPERT_FP4 if self.bits == 4 else P.EXPERT_FP8, scaleRows=1 if self.bits == 4 else 128,
                                dataType=TYPE, routerType=P.DATA_F32, strideX=D, strideOut=D)
        w1, w2 = self.served
        P.launch("launchExpertLayer", C.byref(o), h, p["router"], None, w1.q, w1.s, w2.q, w2.s, f, T, stream())
        o = self.norm_option(P.NORM_RMS, P.NORM_NONE, T, 1.0)
        P.launch("launchNormGateResidual", C.byref(o), x, f, p["gate"].to(DT), p["norm_out"], None, None, None, y, None, T, stream())
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


def clip(grads, max_norm, loss_scale):
    """Scales gradients in place to at most max_norm, which counts without the loss scale.  Their norm before."""
    norm = empty(1, dtype=torch.float32)
    list_ = (P.GradTensor * len(grads))(*[P.GradTensor(data=t.data_ptr(), n=t.numel(), dataType=CODES[t.dtype]) for t in grads])
    P.launch("launchGradNormClip", list_, len(grads), P.GRAD_NORM_2, loss_scale, max_norm, P.GRAD_NONFINITE_ZERO, norm, stream())
    return norm


def colours(block, head, points):
    """The field's colours at up to 64 points, by the block's answers."""
    return block.answer(embed(points, block.dim).to(DT)).float() @ head.t()


def train(steps=200, tokens=8192, dim=256, hidden=512, experts=8, topk=2, lr=2e-3, loss_scale=1024.0, verbose=True, max_norm=None,
          answer_bits=None):
    """The losses of the steps; with answer_bits also of 64 points that the trained block answers with weights of so many."""
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
        if max_norm is not None:
            clip(list(grad.values()), max_norm, loss_scale)
        for n, t in params.items():
            d = grad[n] / loss_scale
            m[n].mul_(0.9).add_(d, alpha=0.1)
            v[n].mul_(0.99).addcmul_(d, d, value=0.01)
            t.addcdiv_(m[n] / (1 - 0.9 ** step), (v[n] / (1 - 0.99 ** step)).sqrt() + 1e-8, value=-lr)
        if verbose and (step == 1 or step % 50 == 0):
            print(f"step {step} loss {float(losses[-1]):.5f}", flush=True)
    if answer_bits:
        block.prepare(answer_bits)
        points = torch.rand(P.EXPERT_LAYER_TOKENS, 3, generator=g, device="cuda")
        losses.append((colours(block, params["head"], points) - scene(points)).square().mean())
        if verbose:
            print(f"{len(points)} points answered with weights of {answer_bits} bits: loss {float(losses[-1]):.5f}", flush=True)
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--max-norm", type=float, default=None)
    ap.add_argument("--answer-bits", type=int, choices=[4, 8], default=8)
    a = ap.parse_args()
    train(a.steps, a.tokens, max_norm=a.max_norm, answer_bits=a.answer_bits)
