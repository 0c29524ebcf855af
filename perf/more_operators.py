"""Operators that serve a mixture-of-experts block in few bits and for few tokens, and the clipping that trains it, as
cases that can be timed and compared.

Kinds:
  fp4          launchFp4Quantize + launchFp4Product: activations times a weight matrix, both in 4 bits with a power-of-two
               scale for each block of 32
  fp4_experts  gather + quantise, the experts' products in 4 bits, launchExpertCombine
  layer        launchExpertLayer: router, routing, both products of each token's experts, their weighted sum, for few tokens
  clip         launchGradNormClip: the norm over all gradients, and the gradients scaled to at most a given norm
  grad_norm    launchGradNorm: that norm alone

Sizes: the example's block, sample batches and networks of the repository's configurations, and generic widths.
Everything is made from the seed with torch generators.
"""
from __future__ import annotations

import ctypes as C
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def _pkg():
    return importlib.import_module("3dmaker_amd")


def listed():
    return [
        # One token by a square matrix in serving: latency and the weights' bytes.
        dict(name="fp4_token", kind="fp4", rows=1, n=4096, k=4096, rule="cover", dtype="bf16"),
        # A ragged batch through a wide layer: the matrix cores.
        dict(name="fp4_dense", kind="fp4", rows=8191, n=5120, k=4096, rule="floor", dtype="bf16"),
        # A batch of a field's experts, rows by expert.
        dict(name="fp4_experts", kind="fp4_experts", tokens=1 << 15, experts=8, topk=2, n=2048, k=1024, rule="cover",
             dtype="f16"),
        # The example's block queried at one point: latency alone.
        dict(name="layer_token", kind="layer", tokens=1, experts=8, topk=2, dim=256, hidden=512, act="relu", gated=False,
             weights="fp8", score="softmax", groups=1, kept=1, bias=False, renorm=True, router="f32", dtype="f16"),
        # A few tokens of many experts in 4 bits: half of the experts' bytes, in small pieces.
        dict(name="layer_few", kind="layer", tokens=7, experts=64, topk=6, dim=2048, hidden=1024, act="silu", gated=True,
             weights="fp4", score="softmax", groups=1, kept=1, bias=False, renorm=False, router="bf16", dtype="bf16"),
        # A ragged batch of queries over most of 128 experts in groups, balanced by a bias: the weights' bytes.
        dict(name="layer_groups", kind="layer", tokens=27, experts=128, topk=8, dim=2048, hidden=768, act="silu", gated=True,
             weights="fp8", score="sigmoid", groups=8, kept=4, bias=True, renorm=True, router="f32", dtype="bf16"),
        # The most tokens a call takes, many for each expert, unrounded activations.
        dict(name="layer_most", kind="layer", tokens=64, experts=8, topk=2, dim=4096, hidden=2048, act="gelu", gated=False,
             weights="fp8", score="softmax", groups=1, kept=1, bias=False, renorm=True, router="f32", dtype="f32"),
        # The gradients of the two heads (32-64-16 and 32-64-64-8): latency.
        dict(name="clip_heads", kind="clip", sizes="heads", total=0, count=10, packed=False, dtype="f32", over=2.0),
        # Heads and a hash table of 16 levels of 2^19 entries, clipped: memory, one tensor above all others.
        dict(name="clip_field", kind="clip", sizes="field", total=1 << 24, count=11, packed=False, dtype="f32", over=1.7),
        # Many tensors of a mixture of experts in 16 bits, odd lengths, far above the norm.
        dict(name="clip_many", kind="clip", sizes="many", total=400_000_003, count=390, packed=False, dtype="bf16",
             over=30.0),
        # Small tensors, as norms and biases are, for the log of a step.
        dict(name="norm_small", kind="grad_norm", sizes="many", total=70_001, count=61, packed=True, dtype="f16", over=1.0),
        # The example's parameters at a larger width, in 32 bits.
        dict(name="norm_experts", kind="grad_norm", sizes="many", total=100_000_007, count=23, packed=False, dtype="f32",
             over=1.0),
    ]


def _size(rng, lo, hi):
    """Log-uniform, odd as often as not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.5 else n & ~15 or n))


def _width(rng, lo, hi, step):
    """Log-uniform multiple of `step`, any width one time in three."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n if rng.random() < 1 / 3 else max(1, n // step) * step))


LAYER_WEIGHTS = 128 * 3 * 2048 * 768  # the largest listed layer's


def draw(rng):
    kind = rng.choice(["fp4", "fp4", "fp4_experts", "layer", "layer", "layer", "clip", "clip", "grad_norm"])
    dtype = rng.choice(list(TYPES))
    if kind == "fp4":
        return dict(kind=kind, rows=_size(rng, 1, 8191), n=_width(rng, 64, 5120, 64), k=_width(rng, 32, 4096, 64),
                    rule=rng.choice(["floor", "cover"]), dtype=dtype)
    if kind == "fp4_experts":
        return dict(kind=kind, tokens=_size(rng, 1, 1 << 15), experts=rng.choice([2, 4, 8, 16, 32]), topk=rng.randint(1, 2),
                    n=_width(rng, 64, 2048, 64), k=_width(rng, 64, 1024, 64), rule=rng.choice(["floor", "cover"]),
                    dtype=rng.choice(["f16", "bf16"]))
    if kind == "layer":
        experts = rng.choice([4, 8, 16, 60, 64, 128])
        groups = rng.choice([1, 1, 4])
        kept = 1 if groups == 1 else rng.randint(2, groups)
        gated = rng.random() < 0.5
        dim = _width(rng, 64, 4096, 64)
        hidden = _width(rng, 64, max(65, min(2048, LAYER_WEIGHTS // (experts * dim * (3 if gated else 2)))), 64)
        return dict(kind=kind, tokens=_size(rng, 1, 64), experts=experts,
                    topk=rng.randint(1, max(1, min(8, experts // groups * kept - 1))), dim=dim, hidden=hidden,
                    act=rng.choice(["relu", "silu", "gelu"]), gated=gated, weights=rng.choice(["fp8", "fp4"]),
                    score=rng.choice(["softmax", "sigmoid"]), groups=groups, kept=kept, bias=rng.random() < 0.5,
                    renorm=rng.random() < 0.7, router=rng.choice(list(TYPES)), dtype=dtype)
    count = _size(rng, 1, 390)
    return dict(kind=kind, sizes="many", total=_size(rng, 16 * count, 100_000_007), count=count,
                packed=rng.random() < 0.3, dtype=dtype, over=rng.choice([0.5, 1.5, 30.0]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (seed + 1))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _weights(g, fmt, experts, rows, cols):
    """Random matrices as a program keeps them, quantised once."""
    w = _randn(g, experts, rows, cols) / math.sqrt(cols)
    if fmt == "fp8":
        return _store8(*_quantize8(w))
    return _store4(*_quantize4(w, "cover"))


def _capacity(case):
    """Rows of the plan: every slot, and each expert's segment filled up to whole blocks of 128."""
    slots, experts = case["tokens"] * case["topk"], case["experts"]
    return -(-(slots + min(experts, slots) * 127) // 128) * 128


def _tensor_sizes(case):
    if case["sizes"] in ("heads", "field"):
        heads = [64 * 32, 64, 16 * 64, 16, 64 * 32, 64, 64 * 64, 64, 8 * 64, 8]
        return heads + ([case["total"]] if case["sizes"] == "field" else [])
    r = random.Random(case["total"] + case["count"])
    cut = [r.random() ** 3 + 1e-4 for _ in range(case["count"])]  # some large, most small
    sizes = [max(1, int(case["total"] * c / sum(cut))) for c in cut]
    sizes[0] += case["total"] - sum(sizes) if case["total"] > sum(sizes) else 0
    return sizes


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    dt, code = TYPES[case["dtype"]]
    s = dict(case=case, dt=dt, code=code)
    if kind == "fp4":
        M, N, K = case["rows"], case["n"], case["k"]
        s["x"] = _randn(g, M, K).to(dt)
        s["w"], s["w_scale"] = _weights(g, "fp4", 1, N, K)
        s["xq"], s["xs"] = _buffers4(M, K)
        s["out"] = torch.empty(M, N, dtype=dt, device=DEV)
    elif kind == "fp4_experts":
        T, E, N, K, k = case["tokens"], case["experts"], case["n"], case["k"], case["topk"]
        # distinct experts, some of them asked for more than others, and the plan that a program has from the router
        u = torch.rand(T, E, generator=g, device=DEV).clamp(1e-7, 1 - 1e-7)
        score = _randn(g, 1, E) * 0.7 - torch.log(-torch.log(u))
        indices = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
        s["indices"], s["weights"] = indices, torch.softmax(_randn(g, T, k), 1).contiguous()
        cap = _capacity(case)
        s["offsets"], s["order"], s["position"] = _plan(indices, E, cap)
        s["longest"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["x"] = _randn(g, T, K).to(dt)
        s["w"], s["w_scale"] = _weights(g, "fp4", E, N, K)
        s["xq"], s["xs"] = _buffers4(cap, K)
        s["rows"] = torch.empty(cap, N, dtype=dt, device=DEV)
        s["out"] = torch.empty(T, N, dtype=dt, device=DEV)
    elif kind == "layer":
        E, D, H = case["experts"], case["dim"], case["hidden"]
        s["router"] = (_randn(g, E, D) * 1.5 / math.sqrt(D)).to(TYPES[case["router"]][0])
        s["bias"] = _randn(g, E) * 0.05 if case["bias"] else None
        s["x"] = _layer_tokens(case, g, s["router"], s["bias"], dt)
        s["w1"], s["w1_scale"] = _weights(g, case["weights"], E, H * (2 if case["gated"] else 1), D)
        s["w2"], s["w2_scale"] = _weights(g, case["weights"], E, D, H)
        s["out"] = torch.empty(case["tokens"], D, dtype=dt, device=DEV)
    else:
        sizes = _tensor_sizes(case)
        # gradients of a step whose loss is scaled by 128, of another size in each tensor
        spread = torch.exp2(torch.randint(-6, 3, (len(sizes),), generator=g, device=DEV).float()).tolist()
        s["flat"], s["grads"] = _flat(case, sizes, dt)
        for t, a in zip(s["grads"], spread):
            t.copy_(_randn(g, t.numel()) * (0.5 * a))
        s["scale"] = 128.0
        norm = math.sqrt(sum(float(torch.sum(t.float().square(), dtype=torch.float64)) for t in s["grads"])) / s["scale"]
        s["max_norm"] = _f32(norm / case["over"])
        s["norm"] = torch.empty(1, dtype=torch.float32, device=DEV)
        if kind == "clip":
            s["clipped"], s["views"] = _flat(case, sizes, dt)
    return s


def _flat(case, sizes, dt):
    """One buffer with room for tensors of these sizes, and the tensors: each from a multiple of 128 elements on, or back
    to back as a bucket for a collective holds them."""
    step = 1 if case["packed"] else 128
    at = [0]
    for n in sizes:
        at.append(_up(at[-1] + n, step))
    flat = torch.zeros(at[-1], dtype=dt, device=DEV)
    return flat, [flat[a:a + n] for a, n in zip(at, sizes)]


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _layer_tokens(case, g, router, bias, dt):
    """Tokens whose selection does not hang on the last bits of a score: the last expert (or group) that is taken and the
    first that is not are 1e-4 apart."""
    T, E, G, D = case["tokens"], case["experts"], case["groups"], case["dim"]
    x = _randn(g, T, D).to(dt)
    for _ in range(50):
        z = x.double() @ router.double().t().contiguous()
        c = torch.softmax(z, 1) if case["score"] == "softmax" else torch.sigmoid(z)
        c = c if bias is None else c + bias.double()
        bad = torch.zeros(T, dtype=torch.bool, device=DEV)

        def near(v, n):
            v = torch.sort(v, dim=1, descending=True).values
            return (v[:, n - 1] - v[:, n]) < 1e-4 * v[:, n - 1].abs()

        if G > 1:
            best = torch.sort(c.view(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
            if case["kept"] < G:
                bad |= near(best, case["kept"])
            keep = torch.zeros(T, G, dtype=torch.bool, device=DEV)
            keep.scatter_(1, torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["kept"]], True)
            c = c.masked_fill(~keep.repeat_interleave(E // G, 1), -1e9)
        if case["topk"] < E:
            bad |= near(c, case["topk"])
        n = int(bad.sum())
        if n == 0:
            break
        x[bad] = _randn(g, n, D).to(dt)
    return x


def _plan(indices, experts, capacity):
    """Stable counting sort of the slots by expert, each expert's rows from a multiple of 128 on."""
    flat = indices.reshape(-1).long()
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.cumsum((counts + 127) // 128 * 128, 0)
    by = torch.sort(flat, stable=True).indices
    first = torch.cumsum(counts, 0) - counts
    at = offsets[flat[by]] + torch.arange(flat.numel(), device=flat.device) - first[flat[by]]
    order = torch.full((capacity,), -1, dtype=torch.int32, device=flat.device)
    order[at] = by.to(torch.int32)
    position = torch.empty(flat.numel(), dtype=torch.int32, device=flat.device)
    position[by] = at.to(torch.int32)
    return offsets.to(torch.int32), order, position.view(indices.shape)


# ---------------------------------------------------------------------------
# the stored forms: e4m3 with a scale for 128 x 128, e2m1 with a scale for 32 of a row
# ---------------------------------------------------------------------------

def _up(n, m):
    return -(-n // m) * m


def _power(e):
    """2^e in 32 bits, e in -126 .. 127."""
    return ((127 + e.to(torch.int32)) << 23).view(torch.float32)


def _quantize8(x):
    """x [B, R, C] to e4m3 and the scales' exponents [B, R', C']: the smallest power of two that brings a block of
    128 x 128 within 448."""
    B, R, Cc = x.shape
    rb, cb = -(-R // 128), -(-Cc // 128)
    p = torch.nn.functional.pad(x, (0, cb * 128 - Cc, 0, rb * 128 - R)).view(B, rb, 128, cb, 128)
    m, e = torch.frexp(p.abs().amax((2, 4)))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-126, 126)
    q = (p * _power(-e)[:, :, None, :, None]).reshape(B, rb * 128, cb * 128)[:, :R, :Cc]
    return q.to(torch.float8_e4m3fn), e


def _store8(q, e):
    B, R, Cc = q.shape
    bytes_ = torch.zeros(B, R, _up(Cc, 128), dtype=torch.uint8, device=DEV)
    bytes_[:, :, :Cc] = q.view(torch.uint8)
    scale = torch.full((B, e.shape[1], _up(e.shape[2], 4)), 127, dtype=torch.uint8, device=DEV)
    scale[:, :, :e.shape[2]] = (e + 127).to(torch.uint8)
    return bytes_, scale


def _values8(bytes_, scale, cols):
    """The 32-bit values of stored matrices [B, R, cols]."""
    B, R, pitch = bytes_.shape
    s = (scale.to(torch.int32) << 23).view(torch.float32)[:, :, :pitch // 128].repeat_interleave(128, 1)[:, :R]
    return (bytes_.view(torch.float8_e4m3fn).float().view(B, R, -1, 128) * s[:, :, :, None]).view(B, R, pitch)[:, :, :cols]


def _round4(v):
    """To the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6, ties to the even one; beyond 6 is 6."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _quantize4(x, rule):
    """x [B, R, C] to e2m1 values and the scales' exponents [B, R, C / 32]: the power of two of the block's largest over
    that of the type's (floor), or the smallest that brings the block within 6 (cover)."""
    B, R, Cc = x.shape
    pitch = _up(Cc, 128)
    p = torch.nn.functional.pad(x, (0, pitch - Cc)).view(B, R, pitch // 32, 32)
    m, e = torch.frexp(p.abs().amax(3))
    e = e - 3 if rule == "floor" else torch.where(m <= 0.75, e - 3, e - 2)
    e = e.clamp(-126, 126)
    return _round4(p * _power(-e)[:, :, :, None]).view(B, R, pitch), e


def _dequantize4(q, e, cols):
    B, R, pitch = q.shape
    return (q.view(B, R, -1, 32) * _power(e)[:, :, :, None]).view(B, R, pitch)[:, :, :cols]


def _store4(q, e):
    """As the entry points take it: two values a byte, the even column in the low four bits; scale bytes."""
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code |= torch.signbit(q).to(torch.uint8) << 3
    return code[:, :, 0::2] | (code[:, :, 1::2] << 4), (e + 127).to(torch.uint8)


def _values4(bytes_, scale, cols):
    """The 32-bit values of stored matrices [B, R, cols]."""
    B, R, half = bytes_.shape
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=bytes_.device)
    b = bytes_.to(torch.int32)
    q = torch.stack([table[b & 15], table[b >> 4]], 3).view(B, R, half // 16, 32)
    return (q * (scale.to(torch.int32) << 23).view(torch.float32)[:, :, :, None]).view(B, R, half * 2)[:, :, :cols]


def _buffers4(rows, cols):
    pitch = _up(cols, 128)
    return (torch.empty(rows, pitch // 2, dtype=torch.uint8, device=DEV),
            torch.empty(rows, pitch // 32, dtype=torch.uint8, device=DEV))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _fp4_plain(s):
    case = s["case"]
    x = _dequantize4(*_quantize4(s["x"].float()[None], case["rule"]), case["k"])[0]
    w = _values4(s["w"], s["w_scale"], case["k"])[0]
    return (x @ w.t().contiguous()).to(s["dt"])


def _fp4_experts_plain(s):
    case, k = s["case"], s["case"]["topk"]
    slot = s["order"].long().clamp(min=0)
    x = s["x"].float()[slot // k] * (s["order"] >= 0)[:, None]
    x = _dequantize4(*_quantize4(x[None], case["rule"]), case["k"])[0]
    w = _values4(s["w"], s["w_scale"], case["k"])
    o = s["offsets"].long()
    at = o[:-1, None] + torch.arange(s["longest"], device=DEV)  # each expert's places
    fine = at < o[1:, None]
    at = torch.where(fine, at, 0)
    y = torch.bmm(x[at] * fine[:, :, None], w.transpose(1, 2).contiguous())
    rows = torch.zeros(x.shape[0] + 1, case["n"], device=DEV)
    rows[torch.where(fine, at, x.shape[0])] = y
    return (rows[s["position"].long()] * s["weights"][:, :, None]).sum(1).to(s["dt"])


SCALE = 1.5  # the routing weights' factor


def _activation(name, v):
    if name == "relu":
        return torch.where(v > 0, v, 0.0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))


def _layer_plain(s):
    """All tokens through all experts, times weights that are 0 for most."""
    c = s["case"]
    T, E, G, D, H = c["tokens"], c["experts"], c["groups"], c["dim"], c["hidden"]
    x = s["x"].float()
    z = x @ s["router"].float().t().contiguous()
    if c["score"] == "softmax":
        p = torch.exp(z - z.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-z))
    v = p if s["bias"] is None else p + s["bias"]
    if G > 1:
        best = torch.sort(v.view(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["kept"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        v = v.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    idx = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :c["topk"]]
    w = p.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    share = torch.zeros(T, E, device=DEV).scatter_(1, idx, w * SCALE)
    values = _values8 if c["weights"] == "fp8" else _values4
    h = torch.bmm(x.expand(E, T, D).contiguous(), values(s["w1"], s["w1_scale"], D).transpose(1, 2).contiguous())
    a = _activation(c["act"], h[:, :, :H])
    if c["gated"]:
        a = a * h[:, :, H:]
    y = torch.bmm(a.contiguous(), values(s["w2"], s["w2_scale"], H).transpose(1, 2).contiguous())
    return (y * share.t()[:, :, None]).sum(0).to(s["dt"])


def _norm_plain(s):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in s["grads"]:
        total = total + torch.sum(t.float() * t.float(), dtype=torch.float64)
    return (torch.sqrt(total) / s["scale"]).to(torch.float32)


def _clip_plain(s):
    norm = _norm_plain(s)
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
    return dict(norm=norm.view(1), clipped=(s["flat"].float() * factor).to(s["dt"]))


PLAIN = {"fp4": _fp4_plain, "fp4_experts": _fp4_experts_plain, "layer": _layer_plain, "clip": _clip_plain,
         "grad_norm": lambda s: _norm_plain(s).view(1)}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

def _stream():
    return torch.cuda.current_stream().cuda_stream


def _quantize_own(P, s, rows, order, slots):
    c = s["case"]
    if "quant" not in s:
        rule = P.FP4_SCALE_FLOOR if c["rule"] == "floor" else P.FP4_SCALE_COVER
        s["quant"] = P.Fp4QuantOption(rows=rows, cols=c["k"], batch=1, scaleRule=rule, srcType=s["code"], slotsPerRow=slots,
                                      srcRows=s["x"].shape[0], srcStride=c["k"], srcBatchStride=0)
    P.launch("launchFp4Quantize", C.byref(s["quant"]), s["x"], order, s["xq"], s["xs"], _stream())


def _fp4_own(s):
    P, c = _pkg(), s["case"]
    M, N, K = c["rows"], c["n"], c["k"]
    _quantize_own(P, s, M, None, 1)
    if "product" not in s:
        s["product"] = P.Fp4ProductOption(m=M, n=N, k=K, numExperts=1, grouping=P.PRODUCT_DENSE, activation=0,
                                          outType=s["code"], outStride=N)
    P.launch("launchFp4Product", C.byref(s["product"]), s["xq"], s["xs"], s["w"], s["w_scale"], None, s["out"], _stream())
    return s["out"]


def _fp4_experts_own(s):
    P, c = _pkg(), s["case"]
    T, N, K, E, k = c["tokens"], c["n"], c["k"], c["experts"], c["topk"]
    cap = s["order"].numel()
    _quantize_own(P, s, cap, s["order"], k)
    if "product" not in s:
        s["product"] = P.Fp4ProductOption(m=cap, n=N, k=K, numExperts=E, grouping=P.PRODUCT_ROWS, activation=0,
                                          outType=s["code"], outStride=N)
    P.launch("launchFp4Product", C.byref(s["product"]), s["xq"], s["xs"], s["w"], s["w_scale"], s["offsets"], s["rows"],
             _stream())
    P.launch("launchExpertCombine", N, s["code"], s["rows"], cap, N, s["position"], s["weights"], s["out"], N, T, k, _stream())
    return s["out"]


def _layer_own(s):
    P, c = _pkg(), s["case"]
    D = c["dim"]
    if "option" not in s:
        score = P.ROUTE_SOFTMAX if c["score"] == "softmax" else P.ROUTE_SIGMOID
        route = P.RouteOption(numExperts=c["experts"], topK=c["topk"], scoreType=score, numGroups=c["groups"],
                              topGroups=c["kept"], groupScore=2, renormalize=int(c["renorm"]), scale=SCALE,
                              logitsType=P.DATA_F32)
        s["option"] = P.ExpertLayerOption(
            route=route, dim=D, hidden=c["hidden"], gated=int(c["gated"]),
            activation=dict(relu=P.EXPERT_RELU, silu=P.EXPERT_SILU, gelu=P.EXPERT_GELU)[c["act"]],
            weightFormat=P.EXPERT_FP8 if c["weights"] == "fp8" else P.EXPERT_FP4, scaleRows=128 if c["weights"] == "fp8" else 1,
            dataType=s["code"], routerType=TYPES[c["router"]][1], strideX=D, strideOut=D)
    P.launch("launchExpertLayer", C.byref(s["option"]), s["x"], s["router"], s["bias"], s["w1"], s["w1_scale"], s["w2"],
             s["w2_scale"], s["out"], c["tokens"], _stream())
    return s["out"]


def _tensors(P, s):
    if "tensors" not in s:
        out = s.get("views", [None] * len(s["grads"]))
        s["tensors"] = (P.GradTensor * len(out))(*(
            P.GradTensor(data=t.data_ptr(), out=o.data_ptr() if o is not None else None, n=t.numel(), dataType=s["code"])
            for t, o in zip(s["grads"], out)))
    return s["tensors"], len(s["tensors"])


def _clip_own(s):
    P = _pkg()
    P.launch("launchGradNormClip", *_tensors(P, s), P.GRAD_NORM_2, s["scale"], s["max_norm"], P.GRAD_NONFINITE_KEEP, s["norm"],
             _stream())
    return dict(norm=s["norm"], clipped=s["clipped"])


def _grad_norm_own(s):
    P = _pkg()
    P.launch("launchGradNorm", *_tensors(P, s), P.GRAD_NORM_2, s["scale"], s["norm"], _stream())
    return s["norm"]


OWN = {"fp4": _fp4_own, "fp4_experts": _fp4_experts_own, "layer": _layer_own, "clip": _clip_own, "grad_norm": _grad_norm_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    b = 4 if case["dtype"] == "f32" else 2
    if kind == "fp4":
        M, N, K = case["rows"], case["n"], case["k"]
        return {"bytes": M * K * b + N * K * 17 / 32 + M * N * b, "flops": 2.0 * M * N * K}
    if kind == "fp4_experts":
        T, E, N, K, k = case["tokens"], case["experts"], case["n"], case["k"], case["topk"]
        return {"bytes": T * K * b + min(E, T * k) * N * K * 17 / 32 + T * N * b + 12 * T * k, "flops": 2.0 * T * k * N * K}
    if kind == "layer":
        T, E, k, D, H = case["tokens"], case["experts"], case["topk"], case["dim"], case["hidden"]
        used = E * (1 - (1 - k / E) ** T)  # experts that some token takes, if all are alike
        m = 3 if case["gated"] else 2
        each = m * D * H * (1 + 1 / 16384 if case["weights"] == "fp8" else 17 / 32)
        router = E * D * (4 if case["router"] == "f32" else 2) + (4 * E if case["bias"] else 0)
        return {"bytes": used * each + router + 2 * T * D * b, "flops": 2.0 * T * k * m * D * H + 2.0 * T * E * D}
    n = case["total"] + (10000 if case["sizes"] != "many" else 0)
    if kind == "grad_norm":
        return {"bytes": n * b, "flops": 2.0 * n}
    return {"bytes": 2 * n * b, "flops": 3.0 * n}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"fp4": _exact_fp4, "fp4_experts": _exact_fp4_experts, "layer": _exact_layer, "clip": _exact_clip,
            "grad_norm": lambda t: _exact_norm(t).view(1)}[case["kind"]](s)


GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_blocks(x, rule):
    """x [R, C] in 64 bits to the values that its 4-bit form stands for, by counting the midpoints below a magnitude."""
    R, Cc = x.shape
    p = torch.zeros(R, _up(Cc, 128), dtype=torch.float64, device=DEV)
    p[:, :Cc] = x
    p = p.view(R, -1, 32)
    top = p.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(torch.clamp(top, min=1e-300)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e) - 2
    if rule == "cover":
        e = torch.where(top > 6 * torch.exp2(e), e + 1, e)
    e = e.clamp(-126, 126)
    v = (p * torch.exp2(-e))
    n = torch.zeros_like(v, dtype=torch.int64)
    for i in range(7):
        half = (GRID[i] + GRID[i + 1]) / 2
        n += (v.abs() > half) if i % 2 == 0 else (v.abs() >= half)  # a tie goes to the even place
    q = torch.tensor(GRID, dtype=torch.float64, device=DEV)[n] * torch.sign(v)
    return (q * torch.exp2(e)).view(R, -1)[:, :Cc]


def _exact_stored4(bytes_, scale, cols):
    low, high = (bytes_ & 15).long(), (bytes_ >> 4).long()
    code = torch.zeros(*bytes_.shape[:-1], bytes_.shape[-1] * 2, dtype=torch.int64, device=DEV)
    code[..., 0::2], code[..., 1::2] = low, high
    v = torch.tensor(GRID, dtype=torch.float64, device=DEV)[code & 7] * (1 - 2 * (code >> 3)).double()
    return (v * torch.exp2(scale.double() - 127).repeat_interleave(32, -1))[..., :cols]


def _exact_stored8(bytes_, scale, cols):
    q = bytes_[..., :cols].contiguous().view(torch.float8_e4m3fn).double()
    e = (scale.double() - 127)[torch.arange(q.shape[0], device=DEV) // 128]
    return q * torch.exp2(e[:, torch.arange(cols, device=DEV) // 128])


def _exact_fp4(s):
    c = s["case"]
    return _exact_blocks(s["x"].double(), c["rule"]) @ _exact_stored4(s["w"][0], s["w_scale"][0], c["k"]).t().contiguous()


def _exact_fp4_experts(s):
    c = s["case"]
    x = _exact_blocks(s["x"].double(), c["rule"])
    out = torch.zeros(c["tokens"], c["n"], dtype=torch.float64, device=DEV)
    for e in range(c["experts"]):
        t, j = torch.nonzero(s["indices"] == e, as_tuple=True)
        w = _exact_stored4(s["w"][e], s["w_scale"][e], c["k"]).t().contiguous()
        out.index_add_(0, t, (x[t] @ w) * s["weights"][t, j].double()[:, None])
    return out


def _exact_layer(s):
    """Expert by expert, the tokens that take it."""
    c = s["case"]
    T, E, G, D, H = c["tokens"], c["experts"], c["groups"], c["dim"], c["hidden"]
    x = s["x"].double()
    z = x @ s["router"].double().t().contiguous()
    p = torch.softmax(z, 1) if c["score"] == "softmax" else torch.sigmoid(z)
    v = p + s["bias"].double() if s["bias"] is not None else p.clone()
    if G > 1:
        t = v.view(T, G, E // G).topk(min(2, E // G), dim=2).values.sum(2)
        allowed = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, t.topk(c["kept"], dim=1).indices, True)
        v = torch.where(allowed[:, torch.arange(E, device=DEV) // (E // G)], v, -math.inf)
    idx = v.topk(c["topk"], dim=1).indices
    w = p.gather(1, idx) * SCALE
    if c["renorm"]:
        w = w / (p.gather(1, idx).sum(1, keepdim=True) + 1e-20)
    act = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[c["act"]]
    stored = _exact_stored8 if c["weights"] == "fp8" else _exact_stored4
    out = torch.zeros(T, D, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t] @ stored(s["w1"][e], s["w1_scale"][e], D).t().contiguous()
        a = act(h[:, :H]) * h[:, H:] if c["gated"] else act(h)
        out.index_add_(0, t, (a @ stored(s["w2"][e], s["w2_scale"][e], H).t().contiguous()) * w[t, j][:, None])
    return out


def _exact_norm(s):
    parts = [float(torch.linalg.vector_norm(t.double())) / s["scale"] for t in s["grads"]]
    return torch.tensor(math.hypot(*parts), dtype=torch.float64, device=DEV)


def _exact_clip(s):
    norm = _exact_norm(s)
    factor = min(1.0, s["max_norm"] / float(norm))
    return dict(norm=norm.view(1), clipped=s["flat"].double() * factor)
