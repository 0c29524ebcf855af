"""The operators of a mixture-of-experts residual block, as cases that can be timed and compared.

Kinds:
  route      launchRouteExperts + launchRoutePlan: a router's logits to experts, weights and the experts' row plan
  route_bwd  launchRouteExpertsBackward: the weights' gradient back to the logits
  product    launchFp8Quantize + launchFp8Product: activations times a weight matrix, both in 8 bits with a
             power-of-two scale for each block of 128
  experts    gather + quantise, the experts' products, launchExpertCombine: rows of each expert times its own matrix
  experts_bwd  the same backward: gradients of the activations, the matrices and the routing weights
  norm       launchNormGateResidual: the norm behind a block, its gate, the residual, the next block's norm
  norm_bwd   launchNormGateResidualBackward: every gradient of it

Sizes: sample batches of the repository's configurations (2^18 samples, 2^16 rays, a 2^15 and a 2^14 batch), and
generic widths.  Everything is made from the seed with torch generators.
"""
from __future__ import annotations

import ctypes as C
import importlib
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def _pkg():
    return importlib.import_module("3dmaker_amd")


def listed():
    return [
        # One token's routing in serving: two launches' latency.
        dict(name="route_token", kind="route", tokens=1, experts=64, topk=6, score="softmax", groups=1, kept=1, bias=False,
             renorm=False, dtype="bf16", align=1),
        # A field split over eight experts: one training batch of 2^18 samples, two experts each, rows for the 8-bit products.
        dict(name="route_field", kind="route", tokens=1 << 18, experts=8, topk=2, score="softmax", groups=1, kept=1,
             bias=False, renorm=True, dtype="f32", align=128),
        # Many experts in groups, balanced by a bias: a ragged training batch.
        dict(name="route_groups", kind="route", tokens=16391, experts=256, topk=8, score="sigmoid", groups=8, kept=4,
             bias=True, renorm=True, dtype="bf16", align=128),
        # The router's gradient of a batch of 2^16 samples.
        dict(name="route_backward", kind="route_bwd", tokens=1 << 16, experts=64, topk=6, score="softmax", groups=1, kept=1,
             bias=True, renorm=True, dtype="f32", align=1),
        # One token through a dense 8-bit layer in serving: the weights' bytes.
        dict(name="product_token", kind="product", rows=1, n=4096, k=4096, dtype="bf16"),
        # A ragged batch through a wide layer: the matrix cores.
        dict(name="product_dense", kind="product", rows=8191, n=5120, k=4096, dtype="bf16"),
        # A few tokens over many experts in serving: most experts have no row.
        dict(name="experts_few", kind="experts", tokens=7, experts=16, topk=2, n=2048, k=1024, dtype="bf16"),
        # The experts' products of a training batch.
        dict(name="experts_field", kind="experts", tokens=1 << 15, experts=8, topk=2, n=2048, k=1024, dtype="bf16"),
        # Their backward: dX, dW and the routing weights' gradient.
        dict(name="experts_backward", kind="experts_bwd", tokens=1 << 14, experts=8, topk=2, n=2048, k=1024, dtype="f16"),
        # One token between two blocks in serving.
        dict(name="norm_token", kind="norm", rows=1, dim=4096, post="rms", pre="rms", gate_rows=1 << 20, dtype="bf16"),
        # A whole batch between two blocks, gated by channel: memory.
        dict(name="norm_batch", kind="norm", rows=32769, dim=2048, post="rms", pre="rms", gate_rows=1 << 20, dtype="bf16"),
        # Training a block that is modulated for each image of 1,024 rows: layer norms, every gradient.
        dict(name="norm_backward", kind="norm_bwd", rows=16389, dim=1280, post="layer", pre="layer", gate_rows=1024,
             dtype="f16"),
    ]


def _size(rng, lo, hi):
    """Log-uniform, odd as often as not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n | 1 if rng.random() < 0.5 else n & ~15 or n))
    return n if n != 3 << 10 else n + 1


def _width(rng, lo, hi, step):
    """Log-uniform multiple of `step`, any width one time in three."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n if rng.random() < 1 / 3 else max(1, n // step) * step))
    return n if n != 3 << 10 else n - step


def draw(rng):
    kind = rng.choice(["route", "route", "route_bwd", "product", "experts", "experts_bwd", "norm", "norm_bwd"])
    if kind in ("route", "route_bwd"):
        experts = rng.choice([4, 8, 16, 60, 64, 128, 160, 256])
        groups = rng.choice([1, 1, 4, 8] if experts % 8 == 0 else [1, 1, 4])
        kept = 1 if groups == 1 else rng.randint(max(1, groups // 2), groups)
        topk = rng.randint(1, max(1, min(8, experts // groups * kept)))
        score = rng.choice(["softmax", "sigmoid"])
        return dict(kind=kind, tokens=_size(rng, 1, min(1 << 18, (1 << 22) // experts)), experts=experts, topk=topk,
                    score=score, groups=groups, kept=kept, bias=rng.random() < 0.5, renorm=rng.random() < 0.7,
                    dtype=rng.choice(list(TYPES)), align=rng.choice([1, 16, 128]))
    if kind == "product":
        return dict(kind=kind, rows=_size(rng, 1, 8191), n=_width(rng, 64, 5120, 64), k=_width(rng, 64, 4096, 64),
                    dtype=rng.choice(list(TYPES)))
    if kind in ("experts", "experts_bwd"):
        experts = rng.choice([2, 4, 8, 16, 32])
        return dict(kind=kind, tokens=_size(rng, 1, (1 << 15) if kind == "experts" else 1 << 14), experts=experts,
                    topk=rng.randint(1, 2), n=_width(rng, 64, 2048, 64), k=_width(rng, 64, 1024, 64),
                    dtype=rng.choice(["f16", "bf16"]))
    dim = _width(rng, 64, 8192, 64)
    rows = _size(rng, 1, max(1, min(1 << 17, ((1 << 26) if kind == "norm" else (1 << 24)) // dim)))
    return dict(kind=kind, rows=rows, dim=dim, post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["none", "rms", "layer"]),
                gate_rows=rng.choice([0, 1, 64, 1000, 1 << 20]), dtype=rng.choice(list(TYPES)))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (seed + 1))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _types(case):
    return TYPES[case["dtype"]]


def _capacity(case):
    """Rows of the plan: every slot, and each expert's segment filled up to `align`."""
    slots, experts, align = case["tokens"] * case["topk"], case["experts"], case.get("align", 128)
    return -(-(slots + min(experts, slots) * (align - 1)) // align) * align


def _router_inputs(case, g):
    """Logits and bias whose selection does not hang on the last bits of a score: two experts (or groups) that are
    ranked against each other are tied exactly or at least 3e-6 of their size apart."""
    T, E, G = case["tokens"], case["experts"], case["groups"]
    dt = _types(case)[0]
    bias = _randn(g, E) * 0.05 if case["bias"] else None
    z = (_randn(g, T, E) * 1.5 + _randn(g, 1, E) * 0.5).to(dt)
    for _ in range(20):
        zz = z.double()
        s = torch.softmax(zz, 1) if case["score"] == "softmax" else torch.sigmoid(zz)
        c = s if bias is None else s + bias.double()
        bad = torch.zeros(T, dtype=torch.bool, device=DEV)

        def near(v, pairs):
            v = torch.sort(v, dim=1, descending=True).values[:, :pairs + 1]
            a, b = v[:, :-1], v[:, 1:]
            gap = a - b
            return ((gap > 0) & (gap < 3e-6 * torch.maximum(a.abs(), b.abs()))).any(1)

        if G > 1:
            best = torch.sort(c.view(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
            bad |= near(best, min(case["kept"], G - 1))
            keep = torch.zeros(T, G, dtype=torch.bool, device=DEV)
            keep.scatter_(1, torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["kept"]], True)
            c = c.masked_fill(~keep.repeat_interleave(E // G, 1), -1e9)
        bad |= near(c, min(case["topk"], E - 1))
        n = int(bad.sum())
        if n == 0:
            break
        z[bad] = (_randn(g, n, E) * 1.5).to(dt)
    return z, bias


def _plan_inputs(case, g):
    """Indices of distinct experts, some of them asked for more than others, the weights, and the plan that a program
    has from the router, with the longest segment as a host number."""
    T, E, k = case["tokens"], case["experts"], case["topk"]
    pop = _randn(g, 1, E) * 0.7
    gumbel = -torch.log(-torch.log(torch.rand(T, E, generator=g, device=DEV).clamp(1e-7, 1 - 1e-7)))
    indices = torch.sort(pop + gumbel, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
    weights = torch.softmax(_randn(g, T, k), 1).contiguous()
    offsets, order, position = _plan_plain(indices, E, 128, _capacity(case))
    longest = int((offsets[1:] - offsets[:-1]).max())
    return dict(indices=indices, weights=weights, offsets=offsets, order=order, position=position, longest=longest)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    dt, code = _types(case)
    s = dict(case=case, dt=dt, code=code)
    if kind in ("route", "route_bwd"):
        T, k = case["tokens"], case["topk"]
        s["logits"], s["bias"] = _router_inputs(case, g)
        s["indices"] = torch.empty(T, k, dtype=torch.int32, device=DEV)
        s["weights"] = torch.empty(T, k, dtype=torch.float32, device=DEV)
        if kind == "route":
            cap = _capacity(case)
            s.update(capacity=cap, offsets=torch.empty(case["experts"] + 1, dtype=torch.int32, device=DEV),
                     order=torch.empty(cap, dtype=torch.int32, device=DEV),
                     position=torch.empty(T, k, dtype=torch.int32, device=DEV))
        else:
            s["indices"] = _route_plain(case, s["logits"], s["bias"])[0]
            s["dweights"] = _randn(g, T, k)
            s["dlogits"] = torch.empty_like(s["logits"])
    elif kind == "product":
        M, N, K = case["rows"], case["n"], case["k"]
        s["x"] = _randn(g, M, K).to(dt)
        w = _randn(g, N, K) / math.sqrt(K)
        s["w"], s["w_scale"] = _store(*_quantize(w[None], 128), 1)
        s["xq"], s["xs"] = _q_buffers(M, K)
        s["out"] = torch.empty(M, N, dtype=dt, device=DEV)
    elif kind in ("experts", "experts_bwd"):
        T, E, N, K = case["tokens"], case["experts"], case["n"], case["k"]
        s.update(_plan_inputs(case, g))
        cap = s["order"].numel()
        s["x"] = _randn(g, T, K).to(dt)
        w = _randn(g, E, N, K) / math.sqrt(K)
        q, e = _quantize(w, 128)
        s["w"], s["w_scale"] = _store(q, e, E)
        s["rows"] = torch.empty(cap, N, dtype=dt, device=DEV)
        s["xq"], s["xs"] = _q_buffers(cap, K)
        s["out"] = torch.empty(T, N, dtype=dt, device=DEV)
        if kind == "experts_bwd":
            s["wt"], s["wt_scale"] = _store(q.transpose(1, 2).contiguous(), e.transpose(1, 2).contiguous(), E)
            s["rows"] = _randn(g, cap, N).to(dt)  # the forward's rows
            s["dout"] = (_randn(g, T, N) * 0.02).to(dt)
            s["gq"], s["gs"] = _q_buffers(cap, N)
            s["gtq"], s["gts"] = _q_buffers(N, cap)
            s["xtq"], s["xts"] = _q_buffers(K, cap)
            s["drows"] = torch.empty(cap, K, dtype=dt, device=DEV)
            s["dx"] = torch.empty(T, K, dtype=dt, device=DEV)
            s["dw"] = torch.empty(E, N, K, dtype=torch.float32, device=DEV)
            s["dweights"] = torch.empty(T, case["topk"], dtype=torch.float32, device=DEV)
    else:
        R, D, gr = case["rows"], case["dim"], case["gate_rows"]
        s["x"] = (_randn(g, R, D) * 2).to(dt)
        s["f"] = (_randn(g, R, D) * 0.7 + 0.1).to(dt)
        s["gate"] = (1 + 0.3 * _randn(g, -(-R // gr), D)).to(dt) if gr else None
        for side in ("post", "pre"):
            s[side + "_w"] = 1 + 0.1 * _randn(g, D) if case[side] != "none" else None
            s[side + "_b"] = 0.1 * _randn(g, D) if case[side] == "layer" else None
        s["y"], s["h"] = torch.empty(R, D, dtype=dt, device=DEV), torch.empty(R, D, dtype=dt, device=DEV)
        if kind == "norm_bwd":
            s["dy"], s["dh"] = (_randn(g, R, D) * 0.1).to(dt), (_randn(g, R, D) * 0.1).to(dt)
            s["dx"], s["df"] = torch.empty_like(s["x"]), torch.empty_like(s["f"])
            s["dgate"] = torch.empty_like(s["gate"]) if gr else None
            for p in ("post_w", "post_b", "pre_w", "pre_b"):
                s["d" + p] = torch.empty(D, dtype=torch.float32, device=DEV) if s[p] is not None else None
    return s


# ---------------------------------------------------------------------------
# the stored form of 8-bit matrices: rows of bytes filled up to whole blocks of 128, scales in rows of whole fours
# ---------------------------------------------------------------------------

def _up(n, m):
    return -(-n // m) * m


def _q_buffers(rows, cols):
    blocks = _up(cols, 128) // 128
    return (torch.empty(rows, blocks * 128, dtype=torch.uint8, device=DEV),
            torch.empty(rows, _up(blocks, 4), dtype=torch.uint8, device=DEV))


def _quantize(x, block_rows):
    """x [B, R, C] in 32 bits to e4m3 values (as bytes' values, float8) and exponents of the scales [B, R', C']:
    a scale for `block_rows` rows by 128 columns, the smallest power of two that brings the block within 448."""
    B, R, Cc = x.shape
    rb, cb = -(-R // block_rows), -(-Cc // 128)
    p = torch.nn.functional.pad(x, (0, cb * 128 - Cc, 0, rb * block_rows - R)).view(B, rb, block_rows, cb, 128)
    m, e = torch.frexp(p.abs().amax((2, 4)))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-126, 126).to(torch.int32)
    inverse = ((127 - e) << 23).view(torch.float32)
    q = (p * inverse[:, :, None, :, None]).reshape(B, rb * block_rows, cb * 128)[:, :R, :Cc]
    return q.to(torch.float8_e4m3fn), e


def _dequantize(q, e, block_rows):
    """The values that q and the scales' exponents stand for, in 32 bits."""
    scale = ((127 + e) << 23).view(torch.float32)
    rows = scale.repeat_interleave(block_rows, 1)[:, :q.shape[1]]
    return q.float() * rows.repeat_interleave(128, 2)[:, :, :q.shape[2]]


def _store(q, e, batch):
    """As the entry points take it: bytes [batch * rows, whole blocks], scale bytes [batch * block rows, whole fours]."""
    B, R, Cc = q.shape
    bytes_ = torch.zeros(B, R, _up(Cc, 128), dtype=torch.uint8, device=DEV)
    bytes_[:, :, :Cc] = q.view(torch.uint8)
    scale = torch.full((B, e.shape[1], _up(e.shape[2], 4)), 127, dtype=torch.uint8, device=DEV)
    scale[:, :, :e.shape[2]] = (e + 127).to(torch.uint8)
    return bytes_.contiguous(), scale.contiguous()


def _stored_values(bytes_, scale, cols, block_rows):
    """The 32-bit values of a stored matrix [B, R, cols]."""
    q = bytes_.view(torch.float8_e4m3fn).float()[:, :, :cols]
    s = (scale.to(torch.int32) << 23).view(torch.float32)
    s = s.repeat_interleave(block_rows, 1)[:, :q.shape[1]].repeat_interleave(128, 2)[:, :, :cols]
    return q * s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _scores(case, logits):
    z = logits.float()
    if case["score"] == "softmax":
        e = torch.exp(z - z.amax(1, keepdim=True))
        return e / e.sum(1, keepdim=True)
    return 1 / (1 + torch.exp(-z))


def _route_plain(case, logits, bias):
    T, E, G = case["tokens"], case["experts"], case["groups"]
    s = _scores(case, logits)
    c = s if bias is None else s + bias
    if G > 1:
        best = torch.sort(c.view(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=c.device).scatter_(1, kept, True)
        c = c.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    idx = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :case["topk"]]
    w = s.gather(1, idx)
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return idx.to(torch.int32), w * _scale(case)


def _scale(case):
    return 2.5 if case["groups"] > 1 else 1.0


def _plan_plain(indices, experts, align, capacity):
    """Stable counting sort of the slots by expert, each expert's rows from a multiple of `align` on."""
    flat = indices.reshape(-1).long()
    slots = flat.numel()
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.cumsum((counts + align - 1) // align * align, 0)
    by = torch.sort(flat, stable=True).indices
    first = torch.cumsum(counts, 0) - counts
    e = flat[by]
    at = offsets[e] + torch.arange(slots, device=flat.device) - first[e]
    order = torch.full((capacity,), -1, dtype=torch.int32, device=flat.device)
    order[at] = by.to(torch.int32)
    position = torch.empty(slots, dtype=torch.int32, device=flat.device)
    position[by] = at.to(torch.int32)
    return offsets.to(torch.int32), order, position.view(indices.shape)


def _route_bwd_plain(s):
    case = s["case"]
    p = _scores(case, s["logits"])
    idx = s["indices"].long()
    sel, g = p.gather(1, idx), s["dweights"] * _scale(case)
    if case["renorm"]:
        total = sel.sum(1, keepdim=True) + 1e-20
        g = (g - (g * sel).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(p).scatter_(1, idx, g)
    if case["score"] == "softmax":
        return (p * (ds - (ds * p).sum(1, keepdim=True))).to(s["dt"])
    return (ds * p * (1 - p)).to(s["dt"])


def _product_plain(s):
    case = s["case"]
    x = _dequantize(*_quantize(s["x"].float()[None], 1), 1)[0]
    w = _stored_values(s["w"], s["w_scale"], case["k"], 128)[0]
    return (x @ w.t().contiguous()).to(s["dt"])


def _by_expert(s):
    """Row of the plan for each expert's places [E, longest], and which of them exist."""
    o = s["offsets"].long()
    at = o[:-1, None] + torch.arange(s["longest"], device=DEV)
    fine = at < o[1:, None]
    return torch.where(fine, at, 0), fine


def _experts_plain(s):
    case, k = s["case"], s["case"]["topk"]
    slot = s["order"].long().clamp(min=0)
    x = s["x"].float()[slot // k] * (s["order"] >= 0)[:, None]
    x = _dequantize(*_quantize(x[None], 1), 1)[0]
    w = _stored_values(s["w"], s["w_scale"], case["k"], 128)
    at, fine = _by_expert(s)
    y = torch.bmm(x[at] * fine[:, :, None], w.transpose(1, 2).contiguous())
    rows = torch.zeros(x.shape[0] + 1, case["n"], device=DEV)
    rows[torch.where(fine, at, x.shape[0])] = y
    return (rows[s["position"].long()] * s["weights"][:, :, None]).sum(1).to(s["dt"])


def _experts_bwd_plain(s):
    case, k = s["case"], s["case"]["topk"]
    K, N = case["k"], case["n"]
    there = (s["order"] >= 0)[:, None]
    slot = s["order"].long().clamp(min=0)
    token = slot // k
    g = s["dout"].float()[token] * s["weights"].reshape(-1)[slot][:, None] * there
    x = s["x"].float()[token] * there
    at, fine = _by_expert(s)
    fine = fine[:, :, None]
    w = _stored_values(s["wt"], s["wt_scale"], N, 128)  # [E, K, N]
    gr = _dequantize(*_quantize(g[None], 1), 1)[0]
    dr = torch.bmm(gr[at] * fine, w.transpose(1, 2).contiguous())
    drows = torch.zeros(g.shape[0] + 1, K, device=DEV)
    drows[torch.where(fine[:, :, 0], at, g.shape[0])] = dr
    dx = drows[s["position"].long()].sum(1).to(s["dt"])
    gt = _dequantize(*_quantize(g.t().contiguous()[None], 1), 1)[0].t()
    xt = _dequantize(*_quantize(x.t().contiguous()[None], 1), 1)[0].t()
    dw = torch.bmm((gt[at] * fine).transpose(1, 2).contiguous(), (xt[at] * fine).contiguous())
    dweights = (s["dout"].float()[:, None, :] * s["rows"].float()[s["position"].long()]).sum(2)
    return dict(dx=dx, dw=dw, dweights=dweights)


def _norm_of(x, kind, w, b):
    """(normalised, its scale of the row, output)"""
    if kind == "none":
        return x, None, x
    c = x - x.mean(1, keepdim=True) if kind == "layer" else x
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    n = c * r
    return n, r, n * w + (b if b is not None else 0)


def _norm_back(d, n, r, kind, w):
    """(dL/dinput, dL/dw, dL/db) of a norm's output gradient d."""
    if kind == "none":
        return d, None, None
    dn = d * w
    m = dn.mean(1, keepdim=True) if kind == "layer" else 0
    return r * (dn - m - n * (dn * n).mean(1, keepdim=True)), (d * n).sum(0), d.sum(0) if kind == "layer" else None


ALPHA, BETA = 0.9, 0.5


def _gate_rows(s, rows):
    gr = s["case"]["gate_rows"]
    return torch.arange(rows, device=s["x"].device) // gr


def _norm_plain(s):
    case = s["case"]
    x, f = s["x"].float(), s["f"].float()
    u = _norm_of(f, case["post"], s["post_w"], s["post_b"])[2]
    if s["gate"] is not None:
        u = u * s["gate"].float()[_gate_rows(s, x.shape[0])]
    y = ALPHA * x + BETA * u
    h = _norm_of(y, case["pre"], s["pre_w"], s["pre_b"])[2]
    return dict(y=y.to(s["dt"]), h=h.to(s["dt"]))


def _norm_bwd_plain(s):
    case = s["case"]
    x, f, dy, dh = s["x"].float(), s["f"].float(), s["dy"].float(), s["dh"].float()
    n1, r1, u = _norm_of(f, case["post"], s["post_w"], s["post_b"])
    row = _gate_rows(s, x.shape[0]) if s["gate"] is not None else None
    gate = s["gate"].float()[row] if row is not None else 1.0
    n2, r2, _ = _norm_of(ALPHA * x + BETA * gate * u, case["pre"], s["pre_w"], s["pre_b"])
    d, dw2, db2 = _norm_back(dh, n2, r2, case["pre"], s["pre_w"])
    d = d + dy
    du = BETA * gate * d
    df, dw1, db1 = _norm_back(du, n1, r1, case["post"], s["post_w"])
    out = dict(dx=(ALPHA * d).to(s["dt"]), df=df.to(s["dt"]), dpost_w=dw1, dpost_b=db1, dpre_w=dw2, dpre_b=db2)
    if row is not None:
        gr, whole = min(case["gate_rows"], x.shape[0]), s["gate"].shape[0]
        d = torch.nn.functional.pad(BETA * d * u, (0, 0, 0, whole * gr - x.shape[0]))
        out["dgate"] = d.view(whole, gr, x.shape[1]).sum(1).to(s["dt"])
    return out


PLAIN = {"route": lambda s: _named_route(*_route_plain(s["case"], s["logits"], s["bias"]), s), "route_bwd": _route_bwd_plain,
         "product": _product_plain, "experts": _experts_plain, "experts_bwd": _experts_bwd_plain,
         "norm": _norm_plain, "norm_bwd": _norm_bwd_plain}


def _named_route(idx, w, s):
    offsets, order, position = _plan_plain(idx, s["case"]["experts"], s["case"]["align"], s["capacity"])
    return dict(indices=idx, weights=w, offsets=offsets, order=order, position=position)


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

def _stream():
    return torch.cuda.current_stream().cuda_stream


def _route_option(P, s):
    c = s["case"]
    return P.RouteOption(numExperts=c["experts"], topK=c["topk"], scoreType=0 if c["score"] == "softmax" else 1,
                         numGroups=c["groups"], topGroups=c["kept"], groupScore=2, renormalize=int(c["renorm"]),
                         scale=_scale(c), logitsType=s["code"])


def _route_own(s):
    P, c = _pkg(), s["case"]
    T, k, E = c["tokens"], c["topk"], c["experts"]
    o = _route_option(P, s)
    P.launch("launchRouteExperts", C.byref(o), s["logits"], E, s["bias"], s["indices"], s["weights"], T, _stream())
    P.launch("launchRoutePlan", s["indices"], T, k, E, c["align"], s["capacity"], s["offsets"], s["order"], s["position"],
             _stream())
    return {n: s[n] for n in ("indices", "weights", "offsets", "order", "position")}


def _route_bwd_own(s):
    P, c = _pkg(), s["case"]
    o = _route_option(P, s)
    P.launch("launchRouteExpertsBackward", C.byref(o), s["logits"], c["experts"], s["indices"], s["dweights"],
             s["dlogits"], c["experts"], c["tokens"], _stream())
    return s["dlogits"]


def _quant_own(P, s, x, rows, cols, slots, weights, order, q=None, scale=None, qt=None, scale_t=None):
    o = P.Fp8QuantOption(rows=rows, cols=cols, batch=1, blockRows=1, srcType=s["code"], slotsPerRow=slots,
                         srcRows=x.shape[0], srcStride=cols, srcBatchStride=0, gateStride=0)
    P.launch("launchFp8Quantize", C.byref(o), x, order, weights, None, q, scale, qt, scale_t, _stream())


def _product_own(s):
    P, c = _pkg(), s["case"]
    M, N, K = c["rows"], c["n"], c["k"]
    _quant_own(P, s, s["x"], M, K, 1, None, None, s["xq"], s["xs"])
    o = P.Fp8ProductOption(m=M, n=N, k=K, numExperts=1, grouping=0, scaleRowsB=128, activation=0, outType=s["code"],
                           outStride=N)
    P.launch("launchFp8Product", C.byref(o), s["xq"], s["xs"], s["w"], s["w_scale"], None, s["out"], _stream())
    return s["out"]


def _experts_own(s):
    P, c = _pkg(), s["case"]
    T, N, K, E, k = c["tokens"], c["n"], c["k"], c["experts"], c["topk"]
    cap = s["order"].numel()
    _quant_own(P, s, s["x"], cap, K, k, None, s["order"], s["xq"], s["xs"])
    o = P.Fp8ProductOption(m=cap, n=N, k=K, numExperts=E, grouping=1, scaleRowsB=128, activation=0, outType=s["code"],
                           outStride=N)
    P.launch("launchFp8Product", C.byref(o), s["xq"], s["xs"], s["w"], s["w_scale"], s["offsets"], s["rows"], _stream())
    P.launch("launchExpertCombine", N, s["code"], s["rows"], cap, N, s["position"], s["weights"], s["out"], N, T, k, _stream())
    return s["out"]


def _experts_bwd_own(s):
    P, c = _pkg(), s["case"]
    T, N, K, E, k = c["tokens"], c["n"], c["k"], c["experts"], c["topk"]
    cap = s["order"].numel()
    _quant_own(P, s, s["dout"], cap, N, k, s["weights"], s["order"], s["gq"], s["gs"], s["gtq"], s["gts"])
    _quant_own(P, s, s["x"], cap, K, k, None, s["order"], None, None, s["xtq"], s["xts"])
    o = P.Fp8ProductOption(m=cap, n=K, k=N, numExperts=E, grouping=1, scaleRowsB=128, activation=0, outType=s["code"],
                           outStride=K)
    P.launch("launchFp8Product", C.byref(o), s["gq"], s["gs"], s["wt"], s["wt_scale"], s["offsets"], s["drows"], _stream())
    P.launch("launchExpertCombine", K, s["code"], s["drows"], cap, K, s["position"], None, s["dx"], K, T, k, _stream())
    o = P.Fp8ProductOption(m=N, n=K, k=cap, numExperts=E, grouping=2, scaleRowsB=1, activation=0, outType=0, outStride=K)
    P.launch("launchFp8Product", C.byref(o), s["gtq"], s["gts"], s["xtq"], s["xts"], s["offsets"], s["dw"], _stream())
    P.launch("launchExpertCombineBackward", N, s["code"], s["rows"], cap, N, s["position"], s["dout"], N, s["dweights"], T, k,
             _stream())
    return dict(dx=s["dx"], dw=s["dw"], dweights=s["dweights"])


NORMS = {"none": 0, "rms": 1, "layer": 2}


def _norm_option(P, s):
    c = s["case"]
    D = c["dim"]
    return P.NormGateOption(dim=D, postNorm=NORMS[c["post"]], preNorm=NORMS[c["pre"]], gateRows=c["gate_rows"],
                            residualScale=ALPHA, blockScale=BETA, epsilon=EPS, dataType=s["code"], strideX=D, strideF=D,
                            strideGate=D, strideY=D, strideH=D)


def _norm_own(s):
    P, c = _pkg(), s["case"]
    o = _norm_option(P, s)
    P.launch("launchNormGateResidual", C.byref(o), s["x"], s["f"], s["gate"], s["post_w"], s["post_b"], s["pre_w"],
             s["pre_b"], s["y"], s["h"], c["rows"], _stream())
    return dict(y=s["y"], h=s["h"])


def _norm_bwd_own(s):
    P, c = _pkg(), s["case"]
    o = _norm_option(P, s)
    P.launch("launchNormGateResidualBackward", C.byref(o), s["x"], s["f"], s["gate"], s["post_w"], s["post_b"], s["pre_w"],
             s["pre_b"], s["dy"], s["dh"], s["dx"], s["df"], s["dgate"], s["dpost_w"], s["dpost_b"], s["dpre_w"],
             s["dpre_b"], c["rows"], _stream())
    out = {n: s[n] for n in ("dx", "df", "dpost_w", "dpost_b", "dpre_w", "dpre_b")}
    if s["gate"] is not None:
        out["dgate"] = s["dgate"]
    return out


OWN = {"route": _route_own, "route_bwd": _route_bwd_own, "product": _product_own, "experts": _experts_own,
       "experts_bwd": _experts_bwd_own, "norm": _norm_own, "norm_bwd": _norm_bwd_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    b = 4 if case["dtype"] == "f32" else 2
    if kind in ("route", "route_bwd"):
        T, E, k = case["tokens"], case["experts"], case["topk"]
        bias = 4 * E if case["bias"] else 0
        if kind == "route":  # logits; indices and weights, position; offsets, order
            return {"bytes": T * E * b + bias + 12 * T * k + 4 * (E + 1) + 4 * _capacity(case), "flops": 4.0 * T * E}
        return {"bytes": 2 * T * E * b + 8 * T * k, "flops": 8.0 * T * E}
    if kind == "product":
        M, N, K = case["rows"], case["n"], case["k"]
        return {"bytes": M * K * b + N * K + N * K / 16384 + M * N * b, "flops": 2.0 * M * N * K}
    if kind in ("experts", "experts_bwd"):
        T, E, N, K, k = case["tokens"], case["experts"], case["n"], case["k"], case["topk"]
        used = min(E, T * k)
        if kind == "experts":
            return {"bytes": T * K * b + used * N * K + T * N * b + 12 * T * k, "flops": 2.0 * T * k * N * K}
        return {"bytes": 2 * T * K * b + T * N * b + T * k * N * b + used * N * K + E * N * K * 4 + 16 * T * k,
                "flops": 4.0 * T * k * N * K + 2.0 * T * k * N}
    R, D, gr = case["rows"], case["dim"], case["gate_rows"]
    gates = (-(-R // gr)) * D * b if gr else 0
    parameters = 4 * D * sum({"none": 0, "rms": 1, "layer": 2}[case[side]] for side in ("post", "pre"))
    if kind == "norm":
        return {"bytes": 4 * R * D * b + gates + parameters, "flops": 14.0 * R * D}
    return {"bytes": 6 * R * D * b + 2 * gates + 2 * parameters, "flops": 40.0 * R * D}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "route_bwd": _exact_route_bwd, "product": _exact_product, "experts": _exact_experts,
            "experts_bwd": _exact_experts_bwd, "norm": _exact_norm, "norm_bwd": _exact_norm_bwd}[case["kind"]](s)


def _exact_scores(s):
    z = s["logits"].double()
    return torch.softmax(z, 1) if s["case"]["score"] == "softmax" else torch.sigmoid(z)


def _exact_route(s):
    """Indices by repeated maximum (argmax of a row reversed twice gives the lowest of equal ones); the plan from a
    sort of (expert, slot) on the host."""
    c = s["case"]
    T, E, G, k = c["tokens"], c["experts"], c["groups"], c["topk"]
    p = _exact_scores(s)
    v = p + s["bias"].double() if s["bias"] is not None else p.clone()

    def lowest_argmax(a):
        top = a.amax(1, keepdim=True)
        return torch.where(a == top, torch.arange(a.shape[1], device=a.device), a.shape[1]).amin(1, keepdim=True)

    if G > 1:
        t = v.view(T, G, E // G).topk(min(2, E // G), dim=2).values.sum(2)
        allowed = torch.zeros(T, G, dtype=torch.bool, device=DEV)
        for _ in range(c["kept"]):
            i = lowest_argmax(t.masked_fill(allowed, -math.inf))
            allowed.scatter_(1, i, True)
        v = torch.where(allowed[:, torch.arange(E, device=DEV) // (E // G)], v, -math.inf)
    picked = []
    for _ in range(k):
        i = lowest_argmax(v)
        picked.append(i)
        v = v.scatter(1, i, -math.inf)
    idx = torch.cat(picked, 1)
    w = torch.gather(p, 1, idx)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return dict(indices=None, weights=w * _scale(c), offsets=None, order=None, position=None)


def _exact_route_bwd(s):
    """By differentiating the definition."""
    c = s["case"]
    with torch.enable_grad():
        z = s["logits"].double().requires_grad_(True)
        p = torch.softmax(z, 1) if c["score"] == "softmax" else torch.sigmoid(z)
        w = p.gather(1, s["indices"].long())
        if c["renorm"]:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
        (w * _scale(c) * s["dweights"].double()).sum().backward()
    return z.grad


def _exact_blocks(x):
    """x [R, C] in 64 bits to the values that its 8-bit form stands for, a scale for each row's 128 columns."""
    R, Cc = x.shape
    p = torch.zeros(R, _up(Cc, 128), dtype=torch.float64, device=DEV)
    p[:, :Cc] = x
    p = p.view(R, -1, 128)
    top = p.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(-126, 126)
    v = p * torch.exp2(-e)
    # e4m3: 3 bits behind the leading one, down to steps of 2^-9; halves to even
    lead = torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -6)))
    lead = torch.where(v.abs() < torch.exp2(lead), lead - 1, lead)
    step = torch.exp2(torch.clamp(lead, min=-6) - 3)
    return (torch.round(v / step) * step * torch.exp2(e)).view(R, -1)[:, :Cc]


def _exact_stored(bytes_, scale, cols, block_rows):
    q = bytes_[:, :, :cols].contiguous().view(torch.float8_e4m3fn).double()
    e = scale.double() - 127
    e = e[:, torch.arange(q.shape[1], device=DEV) // block_rows][:, :, torch.arange(cols, device=DEV) // 128]
    return q * torch.exp2(e)


def _exact_product(s):
    c = s["case"]
    return _exact_blocks(s["x"].double()) @ _exact_stored(s["w"], s["w_scale"], c["k"], 128)[0].t().contiguous()


def _exact_experts(s):
    c, k = s["case"], s["case"]["topk"]
    x = _exact_blocks(s["x"].double())
    w = _exact_stored(s["w"], s["w_scale"], c["k"], 128)
    out = torch.zeros(c["tokens"], c["n"], dtype=torch.float64, device=DEV)
    for e in range(c["experts"]):
        t, j = torch.nonzero(s["indices"] == e, as_tuple=True)
        out.index_add_(0, t, (x[t] @ w[e].t().contiguous()) * s["weights"][t, j].double()[:, None])
    return out


def _exact_experts_bwd(s):
    c = s["case"]
    T, N, K, E = c["tokens"], c["n"], c["k"], c["experts"]
    w = _exact_stored(s["wt"], s["wt_scale"], N, 128)
    dx = torch.zeros(T, K, dtype=torch.float64, device=DEV)
    dw = torch.zeros(E, N, K, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = torch.nonzero(s["indices"] == e, as_tuple=True)
        # the product of the two factors is a 32-bit number: it is what is quantised
        g = (s["dout"][t].float() * s["weights"][t, j][:, None]).double()
        dx.index_add_(0, t, _exact_blocks(g) @ w[e].t().contiguous())
        if t.numel():
            gt, xt = _exact_blocks(g.t().contiguous()), _exact_blocks(s["x"][t].double().t().contiguous())
            dw[e] = gt @ xt.t().contiguous()
    at = s["position"].long()
    dweights = torch.stack([(s["dout"].double() * s["rows"][at[:, j]].double()).sum(1) for j in range(at.shape[1])], 1)
    return dict(dx=dx, dw=dw, dweights=dweights)


def _exact_forward(c, x, f, gate, pw, pb, nw, nb):
    def norm(v, kind, w, b):
        if kind == "none":
            return v
        if kind == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * w
        return v if b is None else v + b

    u = norm(f, c["post"], pw, pb)
    if gate is not None:
        u = u * gate[torch.arange(x.shape[0], device=DEV) // c["gate_rows"]]
    y = ALPHA * x + BETA * u
    return y, norm(y, c["pre"], nw, nb)


NORM_INPUTS = ("x", "f", "gate", "post_w", "post_b", "pre_w", "pre_b")


def _exact_norm(s):
    a = [s[n].double() if s[n] is not None else None for n in NORM_INPUTS]
    y, h = _exact_forward(s["case"], *a)
    return dict(y=y, h=h)


def _exact_norm_bwd(s):
    """By differentiating the definition."""
    with torch.enable_grad():
        a = {n: s[n].double().requires_grad_(True) if s[n] is not None else None for n in NORM_INPUTS}
        y, h = _exact_forward(s["case"], *(a[n] for n in NORM_INPUTS))
        ((y * s["dy"].double()).sum() + (h * s["dh"].double()).sum()).backward()
    out = {"d" + n: v.grad for n, v in a.items() if v is not None}
    return {n: out.get(n) for n in ("dx", "df", "dpost_w", "dpost_b", "dpre_w", "dpre_b", "dgate")}
