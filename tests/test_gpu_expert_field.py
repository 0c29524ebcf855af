"""The mixture-of-experts block as a whole (examples/expert_field.py): its forward and every gradient against the same
chain in 64 bits with the same roundings to 8 bits and fp16, and a short training.

Where both sides round the same number they agree but for those whose fp16 rounding turns on the last bits of a sum (at
most 1 in 30 by the 8-bit sums' 1.5e-5), and 1 in 64 of these move an e4m3 value by its step (9 % of it): 0.2 % of a
2-norm for one such rounding, at most four in a row, and 2^-11 for each fp16 output: 1 %."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_field.py")
    spec = importlib.util.spec_from_file_location("expert_field", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def q8(x):
    """The values that [R, C] stands for in 8 bits, a scale for each row's 128 columns."""
    q, b = R.quantize(x)
    e = torch.exp2(b.double() - 127)
    return q * e.repeat_interleave(128, 1)[:, :x.shape[1]]


def q8_blocks(w):
    q, b = R.quantize(w, 128)
    e = torch.exp2(b.double() - 127)
    return q * e.repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]


@pytest.mark.parametrize("T,D,H,E,k", [(1, 64, 128, 4, 2), (300, 192, 320, 5, 2), (1000, 256, 512, 8, 1)])
def test_block_against_64_bits(T, D, H, E, k):
    M = example()
    block = M.ExpertBlock(D, H, E, k, seed=3)
    g = R.gen(4)
    x, dy = R.randn(g, T, D).half(), R.randn(g, T, D).half()
    y = block.forward(x)
    dx, grad = block.backward(dy)
    torch.cuda.synchronize()

    def near(got, want, what):
        want = want.double()
        off = float((got.double() - want).norm() / want.norm().clamp(min=1e-9))
        assert off <= 0.01, (what, off)

    p = {n: v.double() for n, v in block.p.items()}
    x64 = x.double().requires_grad_(True)
    w_in = p["norm_in"].clone().requires_grad_(True)
    h = R.norm(x64, 1, w_in, None, 1e-6)
    h16 = h.detach().half()
    near(block.h, h16, "h")
    w = block.weight.double()
    w1, w2 = [q8_blocks(v) for v in p["w1"]], [q8_blocks(v) for v in p["w2"]]
    picks = [torch.nonzero(block.index == e, as_tuple=True) for e in range(E)]
    f = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    hid, rows = [], []
    for e, (t, j) in enumerate(picks):
        hid.append(torch.relu(q8(h16[t]) @ w1[e].t()).half() if t.numel() else None)
        rows.append((q8(hid[e]) @ w2[e].t()).half() if t.numel() else None)
        if t.numel():
            f.index_add_(0, t, rows[e].double() * w[t, j][:, None])
    f64 = f.half().double().requires_grad_(True)
    gate, w_out = p["gate"].half().double().requires_grad_(True), p["norm_out"].clone().requires_grad_(True)
    ref = x64 + gate * R.norm(f64, 1, w_out, None, 1e-6)
    near(y, ref.detach(), "y")
    (ref * dy.double()).sum().backward(retain_graph=True)
    near(grad["norm_out"], w_out.grad, "norm_out")
    near(grad["gate"], gate.grad, "gate")
    dx_res, df = x64.grad.half(), f64.grad.half()
    dweight = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    dh = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    dw1, dw2 = torch.zeros_like(p["w1"]), torch.zeros_like(p["w2"])
    for e, (t, j) in enumerate(picks):
        if not t.numel():
            continue
        dweight[t, j] = (df[t].double() * rows[e].double()).sum(1)
        g2 = df[t].float() * block.weight[t, j][:, None]
        dw2[e] = q8(g2.t().contiguous()) @ q8(hid[e].t().contiguous()).t()
        g1 = (q8(g2) @ w2[e]).half() * (hid[e] > 0)
        dw1[e] = q8(g1.t().contiguous()) @ q8(h16[t].t().contiguous()).t()
        dh.index_add_(0, t, (q8(g1) @ w1[e]).half().double())
    near(grad["w2"], dw2, "w2")
    near(grad["w1"], dw1, "w1")
    z = block.logits.double().requires_grad_(True)
    s = torch.softmax(z, 1).gather(1, block.index.long())
    (s / s.sum(1, keepdim=True) * dweight).sum().backward()
    if k > 1:  # one expert's weight is 1
        near(grad["router"], z.grad.t() @ h16.double(), "router")
    dh = dh.half().double() + (z.grad @ p["router"])
    x64.grad = None
    (h * dh).sum().backward()
    near(dx, dx_res.double() + x64.grad, "dx")
    near(grad["norm_in"], w_in.grad, "norm_in")


def test_training_learns():
    losses = example().train(steps=120, tokens=4096, verbose=False)
    assert all(v == v for v in losses)
    assert sum(losses[-10:]) < 0.35 * sum(losses[:3]) / 3 * 10, (losses[0], losses[-1])
