"""Scratch of the launchers that need any (a plan of more than 4,096 slots, the norms' gradients): calls that overlap
on the device do not share it."""
import ctypes as C
import threading

import pytest

torch = pytest.importorskip("torch")

import experts_ref as R  # noqa: E402
from helpers import pkg  # noqa: E402

pytestmark = pytest.mark.gpu
PER_THREAD = 2  # the handle that names another stream in every thread


class Plan:
    def __init__(self, seed, T, k, E, align=16):
        g = R.gen(seed)
        self.size = (T, k, E, align)
        self.idx = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
        self.cap = pkg().lib().routePlanCapacity(T, k, E, align)
        self.out = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, self.cap, T * k)]

    def run(self, stream):
        R.launch("launchRoutePlan", self.idx, *self.size, self.cap, *self.out, stream)

    def clear(self):
        for t in self.out:
            t.fill_(-9)

    def check(self):
        want = R.plan(self.idx, self.size[2], self.size[3], self.cap)
        for got, ref in zip(self.out, want):
            assert got.tolist() == ref


class NormBackward:
    def __init__(self, seed, rows, dim):
        g = R.gen(seed)
        self.rows = rows
        self.x, self.dh = R.randn(g, rows, dim), R.randn(g, rows, dim)
        self.w = 1 + 0.1 * R.randn(g, dim)
        self.out = [torch.empty(rows, dim, device="cuda"), torch.empty(dim, device="cuda")]
        self.o = pkg().NormGateOption(dim=dim, postNorm=0, preNorm=1, gateRows=0, residualScale=1.0, blockScale=1.0,
                                      epsilon=1e-6, dataType=0, strideX=dim, strideF=dim, strideGate=dim, strideY=dim,
                                      strideH=dim)

    def run(self, stream):
        R.launch("launchNormGateResidualBackward", C.byref(self.o), self.x, None, None, None, None, self.w, None, None, self.dh,
                 self.out[0], None, None, None, None, self.out[1], None, self.rows, stream)


def test_streams_of_several_threads():
    """Each thread's own stream under the one handle: every call's results are those of a call by itself."""
    jobs = [[Plan(i, 20000 + 3000 * i, 2, 40 + 30 * i) for i in range(4)], [NormBackward(i, 3000 + 500 * i, 300 + 60 * i) for i in range(4)]]
    for kind in jobs:
        want = []
        for j in kind:
            j.run(R.stream())
            torch.cuda.synchronize()
            want.append([t.clone() for t in j.out])
        errors = []

        def work(j, ref):
            try:
                for _ in range(40):
                    j.run(PER_THREAD)
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(j.out, ref))
            except BaseException as e:  # noqa: BLE001
                errors.append(e)

        threads = [threading.Thread(target=work, args=(j, ref)) for j, ref in zip(kind, want)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
    jobs[0][0].check()


@pytest.mark.parametrize("job,larger", [
    (lambda: Plan(50, 9000, 2, 60), lambda: Plan(51, 400000, 2, 200)),
    (lambda: NormBackward(52, 2000, 200), lambda: NormBackward(53, 8000, 2000))])
def test_a_graph_outlives_larger_calls(job, larger):
    """Captured on a stream whose scratch then grows: what replays use is still theirs."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    j, big = job(), larger()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        j.run(s.cuda_stream)  # its scratch
        s.synchronize()
        want = [t.clone() for t in j.out]
        graph = torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            j.run(s.cuda_stream)
        for i in range(4):
            big.run(s.cuda_stream)
            s.synchronize()
            # whatever was given back is somebody else's now
            others = [torch.full((1 << 18,), -1, dtype=torch.int32, device="cuda") for _ in range(64)]
            for t in j.out:
                t.fill_(-9)
            graph.replay()
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(j.out, want)), i
            assert all(bool((t == -1).all()) for t in others), i
            j.run(s.cuda_stream)
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(j.out, want)), i
            del others
