"""Calls of one kernel with different amounts of LDS beyond 64 KB: captured ones replayed after smaller eager ones, and two
threads' calls at once."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_gpu_expert_layer import Layer  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("large,small,kw", [
    ((64, 8, 2), (40, 8, 2), dict(code=0)), ((64, 1024, 4), (33, 512, 4), dict(code=2, fmt=1)),
    ((64, 64, 32), (36, 64, 32), dict(code=1))])
def test_replayed_after_a_smaller_call(large, small, kw):
    L, less = Layer(*large, 192, 136, act=3, seed=95, **kw), Layer(*small, 192, 136, act=3, seed=96, **kw)
    want, want_less = L.run().clone(), less.run().clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        L.run(s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            L.run(s.cuda_stream)
        for rep in range(4):
            L.out.fill_(-7)
            less.out.fill_(-7)
            less.run(s.cuda_stream)
            graph.replay()
            s.synchronize()
            assert torch.equal(L.out, want) and torch.equal(less.out, want_less), rep


def test_two_threads():
    jobs = [Layer(T, 8, 2, 192, 136, act=3, code=0, seed=97) for T in (64, 36)]
    want = [j.run().clone() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    bad = []

    def work(j, w, s):
        try:
            for _ in range(50):
                j.run(s.cuda_stream)
            s.synchronize()
            if not torch.equal(j.out, w):
                bad.append(j.size)
        except RuntimeError as e:
            bad.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
