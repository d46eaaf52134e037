"""Long rows on either side of the length from which few of them go by parts, and such calls in graphs and on other streams."""
import numpy as np
import pytest
import torch

import class_scores as D
import draw_oracle as R
import score_oracle as O
import test_gpu_sample as G
from test_gpu_class_scores import on_gpu, place
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C,n", [(65_535, 40), (65_536, 40), (65_600, 129), (70_001, 17), (66_000, 385)])
def test_around_the_length(C, n):
    G.test_few_long_rows(C, n)


@pytest.mark.parametrize("C,n", [(16_383, 3), (16_384, 3), (9000, 256), (9000, 257), (20_000, 256), (20_000, 257)])
def test_threads_of_a_row(C, n):
    """A workgroup has more threads where rows are long, and as few as there are CUs."""
    rng = np.random.default_rng(C)
    z = G.rounded(rng.standard_normal((C, n)).astype(np.float32) * 2, torch.float16)
    u = G.numbers(rng, n)
    rows = np.r_[0:3, n // 2, n - 2:n]
    for how in (dict(), dict(p=0.9), dict(k=600, p=0.7, temperature=0.8), dict(min_p=0.05)):
        got = S.sample(place(z, "row", torch.float16, pad=1), torch.from_numpy(u).cuda(), **how)
        G.check(got, R.sample(z[:, rows], u[rows], **how), rows)


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("how", [dict(k=300), dict(p=0.8), dict(k=700, p=0.9, min_p=1e-4)])
def test_streams_graphs_and_repeats(how, order):
    rng = np.random.default_rng(8)
    C, n = 70_000, 9
    z, u = rng.standard_normal((C, n)).astype(np.float32) * 2, G.numbers(rng, n)
    r = D.rules(rng, C, n, sets="each", shown=order == "class")
    want = R.sample(O.adjusted(z, **r), u, **how)
    x, v, g = place(z, order), torch.from_numpy(u).cuda(), on_gpu(r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = S.sample(x, v, **g, **how)
    side.synchronize()
    G.check(first, want)
    graphs = []
    for _ in range(2):  # (each has a workspace of its own)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = S.sample(x, v, **g, **how)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, out in graphs:
            out[0].fill_(-7)
            out[1].fill_(7)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):  # (both at once)
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, first))
        assert all(torch.equal(a, b) for a, b in zip(S.sample(x, v, **g, **how), first))
