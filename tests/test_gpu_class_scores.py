"""The operators on class scores against their restatement (score_oracle.py)."""
import numpy as np
import pytest
import torch

import class_scores as D
import score_oracle as O
import thundergbm_amd as T
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def place(z, order, dtype=torch.float32, pad=0, shift=0):
    """The scores on the GPU: [classes, rows] in an order, `pad` more elements between the lines, `shift` in front of all."""
    x = torch.from_numpy(np.ascontiguousarray(z)).to(dtype)
    lines = x if order == "class" else x.t()
    a, b = lines.shape
    memory = torch.full((shift + a * (b + pad) + 7,), 77.0, dtype=dtype, device="cuda")
    view = memory[shift:shift + a * (b + pad)].view(a, b + pad)[:, :b]
    view.copy_(lines)
    return view if order == "class" else view.t()


def on_gpu(r):
    return {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in r.items()}


def rounded(x, dtype):
    """The scores that the operators see: rounded to their type."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).float().numpy()


def same(got, want):
    """Equal, NaNs being equal to each other."""
    got, want = got.float().cpu().numpy(), np.asarray(want, np.float32)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.nan_to_num(got, nan=0.0, posinf=np.inf, neginf=-np.inf), np.nan_to_num(want, nan=0.0, posinf=np.inf, neginf=-np.inf))


SIZES = [(1, 1), (3, 1), (1, 5), (8, 1000), (31, 65), (33, 64), (100, 16), (129, 63), (257, 300), (1025, 40), (8193, 3), (16400, 2), (70_000, 1)]


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", SIZES)
def test_adjust(C, n, order):
    rng = np.random.default_rng(C * 7 + n)
    for k, dtype in enumerate(TYPES):
        z = rounded(D.scores(rng, C, n, special=0.1), dtype)
        r = D.rules(rng, C, n, sets=("each", "some", "one")[k], longest=(9, 40, 2)[k])
        want = rounded(O.adjusted(z, **r), dtype)
        x = place(z, order, dtype, pad=k, shift=k)
        got = S.adjust(x, **on_gpu(r))
        assert got.dtype == dtype and got.shape == x.shape
        same(got, want)


@pytest.mark.parametrize("bias,sets,shown", [(b, m, h) for b in (False, True) for m in ("none", "one", "some") for h in (False, True)])
@pytest.mark.parametrize("order", ["class", "row"])
def test_adjust_parts_left_out(order, bias, sets, shown):
    rng = np.random.default_rng(3)
    z = D.scores(rng, 70, 90, special=0.05)
    r = D.rules(rng, 70, 90, bias=bias, sets=sets, shown=shown)
    same(S.adjust(place(z, order), **on_gpu(r)), O.adjusted(z, **r))


@pytest.mark.parametrize("order", ["class", "row"])
def test_adjust_writes_only_its_part(order):
    """Into another order, into a part of an array, in place, next to its own input."""
    rng = np.random.default_rng(4)
    C, n = 37, 131
    z = D.scores(rng, C, n)
    r = D.rules(rng, C, n)
    want, g = O.adjusted(z, **r), on_gpu(r)
    for other in ("class", "row"):
        x, out = place(z, order), place(np.zeros((C, n), np.float32), other, pad=3, shift=5)
        memory = out._base if out._base is not None else out
        before = memory.clone()
        assert S.adjust(x, out=out, **g) is out
        same(out, want)
        same(x, z)
        out.copy_(torch.zeros_like(out))
        assert torch.equal(memory, before)
    x = place(z, order, pad=2)
    S.adjust(x, out=x, **g)
    same(x, want)
    both = torch.zeros(C, 2 * n, device="cuda") if order == "class" else torch.zeros(n, 2 * C, device="cuda")
    a, b = (both[:, :n], both[:, n:]) if order == "class" else (both[:, :C].t(), both[:, C:].t())
    a.copy_(torch.from_numpy(z))
    S.adjust(a, out=b, **g)
    same(a, z)
    same(b, want)


def test_adjust_lists_out_of_range():
    """Parts of the list that do not lie in it are cut, rows of one list overlap, a list is very long, one class fills a list."""
    rng = np.random.default_rng(5)
    C, n = 50, 6
    z = D.scores(rng, C, n)
    shown = np.concatenate([rng.integers(0, C, 3000), np.full(70_000, 7)]).astype(np.int32)
    begin = np.array([-5, 10, 4, 3000, 2_000_000, 100, 73_000], np.int64)  # [-5, 10) [10, 4) [4, 3000) [3000, 2e6) [2e6, 100) [100, end)
    r = dict(shown=shown, shown_begin=begin, repetition=0.5, frequency=1e-3, presence=-1.0)
    want = O.adjusted(z, **r)
    assert np.any(want != z)
    for order in ("class", "row"):
        same(S.adjust(place(z, order), **on_gpu(r)), want)


def test_adjust_of_nothing():
    x = torch.zeros(5, 0, device="cuda")
    assert S.adjust(x).shape == (5, 0)
    x = torch.randn(4, 6, device="cuda")
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert torch.equal(S.adjust(x, shown=empty, shown_begin=torch.zeros(7, dtype=torch.int64, device="cuda")), x)


def test_adjust_refuses():
    x = torch.zeros(8, 10, device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    begin = torch.zeros(11, dtype=torch.int64, device="cuda")
    bad = [
        (dict(scores=x.double()), "float32, float16 or bfloat16"),
        (dict(scores=x[0]), "dimensions"),
        (dict(scores=x[:, ::2]), "side by side"),
        (dict(scores=x[:, :1].expand(8, 10)), "side by side"),
        (dict(scores=torch.zeros(0, 3, device="cuda")), "0 classes"),
        (dict(scores=x.clone().requires_grad_()), "autograd"),
        (dict(bias=torch.zeros(7, device="cuda")), "bias"),
        (dict(bias=torch.zeros(8)), "on the GPU"),
        (dict(bias=torch.zeros(8, device="cuda").half()), "bias"),
        (dict(bias=torch.zeros(16, device="cuda")[::2]), "contiguous"),
        (dict(allowed=i32(1, 2)), "allowed"),
        (dict(allowed=i32(3, 1)), "3 sets for 10 rows"),
        (dict(allowed=i32(1)), "allowed"),
        (dict(allowed_set=i32(10)), "without allowed"),
        (dict(allowed=i32(3, 1), allowed_set=i32(9)), "allowed_set"),
        (dict(shown=i32(4)), "belong together"),
        (dict(shown_begin=begin), "belong together"),
        (dict(shown=i32(4), shown_begin=begin[:-1]), "shown_begin"),
        (dict(shown=i32(4), shown_begin=begin.int()), "shown_begin"),
        (dict(shown=i32(4), shown_begin=begin, repetition=0.0), "repetition"),
        (dict(shown=i32(4), shown_begin=begin, frequency=float("nan")), "frequency"),
        (dict(out=torch.zeros(8, 9, device="cuda")), "out"),
        (dict(out=x.half()), "out"),
        (dict(scores=torch.zeros(10, 10, device="cuda").t(), out=None), None),
    ]
    for more, msg in bad:
        if msg is not None:
            with pytest.raises(ValueError, match=msg):
                S.adjust(**dict(dict(scores=x), **more))
    square = torch.zeros(10, 10, device="cuda")
    with pytest.raises(ValueError, match="another order"):
        S.adjust(square, out=square.t())
    wide = torch.zeros(8, 15, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        S.adjust(wide[:, :10], out=wide[:, 5:])


def test_adjust_on_a_stream_and_in_a_graph():
    """Launched on the current stream; a captured call replays on new data, whatever runs in between."""
    rng = np.random.default_rng(6)
    C, n = 300, 200
    z = D.scores(rng, C, n)
    r = D.rules(rng, C, n)
    g, want = on_gpu(r), O.adjusted(z, **r)
    side = torch.cuda.Stream()
    x = place(z, "class")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        got = S.adjust(late, **g)
    torch.cuda.current_stream().wait_stream(side)
    same(got, want)
    graph = torch.cuda.CUDAGraph()
    S.adjust(x, **g)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = S.adjust(x, **g)
    for k in range(4):
        z2 = D.scores(rng, C, n)
        x.copy_(torch.from_numpy(z2))
        graph.replay()
        other = S.adjust(torch.zeros_like(x), **g)
        torch.cuda.synchronize()
        same(captured, O.adjusted(z2, **r))
        same(other, O.adjusted(np.zeros_like(z2), **r))
