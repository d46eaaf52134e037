"""Rows in 8 bits and class scores as their product against their restatement (draw_oracle.py)."""
import numpy as np
import pytest
import torch

import draw_oracle as R
import score_oracle as O
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step of a rounding, relative (32 bits: counted with the other steps)
LEAST = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}  # half a step of the numbers below the least normal one


def strided(x, pad=0, shift=0):
    """A copy on the GPU with `pad` more elements between the rows, `shift` in front of all, nothing of its own behind the last row."""
    rows, width = x.shape
    memory = torch.full((shift + rows * (width + pad) - (pad if rows else 0),), 77, dtype=x.dtype, device="cuda")
    view = memory.as_strided((rows, width), (width + pad, 1), shift)
    view.copy_(x)
    return view


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,F", [(1, 1), (3, 7), (1, 4096), (5, 127), (64, 128), (70, 129), (1000, 28), (2, 65_536), (33, 1000), (9, 16_387), (4, 2048)])
def test_quantise(n, F, dtype):
    rng = np.random.default_rng(n + F)
    x = torch.from_numpy(rng.standard_normal((n, F)).astype(np.float32) * rng.choice([1e-30, 1.0, 1e3], (n, 1)).astype(np.float32)).to(dtype)
    for i in range(0, n, 5):
        x[i, rng.integers(F)] = (0.0, float("inf"), float("nan"), float("-inf"))[i // 5 % 4]
    if n > 2:
        x[2] = 0.0
    for pad in (0, 3):
        q, scale = S.quantise(strided(x, pad, shift=pad))
        want_q, want_scale = R.quantise(x.float().numpy())
        np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
        np.testing.assert_array_equal(q.cpu().numpy(), want_q)
        assert q.stride(0) % 128 == 0 or n == 1
        assert not torch.count_nonzero(q._base[:, F:])


def test_quantise_ends():
    """Halves go to even numbers; the smallest numbers there are; a row whose largest is the largest there is."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5], [254.0, 1.0, 3.0, 5.0, -1.0, -3.0, -253.0], [1e-45, 0, -1e-45, 1e-45, 0, 0, 0],
                      [3.4028235e38, 1.3396e36, -3.4028235e38, 0, 1, 2, 3], [1e-38, -1e-40, 5e-39, 0, 0, 0, 1e-45]], dtype=torch.float32)
    q, scale = S.quantise(x.cuda())
    want_q, want_scale = R.quantise(x.numpy())
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -126]


def case(rng, n, F, C):
    q = torch.from_numpy(rng.integers(-128, 128, (n, F)).astype(np.int8))
    w = torch.from_numpy(rng.integers(-128, 128, (C, F)).astype(np.int8))
    scale = torch.from_numpy((rng.random(n) + 0.5).astype(np.float32) / 100)
    w_scale = torch.from_numpy((rng.random(C) + 0.5).astype(np.float32) / np.float32(F * 3))
    bias = torch.from_numpy(rng.standard_normal(C).astype(np.float32))
    return q, scale, w, w_scale, bias


def check(got, q, scale, w, w_scale, bias, dtype):
    z, room = R.linear(q.numpy(), scale.numpy(), w.numpy(), w_scale.numpy(), None if bias is None else bias.numpy())
    assert got.dtype == dtype and tuple(got.shape) == z.shape
    room = room + HALF[dtype] * (np.abs(z) + room) + LEAST[dtype]
    off = np.abs(got.double().cpu().numpy() - z)
    assert np.all(off <= room), (np.max(off / room), np.argmax(off / room))


SIZES = [(1, 1, 1), (1, 28, 8), (2, 16, 33), (3, 100, 500), (1, 4096, 1000), (1, 200, 70_001), (5, 1000, 257), (16, 64, 64), (17, 129, 65), (24, 1000, 5021), (33, 384, 300),
         (63, 2048, 130), (64, 512, 1024), (65, 130, 129), (100, 8192, 40), (128, 128, 128), (129, 255, 257), (200, 8192, 500), (257, 640, 513), (500, 33, 1000),
         (1000, 1024, 1000), (3000, 200, 2), (10_001, 28, 9), (70_000, 16, 3), (2048, 256, 2049), (4, 65_536, 20), (300, 20_000, 260)]


@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("n,F,C", SIZES)
def test_linear(n, F, C, order):
    rng = np.random.default_rng(n + 3 * F + C)
    q, scale, w, w_scale, bias = case(rng, n, F, C)
    for j, dtype in enumerate(TYPES):
        pad_x, pad_w = ((0, 0), (-F % 16, -F % 128), (5, 3))[(j + n) % 3]
        b = bias if j != 1 else None
        got = S.linear(strided(q, pad_x, shift=j), strided(w, pad_w, shift=16 * (j != 2) + j // 2), w_scale.cuda(), bias=None if b is None else b.cuda(), x_scale=scale.cuda(),
                       order=order, dtype=dtype)
        assert got.is_contiguous() if order == "class" else got.t().is_contiguous()
        check(got, q, scale, w, w_scale, b, dtype)


@pytest.mark.parametrize("n,F,C", [(1, 28, 8), (1, 4096, 3000), (7, 300, 1000), (24, 1000, 700), (130, 129, 260), (1000, 200, 500), (3, 16_387, 40)])
def test_linear_of_floating_rows(n, F, C):
    """They are quantised as `quantise` does."""
    rng = np.random.default_rng(n * F + C)
    _, _, w, w_scale, bias = case(rng, 1, F, C)
    for j, dtype in enumerate(TYPES):
        x = torch.from_numpy(rng.standard_normal((n, F)).astype(np.float32) * 3).to(dtype)
        q, scale = R.quantise(x.float().numpy())
        for order in ("row", "class"):
            weights, of_weights = S.quantise(strided(w).float())  # (laid out as quantise does)
            weights.copy_(w)
            got = S.linear(strided(x, pad=j, shift=j), weights, w_scale.cuda(), bias=bias.cuda(), order=order)
            check(got, torch.from_numpy(q), torch.from_numpy(scale), w, w_scale, bias, torch.float32)


def test_rows_without_a_scale():
    x = torch.randn(6, 40, device="cuda")
    x[1, 3], x[2, 39], x[4] = float("nan"), float("inf"), 0.0
    w, w_scale = S.quantise(torch.randn(9, 40, device="cuda"))
    bias = torch.arange(9.0, device="cuda")
    for order in ("row", "class"):
        z = S.linear(x, w, w_scale, bias=bias, order=order)
        assert bool(torch.isnan(z[:, [1, 2]]).all()) and bool(torch.isfinite(z[:, [0, 3, 4, 5]]).all()) and torch.equal(z[:, 4], bias)


def test_largest_sums():
    """65536 features whose products are all the largest or the least."""
    F = 65_536
    q = torch.full((3, F), -128, dtype=torch.int8)
    w = torch.full((2, F), -128, dtype=torch.int8)
    w[1] = 127
    one = torch.ones(3)
    got = S.linear(q.cuda(), w.cuda(), torch.ones(2, device="cuda"), x_scale=one.cuda())
    assert got.tolist() == [[2.0**30] * 3, [-128.0 * 127 * F] * 3]


def test_nothing_else_is_written_and_repeats_are_equal():
    rng = np.random.default_rng(5)
    for n, F, C in ((5, 100, 70), (300, 256, 400)):
        q, scale, w, w_scale, bias = (v.cuda() for v in case(rng, n, F, C))
        first = S.linear(q, w, w_scale, bias=bias, x_scale=scale)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = S.linear(q, w, w_scale, bias=bias, x_scale=scale)
        side.synchronize()
        assert torch.equal(first, again)
        x = torch.randn(n, F, device="cuda")
        eager = S.linear(x, w, w_scale, bias=bias, order="class")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = S.linear(x, w, w_scale, bias=bias, order="class")
        for _ in range(3):
            out.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            assert torch.equal(S.linear(x, w, w_scale, bias=bias, order="class"), eager)


def test_many_rows():
    """More rows than a launch or a part of the workspace takes."""
    gen = torch.Generator("cuda").manual_seed(1)
    for n, F, C in ((1_300_000, 40, 3), (70_000, 9000, 5)):
        x = torch.randn(n, F, device="cuda", generator=gen, dtype=torch.float32).bfloat16()
        w, w_scale = S.quantise(torch.randn(C, F, device="cuda", generator=gen))
        q, scale = S.quantise(x)
        at = torch.tensor([0, 1, n // 2, (1 << 20) - 1, 1 << 20, 59_578, 59_579, n - 1], device="cuda").clamp(max=n - 1)
        want_q, want_scale = R.quantise(x[at].float().cpu().numpy())
        np.testing.assert_array_equal(q[at].cpu().numpy(), want_q)
        np.testing.assert_array_equal(scale[at].cpu().numpy(), want_scale)
        for order in ("row", "class"):
            z = S.linear(x, w, w_scale, order=order)
            check(z[:, at], torch.from_numpy(want_q), torch.from_numpy(want_scale), w.cpu(), w_scale.cpu(), None, torch.float32)
            assert torch.equal(z, S.linear(q, w, w_scale, x_scale=scale, order=order))


@pytest.mark.parametrize("n,C", [(1024, 32_769), (1024, 32_768 + 130), (33_000, 1000)])
def test_large_tiles_and_what_is_left_behind_them(n, C):
    """Lines behind the last whole tile, which go by smaller ones where they would fill no round of their own; the sums as exact numbers of 64 bits."""
    gen = torch.Generator("cuda").manual_seed(n)
    q, w = (torch.randint(-127, 128, (r, 640), device="cuda", generator=gen, dtype=torch.int32).to(torch.int8) for r in (n, C))
    scale, w_scale, bias = torch.rand(n, device="cuda", generator=gen) + 0.5, torch.rand(C, device="cuda", generator=gen) + 0.5, torch.randn(C, device="cuda", generator=gen)
    total = w.double() @ q.double().t().contiguous()
    for order in ("row", "class"):
        z = S.linear(q, w, w_scale, bias=bias, x_scale=scale, order=order)
        assert torch.equal(z, total.float() * scale * w_scale[:, None] + bias[:, None])


def test_two_streams_at_once():
    """Calls that run side by side have workspaces of their own."""
    gen = torch.Generator("cuda").manual_seed(2)
    x = [torch.randn(700, 300, device="cuda", generator=gen) for _ in range(2)]
    w, w_scale = S.quantise(torch.randn(900, 300, device="cuda", generator=gen))
    u = torch.rand(700, device="cuda", generator=gen)

    def chain(v):
        z = S.linear(v, w, w_scale)
        return (z, *S.sample(z, u, p=0.9), *S.sample(z, u, k=20))

    want = [chain(v) for v in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(chain(x[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


def test_no_rows():
    w, w_scale = S.quantise(torch.randn(9, 40, device="cuda"))
    assert S.linear(torch.zeros(0, 40, device="cuda"), w, w_scale).shape == (9, 0)
    q, scale = S.quantise(torch.zeros(0, 40, device="cuda"))
    assert q.shape == (0, 40) and scale.shape == (0,)


@pytest.mark.parametrize("n,F,C", [(40, 300, 1000), (700, 64, 50)])
def test_a_layer_its_best_classes_and_draws_together(n, F, C):
    """As they are used: scores of a layer, the best classes of them, a draw among those, and the loss of other scores against them."""
    rng = np.random.default_rng(C)
    x = torch.from_numpy(rng.standard_normal((n, F)).astype(np.float32)).cuda()
    w, w_scale = S.quantise(torch.from_numpy(rng.standard_normal((C, F)).astype(np.float32)).cuda())
    u = rng.random(n).astype(np.float32)
    z = S.linear(x, w, w_scale, order="class")
    values, classes, lse = S.top(z, 10)
    drawn, logp = S.sample(z, torch.from_numpy(u).cuda(), k=10)
    want, want_logp = R.sample(z.cpu().numpy(), u, k=10)
    np.testing.assert_array_equal(drawn.cpu().numpy(), want)
    np.testing.assert_allclose(logp.cpu().numpy(), want_logp, rtol=2.0**-24 * 1.01, atol=1e-11)
    assert bool((classes == drawn[:, None]).any(1).all())
    # z against its own ten best classes and what they leave: nothing but rounding, of which the restatement of distill says how much there may be
    loss, pairs = S.distill(z, classes, values, teacher_lse=lse)
    want, want_pairs, room, pairs_room = O.distill(z.cpu().numpy(), classes.cpu().numpy(), values.cpu().numpy(), lse=lse.cpu().numpy())
    assert np.all(np.abs(loss.cpu().numpy() - want) <= room) and np.all(np.abs(pairs.cpu().numpy() - want_pairs) <= pairs_room)


def test_refusals():
    x = torch.zeros(6, 40, device="cuda")
    w, w_scale = S.quantise(torch.ones(9, 40, device="cuda"))
    q, scale = S.quantise(x)
    for args in (dict(x=x.double()), dict(x=x[0]), dict(x=x[:, ::2]), dict(x=x.t()), dict(x=x[:, :39]), dict(x=q), dict(x=x, x_scale=scale), dict(x=q, x_scale=scale[:5]),
                 dict(x=q, x_scale=scale.double()), dict(x=x.clone().requires_grad_()), dict(weight=w.float()), dict(weight=w[0]), dict(weight=w.cpu()), dict(weight_scale=None),
                 dict(weight_scale=w_scale[:8]), dict(weight_scale=w_scale.cpu()), dict(bias=w_scale[:8]), dict(bias=w_scale.half()), dict(order="column"), dict(dtype=torch.int8),
                 dict(dtype=torch.float64), dict(weight=w[:0], weight_scale=w_scale[:0])):
        with pytest.raises(ValueError):
            S.linear(**{**dict(x=x, weight=w, weight_scale=w_scale), **args})
    for bad in (x.double(), x[0], x.t(), x[:, :0], q, torch.zeros(2, 65_537, device="cuda"), x.cpu(), None):
        with pytest.raises(ValueError):
            S.quantise(bad)
