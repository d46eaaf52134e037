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


def check_top(got, x, k, temperature=1.0):
    values, classes, lse = got
    want_values, want_classes, want_lse = O.top(x, k, temperature)
    np.testing.assert_array_equal(classes.cpu().numpy(), want_classes)
    same(values, want_values)
    # Half steps of 2^-24: three in the argument of an exponential, which its weight makes at most ln C of on average, two in
    # its value, one for every addition in a row (at most 32 + 6 + 16 + 9), two in the quotient and the sum with it, four
    # in the logarithm.
    lse, C = lse.cpu().numpy().astype(np.float64), x.shape[0]
    fine = np.isfinite(want_lse)
    np.testing.assert_array_equal(lse[~fine], want_lse[~fine])
    with np.errstate(all="ignore"):
        largest = np.abs(np.where(fine, x.max(0), 0) / temperature)
    room = 2.0**-24 * (7 * np.log(C) + 70 + np.where(fine, largest + np.abs(want_lse), 0))
    assert np.all(np.abs(lse[fine] - want_lse[fine]) <= room[fine])


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", SIZES + [(2, 300), (17, 77), (32, 500), (64, 130), (512, 9), (1024, 33), (2048, 5), (2049, 600)])
def test_top(C, n, order):
    rng = np.random.default_rng(C * 11 + n)
    for j, dtype in enumerate(TYPES):
        special = (0.1, 0.0, 0.02)[j]
        z = rounded(D.scores(rng, C, n, special=special), dtype)
        r = D.rules(rng, C, n, bias=j != 1, sets=("each", "none", "some")[j], shown=j != 2, longest=9)
        x = O.adjusted(z, **r)
        for k, temperature in ((1, 1.0), (min(C, 7), 0.5), (128 if j else 64, 3.0)):
            check_top(S.top(place(z, order, dtype, pad=j, shift=j), k, temperature=temperature, **on_gpu(r)), x, k, temperature)


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", [(30, 40), (1000, 20), (5000, 3), (40_000, 2)])
def test_top_equal_scores(C, n, order):
    """All equal, two values, one class allowed, nothing allowed, the lowest number, infinities."""
    rng = np.random.default_rng(9)
    z = np.zeros((C, n), np.float32)
    for k in (1, 5, 128):
        check_top(S.top(place(z, order), k), z, k)
        z2 = (rng.random((C, n)) < 0.5).astype(np.float32) * np.where(rng.random((C, n)) < 0.5, 0.0, -0.0).astype(np.float32)
        z2[rng.random((C, n)) < 0.01] = 1
        check_top(S.top(place(z2, order), k), z2, k)
        z3 = np.full((C, n), -np.inf, np.float32)
        z3[rng.integers(0, C, n), np.arange(n)] = -3.4028235e38
        check_top(S.top(place(z3, order), k), z3, k)
        z3[:, ::2] = -np.inf
        z3[C // 2:, 1::2] = 3.4028235e38
        check_top(S.top(place(z3, order), k), z3, k)
        z3[C // 3, :] = np.inf
        z3[C // 4, 0] = np.inf
        check_top(S.top(place(z3, order), k), z3, k)
        z3[C // 5, 0] = np.nan
        check_top(S.top(place(z3, order), k), z3, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C", [700, 1024, 2048, 8192, 16_384, 40_000])
def test_top_best_in_few_threads(C, order, dtype):
    """The best classes at distances at which one thread, or one wavefront, holds all of them: more candidates than the list takes."""
    rng = np.random.default_rng(C)
    rows = []
    for step in (64, 256, 512, 1024, 2048, 4096):
        for run in (1, 4, 8):
            z = rng.standard_normal(C).astype(np.float32)
            at = np.arange(C)
            z[at % step < run] += 100
            rows.append(z)
            rows.append(np.where(at % step < run, 2.0, np.round(z / 50)).astype(np.float32))
    rows.append(np.sort(rng.standard_normal(C)).astype(np.float32))
    rows.append(rows[-1][::-1].copy())
    z = rounded(np.stack(rows, 1), dtype)
    for k in (3, 64, 128):
        check_top(S.top(place(z, order, dtype), k), z, k)


def test_top_chunks_of_chunks():
    """So many classes that the chunks' best ones are joined twice."""
    C = 300_000
    z = D.scores(np.random.default_rng(1), C, 2)
    check_top(S.top(place(z, "class"), 128), z, 128)
    check_top(S.top(place(z, "row"), 128), z, 128)


def test_top_refuses():
    x = torch.zeros(8, 10, device="cuda")
    for more, msg in ((dict(k=0), "k is 0"), (dict(k=129), "k is 129"), (dict(k=1.5), "k is 1.5"), (dict(k=2, temperature=0.0), "temperature"),
                      (dict(k=2, temperature=float("nan")), "temperature"), (dict(k=2, bias=torch.zeros(7, device="cuda")), "bias"),
                      (dict(scores=x.int(), k=2), "float32")):
        with pytest.raises(ValueError, match=msg):
            S.top(**dict(dict(scores=x), **more))
    values, classes, lse = S.top(torch.zeros(5, 0, device="cuda"), 3)
    assert values.shape == classes.shape == (0, 3) and lse.shape == (0,)


def test_top_two_graphs():
    """Two captured calls of different sizes and an eager one take turns: each has its own workspace."""
    rng = np.random.default_rng(8)
    shapes = [(40_000, 3, 64), (5000, 7, 20), (300, 500, 10)]
    graphs = []
    for C, n, k in shapes:
        x = place(D.scores(rng, C, n), "row")
        S.top(x, k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = S.top(x, k)
        graphs.append((graph, x, k, got))
    for _ in range(3):
        news = []
        for graph, x, k, got in graphs:
            z = D.scores(rng, *x.shape)
            x.copy_(torch.from_numpy(z))
            news.append(z)
        for graph, *_ in graphs:
            graph.replay()
        eager = S.top(graphs[0][1], 5)
        for (graph, x, k, got), z in zip(graphs, news):
            check_top(got, z, k)
        check_top(eager, news[0], 5)


def check_distill(got, want):
    loss, pairs, loss_room, pairs_room = want
    l = got[0].cpu().numpy().astype(np.float64)
    with np.errstate(all="ignore"):
        assert np.array_equal(np.isfinite(l), np.isfinite(loss)), (l, loss)
        off = np.abs(l - loss)
    fine = np.isfinite(loss)
    assert np.array_equal(l[~fine & ~np.isnan(loss)], loss[~fine & ~np.isnan(loss)])
    assert np.all(off[fine] <= loss_room[fine]), np.max(off[fine] / loss_room[fine])
    if got[1] is not None:
        p = got[1].cpu().numpy().astype(np.float64)
        off = np.abs(p - pairs) / pairs_room
        assert np.all(off <= 1), (off.max(), np.unravel_index(off.argmax(), off.shape))


DISTILL_SIZES = [(1, 1, 1), (3, 1, 2), (8, 1, 8), (8, 1000, 5), (9, 257, 9), (31, 65, 40), (100, 16, 10), (129, 63, 64), (300, 300, 128), (1000, 40, 32), (1300, 17, 20),
                 (5000, 5, 128), (20_000, 2, 7), (30_000, 1, 128), (40_000, 33, 16)]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("C,n,K", DISTILL_SIZES)
def test_distill(C, n, K, rest):
    rng = np.random.default_rng(C + n + K)
    for j, dtype in enumerate(TYPES):
        temperature, weight = ((1.0, 1.0), (2.0, 0.5), (0.7, 0.25))[j]
        z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
        classes, t, full = D.teacher(rng, C, n, K, repeated=j == 1)
        t = rounded(t, dtype)
        lse = np.log(np.exp(full.astype(np.float64) / temperature).sum(1)).astype(np.float32) if rest else None
        labels = rng.integers(0, C, n).astype(np.float32)
        labels[::5] = np.array([-1, C, 0.5, np.nan, np.inf], np.float32)[np.arange(len(labels[::5])) % 5]
        want = O.distill(z, classes, t, labels, lse, temperature, weight)
        g = dict(classes=torch.from_numpy(classes).cuda(), teacher=torch.from_numpy(t).to(dtype).cuda(), temperature=temperature, weight=weight,
                 teacher_lse=None if lse is None else torch.from_numpy(lse).cuda(), labels=torch.from_numpy(labels).cuda())
        x = place(z, "class", pad=j, shift=j)
        check_distill(S.distill(x, **g), want)
        loss, none = S.distill(x, gradient=False, **g)
        assert none is None
        check_distill((loss, None), want)


def test_distill_is_the_objective_without_a_teacher():
    """weight 0: the gradient pairs of multi:softmax."""
    rng = np.random.default_rng(2)
    C, n = 8, 500
    z = (rng.standard_normal((C, n)) * 3).astype(np.float32)
    y = rng.integers(0, C, n).astype(np.float32)
    classes = torch.full((n, 1), -1, dtype=torch.int32, device="cuda")
    loss, pairs = S.distill(place(z, "class"), classes, torch.zeros(n, 1, device="cuda"), labels=torch.from_numpy(y).cuda(), weight=0.0)
    p = np.exp(O.log_softmax(z.astype(np.float64)))
    g = p - (np.arange(C)[:, None] == y)
    # (the room of an exponential, a sum of eight and their quotient; 1 - p as well)
    np.testing.assert_allclose(pairs[..., 0].cpu().numpy(), g, rtol=0, atol=2.0**-24 * 60)
    np.testing.assert_allclose(pairs[..., 1].cpu().numpy(), np.maximum(2 * p * (1 - p), 1e-16), rtol=0, atol=2.0**-24 * 60)


@pytest.mark.parametrize("rest", [False, True])
def test_distill_gradient_is_the_loss_s(rest):
    """The gradient against differences of the loss, in 64 bits in the restatement, and the kernel's against that one."""
    rng = np.random.default_rng(12)
    C, n, K = 6, 9, 3
    z = rng.standard_normal((C, n))
    classes, t, full = D.teacher(rng, C, n, K, repeated=True)
    lse = np.log(np.exp(full.astype(np.float64) / 2).sum(1)).astype(np.float32) if rest else None
    y = rng.integers(0, C, n).astype(np.float32)
    args = (classes, t, y, lse, 2.0, 0.75)
    step = 1e-5
    loss, pairs, *_ = O.distill(z, *args)
    for c in range(C):
        up, down = z.copy(), z.copy()
        up[c] += step
        down[c] -= step
        slope = (O.distill(up, *args)[0] - O.distill(down, *args)[0]) / (2 * step)
        # (a third derivative of at most about T^-1 = 0.5 times step^2 / 6, and 2^-52 of the loss over the step)
        np.testing.assert_allclose(pairs[c, :, 0], slope, rtol=0, atol=1e-9)
    z32 = z.astype(np.float32)
    check_distill(S.distill(place(z32, "class"), torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda(), labels=torch.from_numpy(y).cuda(),
                            teacher_lse=None if lse is None else torch.from_numpy(lse).cuda(), temperature=2.0, weight=0.75), O.distill(z32, *args))


@pytest.mark.parametrize("C,n", [(5, 6), (2000, 6), (40_000, 6)])
def test_distill_far_scores(C, n):
    """The student is far from the teacher: p of the others far below what 32 bits hold, every class named, scores of -inf, NaN."""
    rng = np.random.default_rng(C)
    K = min(C, 5)
    z = (rng.standard_normal((C, n))).astype(np.float32)
    classes = np.tile(np.arange(K, dtype=np.int32), (n, 1))
    t = rng.standard_normal((n, K)).astype(np.float32)
    lse = (np.log(np.exp(t.astype(np.float64)).sum(1)) + 0.3).astype(np.float32)
    z[K:, 0] -= 500        # the others' part is exp(-500)
    z[:K, 1] -= 500        # the named ones'
    z[:, 2] *= 100
    z[K - 1, 3] = -np.inf  # a named class that the student rules out: the loss is infinite
    z[:, 4] = -np.inf      # every class ruled out
    for rest in (None, lse):
        want = O.distill(z, classes, t, None, rest)
        got = S.distill(place(z, "class"), torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda(),
                        teacher_lse=None if rest is None else torch.from_numpy(rest).cuda())
        check_distill(got, want)
        bad = z.copy()
        bad[C // 2, 1] = np.nan
        bad[0, 2] = np.inf
        loss, pairs = S.distill(place(bad, "class"), torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda())
        assert torch.isnan(loss).tolist() == [False, True, True, False, False, False]
        assert torch.isnan(pairs).all(2).all(0).tolist() == [False, True, True, False, False, False]
        assert torch.isfinite(pairs).all(2).all(0).tolist() == [True, False, False, True, True, True]


def test_distill_teacher_s_odd_scores():
    """A NaN or an infinite score of the teacher's makes the row NaN, wherever the entry's class is one; the others keep theirs."""
    rng = np.random.default_rng(6)
    for C, n, K in ((6, 5, 3), (40_000, 5, 3)):
        z = rng.standard_normal((C, n)).astype(np.float32)
        classes = np.tile(np.arange(K, dtype=np.int32), (n, 1))
        t = rng.standard_normal((n, K)).astype(np.float32)
        t[0, 1], t[1, 0], t[2, 2], t[3, 0] = np.nan, np.inf, np.nan, -np.inf
        classes[2, 2] = C  # (left out)
        for lse in (None, torch.full((n,), 3.0, device="cuda")):
            loss, pairs = S.distill(place(z, "class"), torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda(), teacher_lse=lse)
            assert torch.isnan(loss).tolist() == [True, True, False, False, False]
            assert torch.isnan(pairs).all(2).all(0).tolist() == [True, True, False, False, False]
            fine = np.arange(2, 5)
            want = O.distill(z[:, fine], classes[fine], t[fine], None, None if lse is None else np.full(3, 3.0))
            check_distill((loss[2:], pairs[:, 2:]), want)


def test_distill_same_answer_twice():
    rng = np.random.default_rng(3)
    for C, n, K in ((8, 1000, 5), (1000, 100, 32), (40_000, 9, 64)):
        z = place(D.scores(rng, C, n), "class")
        classes, t, _ = D.teacher(rng, C, n, K, repeated=True)
        args = (z, torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda())
        a, b = S.distill(*args), S.distill(*args)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_distill_refuses():
    x = torch.zeros(8, 10, device="cuda")
    c, t = torch.zeros(10, 3, dtype=torch.int32, device="cuda"), torch.zeros(10, 3, device="cuda")
    for more, msg in (
        (dict(scores=torch.zeros(10, 8, device="cuda").t()), "side by side"),
        (dict(scores=x.half()), "float32"),
        (dict(classes=c.long()), "classes"),
        (dict(classes=c[:9]), "classes"),
        (dict(teacher=t.double()), "teacher"),
        (dict(teacher=t[:, :0]), "teacher"),
        (dict(teacher=torch.zeros(10, 129, device="cuda"), classes=torch.zeros(10, 129, dtype=torch.int32, device="cuda")), "128"),
        (dict(teacher=torch.zeros(3, 10, device="cuda").t()), "contiguous"),
        (dict(teacher_lse=torch.zeros(9, device="cuda")), "teacher_lse"),
        (dict(temperature=0.0), "temperature"),
        (dict(weight=1.5), "weight"),
        (dict(weight=float("nan")), "weight"),
        (dict(weight=0.5), "labels"),
        (dict(labels=torch.zeros(10, dtype=torch.int64, device="cuda"), weight=0.5), "labels"),
    ):
        with pytest.raises(ValueError, match=msg):
            S.distill(**dict(dict(scores=x, classes=c, teacher=t), **more))
    loss, pairs = S.distill(torch.zeros(5, 0, device="cuda"), c[:0], t[:0])
    assert loss.shape == (0,) and pairs.shape == (5, 0, 2)


def test_distill_in_a_graph():
    rng = np.random.default_rng(4)
    for C, n, K in ((30, 200, 6), (30_000, 4, 20)):
        z = place(rng.standard_normal((C, n)).astype(np.float32), "class")
        classes, t, _ = D.teacher(rng, C, n, K)
        c, s = torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda()
        S.distill(z, c, s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = S.distill(z, c, s)
        for _ in range(3):
            z2 = rng.standard_normal((C, n)).astype(np.float32)
            z.copy_(torch.from_numpy(z2))
            graph.replay()
            eager = S.distill(z, c, s)
            torch.cuda.synchronize()
            assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
            check_distill(got, O.distill(z2, classes, t))


def test_from_a_teacher_s_scores_to_pairs():
    """A teacher's scores, adjusted and listed, and a student held against them: the calls one behind the other."""
    rng = np.random.default_rng(5)
    C, n, k, temperature = 400, 150, 12, 2.0
    full = rounded(D.scores(rng, C, n), torch.bfloat16)
    r = D.rules(rng, C, n, sets="one")
    x = O.adjusted(full, **r)
    values, classes, lse = S.top(place(full, "row", torch.bfloat16), k, temperature=temperature, **on_gpu(r))
    check_top((values, classes, lse), x, k, temperature)
    after = S.adjust(place(full, "row", torch.float32), **on_gpu(r))
    check_top(S.top(after, k, temperature=temperature), x, k, temperature)
    z = rng.standard_normal((C, n)).astype(np.float32)
    got = S.distill(place(z, "class"), classes, values, teacher_lse=lse, temperature=temperature)
    check_distill(got, O.distill(z, classes.cpu().numpy(), values.cpu().numpy(), None, lse.cpu().numpy(), temperature))
