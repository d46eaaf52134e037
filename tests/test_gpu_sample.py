"""Drawn classes against their restatement (draw_oracle.py).

Classes have to be equal. The sums that decide which one it is are 64 bits on both sides: off by about the number of classes times 2^-52 of the whole, so that a
given random number lies between two answers with odds below 1e-9 a row, but for the ends that are tested by themselves with scores whose
sums are whole numbers. logp is rounded once to 32 bits; in front of that its argument is off by 1e-11 at most."""
import numpy as np
import pytest
import torch

import class_scores as D
import draw_oracle as R
import score_oracle as O
from test_gpu_class_scores import on_gpu, place, rounded
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# (sizes of every way that a call can go: a thread to a row, workgroups of one kind and another, parts of a row)
SIZES = [(1, 1), (2, 70), (8, 700), (9, 65), (16, 64), (17, 300), (32, 257), (33, 64), (65, 130), (300, 40), (1000, 33), (1025, 9), (4099, 5), (8192, 3), (8193, 3), (24_600, 2),
         (70_001, 2), (131_072, 1), (262_147, 1)]


def check(got, want, rows=None):
    classes, logp = (x.cpu().numpy() for x in got)
    if rows is not None:
        classes, logp = classes[rows], logp[rows]
    np.testing.assert_array_equal(classes, want[0])
    assert np.array_equal(np.isfinite(logp), np.isfinite(want[1])) and np.array_equal(np.isnan(logp), np.isnan(want[1]))
    f = np.isfinite(want[1])
    np.testing.assert_allclose(logp[f], want[1][f], rtol=2.0**-24 * 1.01, atol=1e-11)


def numbers(rng, n):
    u = rng.random(n).astype(np.float32)
    u[rng.random(n) < 0.05] = 0
    u[rng.random(n) < 0.05] = R.LARGEST_BELOW_ONE
    return u


SETTINGS = [dict(), dict(k=1), dict(k=7, p=0.9), dict(k=100, min_p=0.05), dict(k=300, p=0.8, temperature=0.7), dict(p=0.95), dict(p=0.5, temperature=2.0), dict(min_p=0.1),
            dict(min_p=1.0), dict(temperature=0.0), dict(k=128, p=0.3, min_p=0.01, temperature=1.5), dict(k=1 << 30, p=0.999)]


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", SIZES)
def test_sample(C, n, order):
    rng = np.random.default_rng(C * 5 + n)
    u = numbers(rng, n)
    for j, how in enumerate(SETTINGS):
        dtype = TYPES[j % 3] if order == "row" else torch.float32
        z = rounded(rng.standard_normal((C, n)).astype(np.float32) * rng.choice([0.3, 3.0, 10.0]), dtype)
        got = S.sample(place(z, order, dtype, pad=j % 4, shift=j % 3), torch.from_numpy(u).cuda(), **how)
        check(got, R.sample(z, u, **how))


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", [(7, 300), (32, 200), (40, 130), (300, 80), (1000, 50), (9000, 6), (40_000, 3)])
def test_rules(C, n, order):
    """Biases, sets of allowed classes (with rows that nothing is left of), lists of shown classes, odd scores."""
    rng = np.random.default_rng(C + n)
    u = numbers(rng, n)
    for j, (dtype, sets) in enumerate(zip(TYPES, ("some", "each", "one"))):
        for how in (dict(), dict(k=20, p=0.9), dict(p=0.7, temperature=1.3), dict(k=200, min_p=0.02)):
            z = rounded(D.scores(rng, C, n, special=0.02 if C < 100 else 0.001), dtype)
            r = D.rules(rng, C, n, sets=sets, shown=j != 1 or C < 100, longest=(9, 40, 300)[j])
            got = S.sample(place(z, order, dtype, pad=j), torch.from_numpy(u).cuda(), **on_gpu(r), **how)
            check(got, R.sample(O.adjusted(z, **r), u, **how))


def test_settings_of_each_row():
    rng = np.random.default_rng(3)
    for C, n in ((6, 900), (30, 700), (100, 500), (3000, 60), (20_000, 40)):
        z = rng.standard_normal((C, n)).astype(np.float32) * 2
        u = numbers(rng, n)
        f = lambda *v: np.array(v, np.float32)[rng.integers(0, len(v), n)]
        how = dict(temperature=f(0, 1e-7, -1, 0.3, 1, 1, 2, 1e7, np.inf, np.nan), p=f(1, 1, 1.5, 0.9, 0.5, 0.01, 0, -2, np.nan), min_p=f(0, 0, 0.1, 0.9, 1, 7, -3, np.nan),
                   k=np.array([0, -4, 1, 3, 50, 129, 1 << 30], np.int32)[rng.integers(0, 7, n)])
        u[::11] = f(np.nan, -1, 1, 5, np.inf)[::11]
        for order in ("class", "row"):
            for names in (("temperature",), ("p", "k"), ("min_p",), tuple(how)):
                some = {name: how[name] for name in names}
                got = S.sample(place(z, order), torch.from_numpy(u).cuda(), **{k: torch.from_numpy(v).cuda() for k, v in some.items()})
                check(got, R.sample(z, u, **some))


@pytest.mark.parametrize("C", [8, 31, 64, 1000, 8200, 70_001])
@pytest.mark.parametrize("T", [1e-6, 1e-3, 1.0, 1e3, 1e6])
def test_equal_and_nearly_equal_scores(C, T):
    """Many classes that have the same probability or nearly: rows of one value, of two, of one at a time larger by a step, of neighbours on the number line, of the
    lowest number, of infinities."""
    rng = np.random.default_rng(C)
    rows = [np.full(C, v, np.float32) for v in (0.0, -7.25, 3e38, -3.4028235e38, np.inf)]
    rows.append(rng.choice(np.array([1.0, 1.5], np.float32), C))
    rows.append(np.where(np.arange(C) == C // 3, np.float32(np.inf), np.float32(1)))
    rows.append(np.where(rng.random(C) < 0.3, np.float32(np.inf), np.float32(np.nan)))
    rows.append((np.float32(5) + np.arange(C, dtype=np.float32) * np.float32(2.0**-21))[rng.permutation(C)])
    rows.append(np.where(rng.random(C) < 0.5, np.float32(-3.4028235e38), np.round(rng.standard_normal(C).astype(np.float32))))
    rows.append(np.where(rng.random(C) < 0.5, np.float32(0.0), np.float32(-0.0)))
    z = np.stack(rows, 1)
    for how in (dict(), dict(p=0.5), dict(k=C // 2 + 1, p=0.75), dict(k=5), dict(min_p=0.5), dict(k=C // 2 + 130)):
        for v in (0.0, 0.25, 0.5, 0.6180339, R.LARGEST_BELOW_ONE):
            u = np.full(z.shape[1], v, np.float32)
            for order in ("class", "row"):
                check(S.sample(place(z, order), torch.from_numpy(u).cuda(), temperature=T, **how), R.sample(z, u, temperature=T, **how))


@pytest.mark.parametrize("C", [4, 64, 256, 16_384])
def test_random_numbers_at_the_borders(C):
    """Equal scores have borders at whole parts of one: a random number on a border is the next class's."""
    n = min(C, 64)
    u = (np.arange(n) * (C // n) / C).astype(np.float32)
    z = np.zeros((C, n), np.float32)
    for order in ("class", "row"):
        classes, logp = S.sample(place(z, order), torch.from_numpy(u).cuda())
        np.testing.assert_array_equal(classes.cpu().numpy(), np.arange(n) * (C // n))
        np.testing.assert_allclose(logp.cpu().numpy(), -np.log(C), rtol=2.0**-24 * 1.01)
        # the fewest that have half of the mass are half of them
        classes, _ = S.sample(place(z, order), torch.full((n,), R.LARGEST_BELOW_ONE, device="cuda"), p=0.5)
        assert bool((classes == C // 2 - 1).all())


def test_shares_of_many_draws():
    """A row's classes come as often as their probabilities say (each within five standard deviations of 200 000 draws)."""
    C, n = 50, 200_000
    z = np.random.default_rng(2).standard_normal(C).astype(np.float32) * 2
    u = torch.rand(n, generator=torch.Generator().manual_seed(3)).cuda()
    for order in ("class", "row"):
        x = torch.from_numpy(z).cuda()[:, None].expand(C, n)
        x = x.contiguous() if order == "class" else x.t().contiguous().t()
        classes, logp = S.sample(x, u, temperature=1.3)
        prob = torch.softmax(torch.from_numpy(z).double() / float(np.float32(1.3)), 0).numpy()
        share = np.bincount(classes.cpu().numpy(), minlength=C) / n
        assert np.all(np.abs(share - prob) <= 5 * np.sqrt(prob * (1 - prob) / n) + 1 / n)
        np.testing.assert_allclose(logp.cpu().numpy(), np.log(prob)[classes.cpu().numpy()], rtol=2.0**-24 * 1.01, atol=1e-11)


def test_many_rows():
    """More rows than one launch or one part of the workspace takes."""
    for C, n, how in ((3, 4_200_000, dict()), (40, 1_300_000, dict(p=0.9)), (5000, 9000, dict(p=0.9))):
        rng = np.random.default_rng(C)
        x = torch.randn(C, n, device="cuda", generator=torch.Generator("cuda").manual_seed(C))
        u = torch.rand(n, device="cuda", generator=torch.Generator("cuda").manual_seed(C + 1))
        rows = np.r_[0:20, n // 2:n // 2 + 20, n - 20:n, rng.integers(0, n, 40)]
        at = torch.from_numpy(rows).cuda()
        check(S.sample(x, u, **how), R.sample(x[:, at].cpu().numpy(), u[at].cpu().numpy(), **how), rows)


@pytest.mark.parametrize("C,n", [(16_384, 128), (16_390, 129), (50_001, 17), (140_000, 64), (600_000, 3)])
def test_few_long_rows(C, n):
    """Rows that go by parts, some of which end the parts' way: equal scores, infinities, nothing allowed, temperatures of 0, numbers that are NaN."""
    rng = np.random.default_rng(C)
    z = rounded(rng.standard_normal((C, n)).astype(np.float32) * rng.choice([0.5, 2.5, 8.0], n).astype(np.float32), torch.bfloat16)
    z[:, ::5] = rng.standard_normal(z[:, ::5].shape[1]).astype(np.float32)  # all of a row's scores are equal
    z[C // 2, 1::7] = np.inf
    z[:, 2] = -np.inf
    z = rounded(z, torch.bfloat16)
    u = numbers(rng, n)
    f = lambda *v: np.array(v, np.float32)[rng.integers(0, len(v), n)]
    each = dict(temperature=f(0, 0.5, 1, 1, 3, 1e6, np.nan), p=f(1, 0.9, 0.3, 0.999, 0, np.nan), min_p=f(0, 0, 0.1, 1))
    counts = dict(k=np.array([0, 1, 3, 50, 700, 9000, C - 1, C, C + 1], np.int32)[rng.integers(0, 9, n)])
    r = D.rules(rng, C, n, sets="some", shown=n < 20)
    for how in (dict(), dict(p=0.9), dict(p=0.5, min_p=0.01), dict(min_p=0.2, temperature=2.0), each, counts, {**counts, **each}, dict(k=500), dict(k=300, p=0.7), dict(k=5000, min_p=0.001, p=0.99)):
        some = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in how.items()}
        check(S.sample(place(z, "row", torch.bfloat16, pad=3), torch.from_numpy(u).cuda(), **some), R.sample(z, u, **how))
    check(S.sample(place(z, "row", torch.bfloat16), torch.from_numpy(u).cuda(), p=0.8, **on_gpu(r)), R.sample(O.adjusted(z, **r), u, p=0.8))
    check(S.sample(place(z, "class"), torch.from_numpy(u).cuda(), p=0.95), R.sample(z, u, p=0.95))


def test_far_apart_rows_and_long_lists():
    """Rows whose places pass 32 bits, long lists of shown classes, one class many times."""
    rng = np.random.default_rng(9)
    C, n, pitch = 9000, 3, 1_500_000_000
    memory = torch.empty(2 * pitch + C, dtype=torch.bfloat16, device="cuda")
    x = memory.as_strided((n, C), (pitch, 1))
    z = rounded(rng.standard_normal((C, n)).astype(np.float32) * 2, torch.bfloat16)
    x.copy_(torch.from_numpy(z).t())
    u = numbers(rng, n)
    lists = [rng.integers(0, C, 20_000), np.full(70_000, 7), rng.integers(0, C, 3)]
    r = dict(shown=np.concatenate(lists).astype(np.int32), shown_begin=np.cumsum([0] + [len(l) for l in lists]).astype(np.int64), repetition=1.1, frequency=1e-3, presence=0.2)
    for how in (dict(p=0.9), dict(k=500), dict(k=40, p=0.8)):
        check(S.sample(x.t(), torch.from_numpy(u).cuda(), **on_gpu(r), **how), R.sample(O.adjusted(z, **r), u, **how))
        check(S.sample(x.t(), torch.from_numpy(u).cuda(), **how), R.sample(z, u, **how))


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", [(20, 20_000), (20, 300), (100, 17_000), (100, 16_384), (128, 50), (129, 257)])
def test_ways_of_few_classes(C, n, order):
    """Few classes with long and short lists of shown ones, many and few rows, counts that cut: each goes another way and wants another workspace."""
    rng = np.random.default_rng(C + n)
    z, u = rng.standard_normal((C, n)).astype(np.float32) * 2, numbers(rng, n)
    rows = np.r_[0:20, n // 2:n // 2 + 10, n - 20:n]
    at = torch.from_numpy(rows).cuda()
    for longest in (0, 10, 120):
        r = D.rules(rng, C, n, sets="some", shown=longest > 0, longest=longest)
        x = O.adjusted(z, **r)[:, rows]
        for how in (dict(k=5), dict(k=15, p=0.8), dict(k=40), dict(p=0.6)):
            got = S.sample(place(z, order), torch.from_numpy(u).cuda(), **on_gpu(r), **how)
            check([v[at] for v in got], R.sample(x, u[rows], **how))


def test_streams_graphs_and_repeats():
    rng = np.random.default_rng(8)
    for C, n, how in ((8, 500, dict()), (700, 200, dict(k=30, p=0.9)), (700, 200, dict(p=0.9)), (20_000, 9, dict(k=300)), (20_000, 9, dict(p=0.8))):
        z, u = rng.standard_normal((C, n)).astype(np.float32) * 2, numbers(rng, n)
        r = D.rules(rng, C, n, sets="each")
        want = R.sample(O.adjusted(z, **r), u, **how)
        x, v, g = place(z, "class"), torch.from_numpy(u).cuda(), on_gpu(r)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            first = S.sample(x, v, **g, **how)
        side.synchronize()
        check(first, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = S.sample(x, v, **g, **how)
        for k in range(3):
            out[0].fill_(-7)
            out[1].fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, first):
                assert torch.equal(a, b)
            assert all(torch.equal(a, b) for a, b in zip(S.sample(x, v, **g, **how), first))


def test_no_rows():
    classes, logp = S.sample(torch.zeros(5, 0, device="cuda"), torch.zeros(0, device="cuda"))
    assert classes.shape == (0,) and logp.shape == (0,) and classes.dtype == torch.int32


def test_refusals():
    x, u = torch.zeros(40, 6, device="cuda"), torch.zeros(6, device="cuda")
    for args in (dict(k=-1), dict(k=2.5), dict(p=0), dict(p=2), dict(min_p=-1), dict(temperature=-1), dict(temperature=float("nan")), dict(k=torch.zeros(6, device="cuda")),
                 dict(p=torch.zeros(5, device="cuda")), dict(p=torch.zeros(6)), dict(temperature=torch.zeros(6, device="cuda", dtype=torch.float64)),
                 dict(min_p=torch.zeros(12, device="cuda")[::2]), dict(allowed_set=torch.zeros(6, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            S.sample(x, u, **args)
    for bad in (u.double(), u[:5], torch.zeros(6), torch.zeros(12, device="cuda")[::2], u.clone().requires_grad_(), None):
        with pytest.raises(ValueError):
            S.sample(x, bad)
    for bad in (x.double(), x[0], x.clone().requires_grad_(), torch.zeros(40, 12, device="cuda")[:, ::2]):
        with pytest.raises(ValueError):
            S.sample(bad, u)
