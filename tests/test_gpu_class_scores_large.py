"""The operators on class scores where lists, rows or classes are many, and where calls meet: other streams, one list of several lengths, rows of several
launches."""
import numpy as np
import pytest
import torch

import class_scores as D
import score_oracle as O
from test_gpu_class_scores import check_distill, check_top, on_gpu, place, rounded, same
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


def lists(rng, C, lengths):
    begin = np.zeros(len(lengths) + 1, np.int64)
    begin[1:] = np.cumsum(lengths)
    shown = (rng.random(begin[-1]) ** 2 * C).astype(np.int32)
    shown[rng.random(begin[-1]) < 0.02] = C
    return dict(shown=shown, shown_begin=begin, repetition=1.25, frequency=0.5, presence=0.125)


LENGTHS = {
    "one_long": lambda rng, n: np.where(np.arange(n) == n // 3, 700, 3),
    "one_of_256": lambda rng, n: np.where(np.arange(n) == n - 1, 256, 1),
    "one_of_255": lambda rng, n: np.where(np.arange(n) == n - 1, 255, 1),
    "many_of_90": lambda rng, n: np.full(n, 90),
    "first_rows": lambda rng, n: np.where(np.arange(n) < 20, 400, 0),
    "one_of_65536": lambda rng, n: np.where(np.arange(n) == n // 2, 65536, 2),
    "all_long": lambda rng, n: rng.integers(150, 2500, n),
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C,n", [(127, 200), (300, 193), (2049, 130), (9000, 40)])
def test_lists_of_several_lengths(C, n, order, lengths):
    """Short lists beside long ones, more entries than a tile stages, a class that a list names often; into another array and in place."""
    rng = np.random.default_rng(C + n)
    z = D.scores(rng, C, n, special=0.02)
    r = dict(D.rules(rng, C, n, shown=False), **lists(rng, C, LENGTHS[lengths](rng, n)))
    want, g = O.adjusted(z, **r), on_gpu(r)
    x = place(z, order, pad=1)
    same(S.adjust(x, **g), want)
    check_top(S.top(x, 5, **g), want, 5)
    assert S.adjust(x, out=x, **g) is x
    same(x, want)


@pytest.mark.parametrize("C,n", [(6, 300), (50, 70), (1000, 40), (40_000, 3)])
def test_distill_nans_of_all_kinds(C, n):
    """Whatever a NaN's bits are, its row is NaN and the others are not."""
    rng = np.random.default_rng(C)
    K = min(C, 20)
    z = rng.standard_normal((C, n)).astype(np.float32)
    rows = np.arange(0, n, 3)
    bits = np.array([0xffc00000, 0xffc00001, 0xffc0007f, 0xffc00080, 0xffffffff, 0x7f800001, 0xff800001, 0x7fc00000, 0x7fffffff], np.uint32)
    z.view(np.uint32)[rng.integers(0, C, len(rows)), rows] = bits[np.arange(len(rows)) % len(bits)]
    classes, t, _ = D.teacher(rng, C, n, K, short=False)
    loss, pairs = S.distill(place(z, "class"), torch.from_numpy(classes).cuda(), torch.from_numpy(t).cuda())
    odd = np.isin(np.arange(n), rows)
    assert np.array_equal(torch.isnan(loss).cpu().numpy(), odd)
    assert np.array_equal(torch.isnan(pairs).all(2).all(0).cpu().numpy(), odd)
    fine = ~odd
    check_distill((loss[torch.from_numpy(fine)], pairs[:, torch.from_numpy(fine)]), O.distill(z[:, fine], classes[fine], t[fine]))


MANY = (1 << 22) + 5  # rows of a launch, and a few


def ends(rows):
    """The rows that are looked at: at the beginning, around the first launch's end, and the last ones."""
    return np.r_[0:3, (1 << 22) - 3:rows]


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("C", [3, 40, 1600])
def test_rows_of_two_launches(C, order):
    """Sets and lists of the rows behind the first launch's are theirs, also where so few rows are left that their classes are shared out."""
    rng = np.random.default_rng(C)
    at = ends(MANY)
    z = rounded(D.scores(rng, C, len(at)), torch.bfloat16)
    x = torch.zeros((C, MANY) if order == "class" else (MANY, C), dtype=torch.bfloat16, device="cuda")
    x = x if order == "class" else x.t()
    where = torch.from_numpy(at).cuda()
    x[:, where] = torch.from_numpy(z).cuda().bfloat16()
    r = D.rules(rng, C, len(at), sets="each")
    words = r["allowed"].shape[1]
    allowed = torch.zeros(MANY, words, dtype=torch.int32, device="cuda")
    allowed[where] = torch.from_numpy(r["allowed"]).cuda()
    lengths = np.zeros(MANY, np.int64)
    lengths[at] = np.diff(r["shown_begin"])
    begin = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)])).cuda()
    g = dict(on_gpu(r), allowed=allowed, shown_begin=begin)
    want = O.adjusted(z, **r)
    k = 4
    values, classes, lse = S.top(x, k, **g)
    check_top((values[where], classes[where], lse[where]), want, k)
    rest = torch.ones(MANY, dtype=torch.bool, device="cuda")
    rest[where] = False
    assert bool((classes[rest] == -1).all()) and bool(torch.isinf(lse[rest]).all())
    same(S.adjust(x, out=x, **g)[:, where] if C > 40 else S.adjust(x, **g)[:, where], rounded(want, torch.bfloat16))


@pytest.mark.parametrize("C,K", [(3, 2), (40, 9), (2100, 5)])
def test_distill_rows_of_two_launches(C, K):
    rng = np.random.default_rng(C)
    at = ends(MANY)
    where = torch.from_numpy(at).cuda()
    z = rng.standard_normal((C, len(at))).astype(np.float32)
    c, t, _ = D.teacher(rng, C, len(at), K, short=False)
    y = rng.integers(0, C, len(at)).astype(np.float32)
    x = torch.zeros(C, MANY, device="cuda")
    x[:, where] = torch.from_numpy(z).cuda()
    classes, scores, labels = torch.zeros(MANY, K, dtype=torch.int32, device="cuda"), torch.zeros(MANY, K, device="cuda"), torch.zeros(MANY, device="cuda")
    classes[where], scores[where], labels[where] = torch.from_numpy(c).cuda(), torch.from_numpy(t).cuda(), torch.from_numpy(y).cuda()
    loss, pairs = S.distill(x, classes, scores, labels, weight=0.5, temperature=2.0, gradient=C < 100)
    check_distill((loss[where], None if pairs is None else pairs[:, where]), O.distill(z, c, t, y, None, 2.0, 0.5))
    assert bool((loss[3:(1 << 22) - 3] == loss[3]).all())


def test_top_and_distill_on_a_stream():
    """Scores that a side stream is still writing, workspaces that another stream's calls take and free meanwhile."""
    rng = np.random.default_rng(6)
    C, n, k = 40_000, 5, 9
    z = D.scores(rng, C, n)
    x = place(z, "class")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        best = S.top(late, k)
        loss = S.distill(late, best[1], best[0], teacher_lse=best[2])
    others = [S.top(torch.zeros_like(x), k) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    check_top(best, z, k)
    check_distill(loss, O.distill(z, best[1].cpu().numpy(), best[0].cpu().numpy(), None, best[2].cpu().numpy()))
    for values, classes, _ in others:
        assert torch.equal(classes, torch.arange(k, dtype=torch.int32, device="cuda").expand(n, k))


@pytest.mark.parametrize("C,n,K", [(33, 16_384, 128), (100, 20_011, 10), (120, 16_389, 7), (300, 16_385, 100), (500, 16_400, 32), (1000, 16_390, 5)])
def test_distill_many_rows(C, n, K):
    """Tiles of the shapes that many rows are cut into; rows are looked at here and there."""
    rng = np.random.default_rng(C)
    at = np.unique(np.r_[0:40, rng.integers(0, n, 150), n - 40:n])
    where = torch.from_numpy(at).cuda()
    z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
    c, t, full = D.teacher(rng, C, n, K, repeated=True)
    t = rounded(t, torch.bfloat16)
    lse = np.log(np.exp(full / 2).sum(1)).astype(np.float32) if C % 200 else None
    y = rng.integers(0, C, n).astype(np.float32)
    loss, pairs = S.distill(place(z, "class", pad=1), torch.from_numpy(c).cuda(), torch.from_numpy(t).cuda().bfloat16(), torch.from_numpy(y).cuda(),
                            None if lse is None else torch.from_numpy(lse).cuda(), 2.0, 0.5)
    want = O.distill(z[:, at], c[at], t[at], y[at], None if lse is None else lse[at], 2.0, 0.5)
    check_distill((loss[where], pairs[:, where]), want)
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(pairs).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("C", [33, 47, 100, 129, 160, 199, 203, 320, 399, 512])
def test_top_of_short_rows(C, dtype):
    """Rows of so few classes that the best ones lie in most of the threads that hold any."""
    rng = np.random.default_rng(C)
    n = 70
    z = rounded(D.scores(rng, C, n, special=0.03), dtype)
    r = D.rules(rng, C, n, sets="some")
    want = O.adjusted(z, **r)
    for order in ("row", "class"):
        x = place(z, order, dtype, pad=3, shift=1)
        for k in (8, 16, 20, 28, 29, 33, 42, 43, 50, 128):
            check_top(S.top(x, k), z, k)
            check_top(S.top(x, k, **on_gpu(r)), want, k)
