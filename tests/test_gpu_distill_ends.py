"""The loss against a teacher where its masses do not come to one, where they are tiny, and where scores are large (teacher_oracle.py)."""
import numpy as np
import pytest
import torch

import class_scores as D
import teacher_oracle as N
from test_gpu_class_scores import DISTILL_SIZES, TYPES, check_distill, place, rounded
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


def on_gpu(x, dtype=None):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dtype)


def check(z, classes, t, labels=None, lse=None, temperature=1.0, weight=1.0, dtype=torch.float32, **layout):
    """With pairs and the loss alone, against the restatement; the call's results."""
    want = N.distill(z, classes, t, labels, lse, temperature, weight)
    x = place(z, "class", **layout)
    args = (x, on_gpu(classes), on_gpu(t, dtype), on_gpu(labels), on_gpu(lse), temperature, weight)
    got = S.distill(*args)
    check_distill(got, want)
    check_distill(S.distill(*args, gradient=False), want)
    return got, want


@pytest.mark.parametrize("C,n,K", DISTILL_SIZES)
def test_teacher_s_rest(C, n, K):
    """The inputs of test_distill with the rest, lists rounded to 16 bits among them: those may have a little more than one together, or less with no class left."""
    rng = np.random.default_rng(C + n + K)
    for j, dtype in enumerate(TYPES):
        temperature, weight = ((1.0, 1.0), (2.0, 0.5), (0.7, 0.25))[j]
        z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
        classes, t, full = D.teacher(rng, C, n, K, repeated=j == 1)
        t = rounded(t, dtype)
        lse = np.log(np.exp(full.astype(np.float64) / temperature).sum(1)).astype(np.float32)
        labels = rng.integers(0, C, n).astype(np.float32)
        labels[::5] = np.array([-1, C, 0.5, np.nan, np.inf], np.float32)[np.arange(len(labels[::5])) % 5]
        check(z, classes, t, labels, lse, temperature, weight, dtype, pad=j, shift=j)


@pytest.mark.parametrize("C,n,K", [(1, 9, 1), (6, 70, 6), (15, 40, 20), (31, 40, 31), (40, 50, 40), (128, 21, 128), (128, 16_400, 128)])
def test_every_class_named_and_some_left_over(C, n, K):
    """A teacher of more classes than the student has: what it left to the others has nowhere to go."""
    rng = np.random.default_rng(C)
    z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
    classes, t, full = D.teacher(rng, C, n, K, short=False)
    lse = (np.log(np.exp(full.astype(np.float64) / 2).sum(1)) + rng.choice([0.0, 0.05, 0.5, 3.0], n)).astype(np.float32)
    y = rng.integers(0, C, n).astype(np.float32)
    for weight in (1.0, 0.4):
        if n < 1000:
            (loss, pairs), want = check(z, classes, t, y, lse, 2.0, weight)
        else:
            at = np.r_[0:30, n - 30:n]
            want = N.distill(z[:, at], classes[at], t[at], y[at], lse[at], 2.0, weight)
            got = S.distill(place(z, "class"), on_gpu(classes), on_gpu(t), on_gpu(y), on_gpu(lse), 2.0, weight)
            check_distill((got[0][on_gpu(at)], got[1][:, on_gpu(at)]), want)


@pytest.mark.parametrize("C,n,K", [(6, 40, 3), (32, 30, 7), (100, 25, 10), (700, 17, 40), (5000, 4, 20), (40_000, 3, 9)])
@pytest.mark.parametrize("form", ["others_out", "more_than_one"])
def test_masses_that_do_not_come_to_one(C, n, K, form):
    """The student rules every class out that is not named; a log-sum-exp that is too low for the entries."""
    rng = np.random.default_rng(C)
    z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
    classes, t, full = D.teacher(rng, C, n, K, short=False, repeated=True)
    lse = np.log(np.exp(full.astype(np.float64) / 2).sum(1)).astype(np.float32)
    if form == "others_out":
        for i in range(n):
            z[np.setdiff1d(np.arange(C), classes[i]), i] = -np.inf
        y = classes[:, 0].astype(np.float32)
    else:
        lse = (np.log(np.exp(np.take_along_axis(full, classes, 1).astype(np.float64) / 2).sum(1)) - rng.choice([1e-4, 0.1, 2.0], n)).astype(np.float32)
        y = rng.integers(0, C, n).astype(np.float32)
    check(z, classes, t, y, lse, 2.0, 0.7)


@pytest.mark.parametrize("rest", [False, True])
def test_lists_with_infinities_beside_them(rest):
    """The rows of test_distill_far_scores, whose log-sum-exp leaves a quarter over, with every class named and with others."""
    for C in (5, 2000, 40_000):
        rng = np.random.default_rng(C)
        n, K = 6, 5
        z = rng.standard_normal((C, n)).astype(np.float32)
        classes = np.tile(np.arange(K, dtype=np.int32), (n, 1))
        t = rng.standard_normal((n, K)).astype(np.float32)
        lse = (np.log(np.exp(t.astype(np.float64)).sum(1)) + 0.3).astype(np.float32) if rest else None
        z[K:, 0] -= 500
        z[:K, 1] -= 500
        z[:, 2] *= 100
        z[K - 1, 3] = -np.inf
        z[:, 4] = -np.inf
        check(z, classes, t, None, lse)


def test_many_rows_with_every_class_named():
    """The inputs of test_distill_many_rows whose lists name every class."""
    C, n, K = 33, 16_384, 128
    rng = np.random.default_rng(C)
    at = np.unique(np.r_[0:40, rng.integers(0, n, 150), n - 40:n])
    z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
    c, t, full = D.teacher(rng, C, n, K, repeated=True)
    t = rounded(t, torch.bfloat16)
    lse = np.log(np.exp(full / 2).sum(1)).astype(np.float32)
    y = rng.integers(0, C, n).astype(np.float32)
    loss, pairs = S.distill(place(z, "class", pad=1), on_gpu(c), on_gpu(t, torch.bfloat16), on_gpu(y), on_gpu(lse), 2.0, 0.5)
    check_distill((loss[on_gpu(at)], pairs[:, on_gpu(at)]), N.distill(z[:, at], c[at], t[at], y[at], lse[at], 2.0, 0.5))


def test_session_whose_teacher_knows_more_classes():
    """A session's gradients add up to nothing also where what the teacher left to classes of its own has nowhere to go."""
    import datasets
    import thundergbm_amd as T
    X, y = datasets.config5(900, seed=4)
    known = np.unique(y)
    C, n, rng = len(known), len(y), np.random.default_rng(4)
    classes, t, full = D.teacher(rng, 2 * C, n, 2 * C, short=False)
    lse = np.log(np.exp(full.astype(np.float64) / 2).sum(1)).astype(np.float32)
    val, rp, col = datasets.dense_to_csr(X)
    s = T.Session(val, rp, col, y, depth=4, n_trees=3, learning_rate=0.3, objective="multi:softprob", num_class=C)
    s.set_teacher(classes, t, lse, 2.0, 0.8)
    for _ in range(2):
        s.gradient()
        loss, pairs, loss_room, pairs_room = N.distill(s.y_pred().reshape(C, n), classes, t, np.searchsorted(known, y).astype(np.float32), lse, 2.0, 0.8)
        assert np.all(np.abs(s.gh().reshape(C, n, 2) - pairs) <= pairs_room)
        assert abs(s.teacher_loss() - loss.mean()) <= loss_room.mean() + 2.0**-24 * np.abs(loss).mean()
        s.boost(1)
    s.close()


@pytest.mark.parametrize("rest", [0.0, 1.0, 40.0, None])
@pytest.mark.parametrize("C", [8, 16, 32, 60, 3000])
def test_masses_that_32_bits_hardly_hold(C, rest):
    """Entries so far below the best one that their q is less than the least normal number, or none: they add nothing to the loss. rest: what the
    log-sum-exp lies above the entries' own."""
    rng = np.random.default_rng(C)
    T, n, K = 0.1, 300, min(C, 8)
    z = rng.standard_normal((C, n)).astype(np.float32)
    classes = np.argsort(rng.random((n, C)), axis=1)[:, :K].astype(np.int32)
    t = np.zeros((n, K), np.float32)
    t[:, 2:] = -T * rng.uniform(40 if rest else 80, 90, (n, K - 2))
    t += rng.standard_normal((n, 1)).astype(np.float32)
    lse = None if rest is None else (np.log(np.exp(t.astype(np.float64) / np.float32(T)).sum(1)) + rest).astype(np.float32)
    got, want = check(z, classes, t, None, lse, T)
    assert np.isfinite(want[0]).all() and bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("offset", [1000.0, -1000.0, 20_000.0])
@pytest.mark.parametrize("T", [1e-3, 0.01, 1.0])
@pytest.mark.parametrize("C,n,K", [(8, 60, 5), (40, 50, 12), (300, 30, 128), (500, 16_400, 3), (5000, 4, 60), (40_000, 3, 20)])
def test_what_a_teacher_s_scores_have_in_common(C, n, K, T, offset):
    """falls out: without a log-sum-exp the q of a row add up to one, and so the gradient to nothing, however large the scores are."""
    rng = np.random.default_rng(C + K)
    z = rng.standard_normal((C, n)).astype(np.float32) * np.float32(min(T, 1) * 2)
    classes, t, _ = D.teacher(rng, C, n, K, short=False)
    # (steps that the offset leaves whole, few enough of them that several entries count)
    t = np.round(t * T * 512) / 512 if T * 512 > 1 else np.round(t / 2) / 512
    t = (t + offset).astype(np.float32)
    if n < 1000:
        (_, pairs), _ = check(z, classes, t, None, None, T)
    else:
        at = np.r_[0:30, n - 30:n]
        got = S.distill(place(z, "class"), on_gpu(classes), on_gpu(t), temperature=T)
        check_distill((got[0][on_gpu(at)], got[1][:, on_gpu(at)]), N.distill(z[:, at], classes[at], t[at], temperature=T))
        pairs = got[1]
    # every p and q is off by at most (4 x + 14 + 4 X + 136 + K + 16) half steps of itself, x of what has a part being a few on average: 600 for all that a row holds
    assert bool((pairs[..., 0].double().sum(0).abs() <= T * 600 * 2.0**-24).all())


@pytest.mark.parametrize("T", [1e-3, 0.05, 30.0, 1e3])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("C,n,K", [(3, 50, 2), (8, 60, 5), (16, 40, 16), (32, 40, 7), (60, 50, 12), (300, 30, 128), (2500, 5, 30), (40_000, 3, 20)])
def test_ends_of_the_temperatures(C, n, K, rest, T):
    """Scores as far apart as the temperature makes them count, and scores of trees."""
    rng = np.random.default_rng(C + K)
    for spread in (min(T, 3.0), 3.0):
        z = (rng.standard_normal((C, n)) * spread).astype(np.float32)
        classes, t, full = D.teacher(rng, C, n, K, short=spread == 3.0)
        t, full = (t * np.float32(spread / 2.5), full * np.float32(spread / 2.5))
        f = full.astype(np.float64) / np.float32(T)
        lse = (f.max(1) + np.log(np.exp(f - f.max(1, keepdims=True)).sum(1))).astype(np.float32) if rest else None
        y = rng.integers(0, C, n).astype(np.float32)
        got, _ = check(z, classes, t, y, lse, T, 0.6)
        assert bool(torch.isfinite(got[0]).all())
