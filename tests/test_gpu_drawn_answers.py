"""The estimator's drawn answers, and a linear layer as its teacher."""
import numpy as np
import pytest
import torch

import class_scores as D
import draw_oracle as R
import score_oracle as O
import thundergbm_amd as T
from test_gpu_teacher import problem
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    X, y, rng = problem()
    known = np.unique(y)
    clf = T.TGBMClassifier(depth=4, n_trees=5, learning_rate=0.5, objective="multi:softprob", num_class=len(known), verbose=0).fit(X, y)
    return clf, X, y, known


def test_drawn_answers(model):
    clf, X, y, known = model
    rng = np.random.default_rng(4)
    C, n = len(known), len(y)
    raw = clf.class_scores(X)
    u = rng.random(n).astype(np.float32)
    bias = (np.round(rng.standard_normal(C) * 16) / 16).astype(np.float32)
    allowed = rng.random((n, C)) < 0.5
    allowed[7] = False
    shown = [rng.choice(known, rng.integers(0, 5)) for _ in range(n)]
    for rows in (n, 1, 9):
        numbers = np.concatenate([np.searchsorted(known, l) for l in shown[:rows]]).astype(np.int32)
        begin = np.concatenate([[0], np.cumsum([len(l) for l in shown[:rows]])]).astype(np.int64)
        rules = dict(bias=bias, allowed=allowed[:rows], shown=shown[:rows], repetition=1.5, frequency=0.25, presence=0.5)
        x = O.adjusted(raw[:, :rows], bias, D.bits_of(allowed[:rows]), None, numbers if len(numbers) else None, begin if len(numbers) else None, 1.5, 0.25, 0.5)
        each = dict(temperature=rng.choice([0.0, 0.5, 1.0], rows).astype(np.float32), k=rng.integers(0, 4, rows).astype(np.int32), p=rng.choice([1.0, 0.7], rows).astype(np.float32))
        for how in (dict(), dict(k=2, temperature=0.7), dict(k=1 << 40), dict(p=0.8), dict(min_p=0.3), dict(temperature=0), each):
            labels, prob = clf.sample_classes(X[:rows], u[:rows], **rules, **how)
            classes, logp = R.sample(x, u[:rows], **how)
            np.testing.assert_array_equal(labels, np.where(classes >= 0, known[np.maximum(classes, 0)], np.nan))
            # (logp in 32 bits, its exponential: 2^-24 of |logp| and two roundings)
            np.testing.assert_allclose(prob, np.exp(logp), rtol=2.0**-24 * (3 + np.abs(logp[np.isfinite(logp)]).max(initial=0)))
    np.testing.assert_array_equal(clf.sample_classes(X, np.zeros(n))[0], known[raw.argmax(0)])


def test_refusals_of_drawn_answers(model):
    clf, X, y, known = model
    u = np.zeros(len(y))
    for kw, msg in ((dict(k=-1), "k is -1"), (dict(p=0), "p is 0"), (dict(min_p=2), "min_p is 2"), (dict(temperature=-1), "temperature is -1"), (dict(u=u[:5]), "u: "),
                    (dict(p=u[:5]), "p: "), (dict(k=np.zeros((2, 2))), "k: "), (dict(allowed=np.ones(2)), "allowed")):
        with pytest.raises(ValueError, match=msg):
            clf.sample_classes(X, **{"u": u, **kw})
    with pytest.raises(ValueError, match="train the model"):
        T.TGBMClassifier(objective="multi:softprob", verbose=0).sample_classes(X, u)


@pytest.mark.parametrize("n,F,C,k", [(1, 5, 3, 2), (500, 30, 9, 4), (3000, 129, 300, 128), (2000, 64, 40_000, 10)])
def test_linear_teacher(n, F, C, k):
    """The lists are those of the operators on the GPU, slice by slice; the scores are the layer's within what 8 bits leave."""
    rng = np.random.default_rng(n + C)
    x, w = rng.standard_normal((n, F)).astype(np.float32), rng.standard_normal((C, F)).astype(np.float32)
    bias, labels = rng.standard_normal(C).astype(np.float32), rng.permutation(C).astype(np.float32) * 2
    teacher = T.Teacher.linear(x, w, labels, bias=bias, k=k, temperature=2.0, weight=0.5)
    q, scale = S.quantise(torch.from_numpy(w).cuda())
    z = S.linear(torch.from_numpy(x).cuda(), q, scale, bias=torch.from_numpy(bias).cuda())
    values, classes, lse = (a.cpu().numpy() for a in S.top(z, min(k, C), temperature=2.0))
    np.testing.assert_array_equal(teacher.scores, values)
    np.testing.assert_array_equal(teacher.labels, labels[classes])
    np.testing.assert_allclose(teacher.lse, lse, rtol=1e-5, atol=1e-5)
    assert (teacher.temperature, teacher.weight) == (2.0, 0.5)
    # every number is off by half a step of its row at most, a product by that of either
    sx, sw = np.abs(x).max(1) / 127, np.abs(w).max(1) / 127
    true = np.take_along_axis(x.astype(np.float64) @ w.T + bias, classes, 1)
    room = 0.5 * (sx[:, None] * np.abs(w).sum(1)[classes] + sw[classes] * np.abs(x).sum(1)[:, None]) + 0.25 * F * sx[:, None] * sw[classes]
    assert np.all(np.abs(values - true) <= 1.001 * room + 1e-4)


def test_fit_with_a_linear_teacher():
    X, y, rng = problem()
    known = np.unique(y)
    w = rng.standard_normal((len(known), X.shape[1])).astype(np.float32)
    teacher = T.Teacher.linear(X, w, known, k=3, weight=0.5)
    clf = T.TGBMClassifier(depth=3, n_trees=2, objective="multi:softprob", num_class=len(known), verbose=0).fit(X, y, teacher=teacher)
    assert np.isfinite(clf.class_scores(X)).all()


def test_refusals_of_linear_teachers():
    x, w, labels = np.zeros((4, 5)), np.zeros((3, 5)), np.arange(3)
    for args, msg in ((dict(x=x[0]), "x: "), (dict(weights=w[:, :4]), "x: "), (dict(labels=labels[:2]), "labels"), (dict(bias=np.zeros(2)), "bias"), (dict(x=x * np.nan), "x: a number"),
                      (dict(weights=w + np.inf), "weights: a number"), (dict(bias=np.full(3, np.nan)), "bias: a number"), (dict(k=0), "k is 0"), (dict(k=129), "k is 129"),
                      (dict(temperature=0), "temperature"), (dict(x=x[:, :0], weights=w[:, :0]), "x: ")):
        with pytest.raises(ValueError, match=msg):
            T.Teacher.linear(**{**dict(x=x, weights=w, labels=labels), **args})
    empty = T.Teacher.linear(np.zeros((0, 5)), w, labels, k=2)
    assert empty.labels.shape == (0, 2)
