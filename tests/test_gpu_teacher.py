"""Training against a teacher's best scores, and answers under rules, through sessions and estimators."""
import os

import numpy as np
import pytest

import class_scores as D
import datasets
import score_oracle as O
import thundergbm_amd as T

pytestmark = pytest.mark.gpu


def problem(n=1500, seed=4):
    X, y = datasets.config5(n, seed=seed)
    rng = np.random.default_rng(seed)
    return X, y, rng


def session(X, y, **kw):
    val, rp, col = datasets.dense_to_csr(X)
    return T.Session(val, rp, col, y, depth=4, n_trees=4, learning_rate=0.3, objective="multi:softprob", num_class=len(np.unique(y)), **kw)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("weight", [1.0, 0.4])
def test_session_trains_on_the_teacher(rest, weight):
    X, y, rng = problem()
    C, n, K = len(np.unique(y)), len(y), 4
    classes, t, full = D.teacher(rng, C, n, K)
    lse = np.log(np.exp(full.astype(np.float64) / 2).sum(1)).astype(np.float32) if rest else None
    s = session(X, y)
    s.set_teacher(classes, t, lse, 2.0, weight)
    labels = np.searchsorted(np.unique(y), y).astype(np.float32)
    for _ in range(2):
        z = s.y_pred().reshape(C, n)
        loss, pairs, loss_room, pairs_room = O.distill(z, classes, t, labels, lse, 2.0, weight)
        assert abs(s.teacher_loss() - loss.mean()) <= loss_room.mean() + 2.0**-24 * np.abs(loss).mean()
        s.gradient()
        gh = s.gh().reshape(C, n, 2)
        assert np.all(np.abs(gh - pairs) <= pairs_room)
        s.boost(1)
    s.set_teacher(None)  # on the labels again: the pairs of a session that never had a teacher
    s.gradient()
    plain = session(X, y)
    plain.set("y_pred", s.y_pred())
    plain.gradient()
    np.testing.assert_array_equal(s.gh(), plain.gh())
    s.close()
    plain.close()


def test_teacher_follows_the_rows():
    """Rows that are re-ordered physically while boosting keep their teacher: the pairs are those of the rows' own lists."""
    X, y, rng = problem(n=3000)
    C, n = len(np.unique(y)), len(y)
    classes, t, _ = D.teacher(rng, C, n, 5)
    labels = np.searchsorted(np.unique(y), y).astype(np.float32)
    os.environ["TGBM_REORDER"] = "always"
    try:
        s = session(X, y)
        s.set_teacher(classes, t, temperature=3.0, weight=0.7)
        for _ in range(3):
            s.boost(1)
            assert s.info("reorders_done") > 0
            s.gradient()
            loss, pairs, loss_room, pairs_room = O.distill(s.y_pred().reshape(C, n), classes, t, labels, None, 3.0, 0.7)
            assert np.all(np.abs(s.gh().reshape(C, n, 2) - pairs) <= pairs_room)
            assert abs(s.teacher_loss() - loss.mean()) <= loss_room.mean() + 2.0**-24 * np.abs(loss).mean()
        s.close()
    finally:
        del os.environ["TGBM_REORDER"]


def test_many_classes_in_a_session():
    """So many classes that a row's scores go by several rows of a workgroup's tile, with sampled columns and resampled rows."""
    rng = np.random.default_rng(1)
    n, C = 900, 60
    X = rng.standard_normal((n, 6)).astype(np.float32)
    y = (rng.permutation(n) % C).astype(np.float32) * 3 + 1
    classes, t, _ = D.teacher(rng, C, n, 20)
    val, rp, col = datasets.dense_to_csr(X)
    s = T.Session(val, rp, col, y, depth=2, n_trees=2, objective="multi:softmax", num_class=C)
    s.set_teacher(classes, t.astype(np.float16), weight=1.0)
    s.gradient()
    _, pairs, _, pairs_room = O.distill(np.zeros((C, n), np.float32), classes, t.astype(np.float16))
    assert np.all(np.abs(s.gh().reshape(C, n, 2) - pairs) <= pairs_room)
    s.boost(2)
    assert np.isfinite(s.y_pred()).all()
    s.close()


def test_classifier_with_a_teacher():
    """The estimator's call is the session's; a class that only the teacher knows, NaN and no label at all are left out."""
    X, y, rng = problem()
    known = np.unique(y)
    C, n = len(known), len(y)
    classes, t, _ = D.teacher(rng, C, n, 3)
    labels = np.where((classes >= 0) & (classes < C), known[np.clip(classes, 0, C - 1)], np.nan)
    labels[::3, 1] = 1000.0
    numbers = np.where(np.isin(labels, known), classes, -1)
    clf = T.TGBMClassifier(depth=4, n_trees=4, learning_rate=0.3, objective="multi:softprob", num_class=C, verbose=0)
    clf.fit(X, y, teacher=T.Teacher(labels, t, temperature=2.0, weight=0.6))
    s = session(X, y)
    s.set_teacher(numbers, t, temperature=2.0, weight=0.6)
    s.boost(4)
    np.testing.assert_allclose(clf.class_scores(X), s.y_pred().reshape(C, n), rtol=1e-5, atol=1e-5)
    assert clf.group_label == known.tolist() and clf.num_class == C
    # without a teacher's part the trees are those of the labels
    a = T.TGBMClassifier(depth=4, n_trees=3, objective="multi:softprob", num_class=C, verbose=0).fit(X, y)
    b = T.TGBMClassifier(depth=4, n_trees=3, objective="multi:softprob", num_class=C, verbose=0).fit(X, y, teacher=T.Teacher(labels, t, weight=0.0))
    np.testing.assert_allclose(a.class_scores(X), b.class_scores(X), rtol=1e-3, atol=1e-3)
    s.close()


def test_answers_under_rules():
    X, y, rng = problem()
    known = np.unique(y)
    C, n = len(known), len(y)
    clf = T.TGBMClassifier(depth=4, n_trees=5, learning_rate=0.5, objective="multi:softprob", num_class=C, verbose=0).fit(X, y)
    raw = clf.class_scores(X)
    p = clf.predict_proba_class_major(X)
    np.testing.assert_allclose(np.exp(O.log_softmax(raw.astype(np.float64))), p, atol=2e-6)
    bias = (np.round(rng.standard_normal(C) * 16) / 16).astype(np.float32)
    allowed = rng.random((n, C)) < 0.5
    allowed[7] = False
    shown = [rng.choice(known, rng.integers(0, 5)) for _ in range(n)]
    shown[3] = np.array([known[0], known[0], 12345.0])
    for rows in (n, 1, 9):
        rules = dict(bias=bias, allowed=allowed[:rows], shown=shown[:rows], repetition=1.5, frequency=0.25, presence=0.5)
        numbers = np.concatenate([np.where(np.isin(l, known), np.searchsorted(known, np.minimum(l, known[-1])), -1) for l in shown[:rows]]).astype(np.int32)
        begin = np.concatenate([[0], np.cumsum([len(l) for l in shown[:rows]])]).astype(np.int64)
        want = O.adjusted(raw[:, :rows], bias, D.bits_of(allowed[:rows]), None, numbers, begin, 1.5, 0.25, 0.5)
        np.testing.assert_array_equal(clf.class_scores(X[:rows], **rules), want)
        labels, prob = clf.top_classes(X[:rows], k=3, temperature=2.0, **rules)
        values, classes, lse = O.top(want, 3, 2.0)
        np.testing.assert_array_equal(labels, np.where(classes >= 0, known[np.maximum(classes, 0)], np.nan))
        with np.errstate(all="ignore"):
            np.testing.assert_allclose(prob, np.where(classes >= 0, np.exp(values / 2.0 - lse[:, None]), 0), rtol=1e-5)
    one = clf.top_classes(X, k=1)[0][:, 0]
    np.testing.assert_array_equal(one, known[raw.argmax(0)])
    np.testing.assert_array_equal(clf.top_classes(X, k=1, allowed=np.arange(C) == 2)[0][:, 0], np.full(n, known[2]))


def test_refusals_of_the_estimator():
    X, y, rng = problem(n=300)
    C, n = len(np.unique(y)), len(y)
    clf = T.TGBMClassifier(depth=2, n_trees=2, objective="multi:softprob", num_class=C, verbose=0)
    ids, t = np.zeros((n, 2)), np.zeros((n, 2), np.float32)
    with pytest.raises(ValueError, match="train the model"):
        clf.top_classes(X)
    for bad, msg in ((T.Teacher(ids[:-1], t[:-1]), "rows"), (T.Teacher(ids, t[:, :1]), "rows"), (T.Teacher(ids, t * np.nan), "NaN"),
                     (T.Teacher(ids, t, temperature=0), "temperature"), (T.Teacher(ids, t, weight=2), "weight"), (T.Teacher(ids, t, lse=np.zeros(3)), "lse"),
                     (T.Teacher(np.zeros((n, 129)), np.zeros((n, 129))), "128")):
        with pytest.raises(ValueError, match=msg):
            clf.fit(X, y, teacher=bad)
    with pytest.raises(ValueError, match="objective"):
        T.TGBMRegressor(verbose=0).fit(X, y, teacher=T.Teacher(ids, t))
    clf.fit(X, y)
    for kw, msg in ((dict(bias=np.zeros(C + 1)), "bias"), (dict(allowed=np.ones((n - 1, C))), "allowed"), (dict(shown=[[1.0]]), "shown"),
                    (dict(shown=[[]] * n, repetition=0), "repetition"), (dict(k=0), "k is 0"), (dict(k=129), "k is 129"), (dict(temperature=0), "temperature")):
        with pytest.raises(ValueError, match=msg):
            clf.top_classes(X, **kw)


def test_session_refuses():
    """What would end the process is said before the library sees it."""
    X, y, rng = problem(n=300)
    s = session(X, y)
    with pytest.raises(ValueError, match="no teacher"):
        s.teacher_loss()
    with pytest.raises(ValueError, match="rows"):
        s.set_teacher(np.zeros((299, 2)), np.zeros((299, 2)))
    s.set_teacher(np.zeros((300, 2)), np.zeros((300, 2)))
    assert np.isfinite(s.teacher_loss())
    s.set_teacher(None)
    with pytest.raises(ValueError, match="no teacher"):
        s.teacher_loss()
    s.close()
    val, rp, col = datasets.dense_to_csr(X)
    s = T.Session(val, rp, col, y, depth=2, n_trees=1, objective="reg:linear")
    with pytest.raises(ValueError, match="objective"):
        s.set_teacher(np.zeros((300, 2)), np.zeros((300, 2)))
    s.close()
