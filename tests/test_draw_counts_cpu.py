"""Counts of each row of `sample_classes`: what reaches the library for arrays of every type, on a library that a fake stands in for."""
import ctypes as C

import numpy as np
import pytest

import thundergbm_amd as T
from thundergbm_amd import estimator as E
from thundergbm_amd.scores import _Sampling

N, CLASSES = 4, 5


class Library:
    """Keeps the counts that a call brings and draws the first class."""

    def tgbm_predict_sample(self, n, val, row_ptr, col, model, n_trees, trees_per_iter, rate, rules, how, u, classes, logp):
        h = C.cast(how, C.POINTER(_Sampling)).contents
        self.counts = None if h.k is None else np.ctypeslib.as_array((C.c_int * n).from_address(h.k)).copy()
        self.count = h.k_all
        for out in (classes, logp):
            C.memset(out, 0, 4 * n)


@pytest.fixture
def model(monkeypatch):
    library = Library()
    monkeypatch.setattr(E._lib, "load", lambda: library)
    clf = T.TGBMClassifier(objective="multi:softprob", num_class=CLASSES, verbose=0)
    clf.model, clf.tree_per_iter, clf.group_label = 1, CLASSES, np.arange(CLASSES, dtype=np.float32)
    yield clf, library
    clf.model = None


def drawn(clf, k):
    return clf.sample_classes(np.ones((N, 2), np.float32), np.zeros(N), k=k)


def test_whole_numbers_of_any_type_keep_their_meaning(model):
    clf, library = model
    for dtype in (np.int8, np.int16, np.int32, np.int64, np.uint8, np.uint32, np.uint64):
        drawn(clf, np.array([0, 1, 4, 100], dtype))
        assert library.counts.tolist() == [0, 1, 4, CLASSES]
    # (beyond 32 bits: 2^32 + 1 is more than there are classes, and not one; what is below 0 is all)
    drawn(clf, np.array([1 << 32, (1 << 32) + 1, -(1 << 40) + 2, (1 << 31) + 3]))
    assert library.counts.tolist() == [CLASSES, CLASSES, 0, CLASSES]
    drawn(clf, np.array([1 << 63, (1 << 63) + 1, 2, 3], np.uint64))
    assert library.counts.tolist() == [CLASSES, CLASSES, 2, 3]
    drawn(clf, [3, 0, 1, 2])
    assert library.counts.tolist() == [3, 0, 1, 2]
    drawn(clf, 1 << 40)
    assert library.counts is None and library.count == CLASSES


def test_more_classes_than_a_small_type_holds(model):
    clf, library = model
    clf.tree_per_iter, clf.group_label = 70_000, np.arange(70_000, dtype=np.float32)
    for dtype, most in ((np.int8, 127), (np.uint8, 255), (np.int16, 32_767), (np.uint16, 65_535), (np.int32, 70_000), (np.uint64, 70_000)):
        drawn(clf, np.array([0, 1, 2, np.iinfo(dtype).max], dtype))
        assert library.counts.tolist() == [0, 1, 2, most]
    drawn(clf, np.array([-128, -1, 0, 5], np.int8))
    assert library.counts.tolist() == [0, 0, 0, 5]


@pytest.mark.parametrize("k", [np.full(N, 0.5), np.full(N, 2.7), np.full(N, 2.0, np.float32), np.full(N, 1 << 32, np.float64), np.full(N, np.nan), np.ones(N, bool),
                               np.array([1, 2, 3, 1 << 70], object), [1, 2, 3.5, 4]])
def test_what_are_no_whole_numbers_is_refused(model, k):
    clf, library = model
    with pytest.raises(ValueError, match="k: whole numbers"):
        drawn(clf, k)
    assert not hasattr(library, "counts")


def test_shapes_are_refused_still(model):
    clf, _ = model
    for k in (np.ones(N + 1, int), np.ones((N, 1), int), np.ones((0,), int)):
        with pytest.raises(ValueError, match="k: a number for each of 4 rows"):
            drawn(clf, k)


def test_no_rows(model):
    clf, library = model
    labels, prob = clf.sample_classes(np.ones((0, 2), np.float32), np.zeros(0), k=[])
    assert labels.shape == prob.shape == (0,)
