"""Arguments of the calls on class scores that are looked at before the library sees them."""
import ctypes as C

import numpy as np
import pytest

import thundergbm_amd as T
from thundergbm_amd import scores as S


@pytest.mark.parametrize("k", [np.int64(3), np.int32(3), np.uint8(3), 3])
def test_lengths_of_lists_are_integers_of_any_type(k):
    assert S._list_length(k) == 3 and type(S._list_length(k)) is int


@pytest.mark.parametrize("k", [0, -1, 129, np.int64(0), np.int64(129), 1.5, 3.0, np.float32(3), "3", None, np.arange(3)])
def test_lengths_of_lists_that_are_refused(k):
    with pytest.raises(ValueError, match="1 to 128"):
        S._list_length(k)
    clf = T.TGBMClassifier(objective="multi:softprob", num_class=3)
    clf.model, clf.tree_per_iter, clf.group_label = C.c_void_p(1 << 20), 3, [0.0, 1.0, 2.0]  # (an address that is never followed)
    try:
        with pytest.raises(ValueError, match="1 to 128"):
            clf.top_classes(np.zeros((2, 2), np.float32), k=k)
    finally:
        clf.model = None


def test_groups_beside_a_teacher_are_refused():
    """They would be dropped."""
    X, y = np.zeros((4, 2), np.float32), np.arange(4, dtype=np.float32)
    clf = T.TGBMClassifier(objective="multi:softprob", num_class=4)
    with pytest.raises(ValueError, match="groups"):
        clf.fit(X, y, groups=[4], teacher=T.Teacher(np.zeros((4, 1)), np.zeros((4, 1))))
    assert clf.model is None
