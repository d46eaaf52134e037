"""Refusals of the operators on class scores: nothing is launched, so no GPU is needed."""
import ctypes as C

import numpy as np
import pytest
import torch

import thundergbm_amd as T
from thundergbm_amd import scores as S


@pytest.fixture(scope="module")
def lib():
    return T.load()


ADDRESS = 1 << 20  # (never followed)


def array(data=ADDRESS, class_stride=10, row_stride=1, kind=0, classes=4, rows=10):
    return S._Scores(data, class_stride, row_stride, kind, classes, rows)


def rules(**fields):
    r = S._Rules(repetition=1.0)
    for k, v in fields.items():
        setattr(r, k, v)
    return r


BAD_ARRAYS = [
    (dict(kind=3), "unknown type"),
    (dict(kind=-1), "unknown type"),
    (dict(classes=0), "0 classes"),
    (dict(classes=(1 << 22) + 1), "classes"),
    (dict(rows=-1), "-1 rows"),
    (dict(data=None), "null data"),
    (dict(class_stride=9), "strides 9 and 1"),
    (dict(class_stride=0), "strides 0 and 1"),
    (dict(class_stride=-10), "strides -10 and 1"),
    (dict(class_stride=2, row_stride=8), "strides 2 and 8"),
    (dict(class_stride=1, row_stride=3), "strides 1 and 3"),
    (dict(class_stride=1, row_stride=0), "strides 1 and 0"),
]
BAD_RULES = [
    (dict(allowed=ADDRESS, allowed_sets=0), "0 allowed sets"),
    (dict(allowed=ADDRESS, allowed_sets=9), "9 allowed sets for 10 rows"),
    (dict(allowed_set=ADDRESS), "allowed_set without allowed"),
    (dict(shown=ADDRESS, n_shown=3), "shown without shown_begin"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=-1), "n_shown is -1"),
    (dict(shown_begin=ADDRESS, n_shown=2), "shown_begin without shown"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=2, repetition=0.0), "repetition is 0"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=2, repetition=-1.0), "repetition is -1"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=2, repetition=float("nan")), "repetition is nan"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=2, frequency=float("inf")), "frequency inf"),
    (dict(shown=ADDRESS, shown_begin=ADDRESS, n_shown=2, presence=float("nan")), "presence"),
]


@pytest.mark.parametrize("fields,msg", BAD_ARRAYS)
def test_adjust_refuses_arrays(lib, capfd, fields, msg):
    for pair in ((array(**fields), array()), (array(), array(**fields))):
        assert lib.tgbm_scores_adjust(C.byref(pair[0]), C.byref(rules()), C.byref(pair[1]), None) == 1
        err = capfd.readouterr().err
        assert err.startswith("tgbm_scores_adjust: ") and msg in err


@pytest.mark.parametrize("fields,msg", BAD_RULES)
def test_adjust_refuses_rules(lib, capfd, fields, msg):
    assert lib.tgbm_scores_adjust(C.byref(array()), C.byref(rules(**fields)), C.byref(array(data=2 * ADDRESS)), None) == 1
    assert msg in capfd.readouterr().err


def test_adjust_refuses_pairs_and_nulls(lib, capfd):
    good, r = array(), rules()
    for args in ((None, r, good), (good, None, good), (good, r, None), (good, r, array(rows=9)), (good, r, array(kind=1)),
                 (good, r, array(classes=3)), (good, r, array(class_stride=1, row_stride=4))):
        assert lib.tgbm_scores_adjust(*(C.byref(a) if a is not None else None for a in args), None) == 1
        assert capfd.readouterr().err.startswith("tgbm_scores_adjust: ")


@pytest.mark.parametrize("away,out", [
    (4, dict()), (36, dict()), (-36, dict()), (156, dict()), (156, dict(class_stride=1, row_stride=4)),
    (4 * 9, dict(class_stride=20)), (4 * 15, dict(class_stride=20)), (4 * 20 - 4, dict(class_stride=20)), (2, dict(kind=1)),
    (4, dict(classes=1, class_stride=0)), (4, dict(rows=1, class_stride=1, row_stride=0)), (8, dict(rows=1, class_stride=2)),
])
def test_adjust_refuses_overlaps(lib, capfd, away, out):
    of_in = {k: v for k, v in out.items() if k in ("kind", "classes", "rows") or out.get("class_stride") in (0, 2, 20) or "rows" in out}
    assert lib.tgbm_scores_adjust(C.byref(array(**of_in)), C.byref(rules()), C.byref(array(data=ADDRESS + away, **out)), None) == 1
    assert "out overlaps in" in capfd.readouterr().err


def test_no_rows_are_no_work(lib):
    assert lib.tgbm_scores_adjust(C.byref(array(rows=0, data=None)), C.byref(rules()), C.byref(array(rows=0, data=None)), None) == 0


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(3, 5)
    with pytest.raises(ValueError, match="on the GPU"):
        S.adjust(x)
    with pytest.raises(ValueError, match="torch tensor"):
        S.adjust(np.zeros((3, 5), np.float32))


def test_parts_of_one_array_are_told_apart():
    at = lambda data, width, pitch: S._Scores(ADDRESS + data, pitch, 1, 0, 4, width)
    assert S._apart(at(0, 4, 10), at(16, 4, 10), 4)
    assert S._apart(at(16, 4, 10), at(0, 4, 10), 4)
    assert S._apart(at(0, 5, 10), at(20, 5, 10), 4)
    assert not S._apart(at(0, 4, 10), at(12, 4, 10), 4)
    assert not S._apart(at(0, 4, 10), at(28, 4, 10), 4)
    assert not S._apart(at(0, 4, 10), at(16, 4, 9), 4)


def test_top_refuses(lib, capfd):
    good, r = array(), rules()

    def call(a=good, rule=r, k=3, temperature=1.0, outs=(ADDRESS,) * 3, room=ADDRESS, size=1 << 20):
        return lib.tgbm_scores_top(C.byref(a), C.byref(rule), k, temperature, *outs, room, size, None)

    for fields, msg in BAD_ARRAYS:
        assert call(a=array(**fields)) == 1 and msg in capfd.readouterr().err
    for fields, msg in BAD_RULES:
        assert call(rule=rules(**fields)) == 1 and msg in capfd.readouterr().err
    large = array(class_stride=1, row_stride=100_000, classes=100_000, rows=2)
    needed = lib.tgbm_scores_top_workspace(C.byref(large), 5)
    assert needed > 0
    for more, msg in ((dict(k=0), "k is 0"), (dict(k=129), "k is 129"), (dict(temperature=0.0), "temperature"), (dict(temperature=float("inf")), "temperature"),
                      (dict(outs=(None, ADDRESS, ADDRESS)), "null"), (dict(outs=(ADDRESS, ADDRESS, None)), "null"),
                      (dict(a=large, k=5, size=needed - 1), "workspace"), (dict(a=large, k=5, room=None, size=needed), "workspace")):
        assert call(**more) == 1 and msg in capfd.readouterr().err
    assert call(a=array(rows=0)) == 0


@pytest.mark.parametrize("by_class", [True, False])
def test_top_workspace(lib, by_class):
    """No workspace for a row that goes in one piece, none asked for by a call that is refused, and always room for the chunks."""
    for classes in (1, 32, 33, 1024, 1025, 16_384, 16_385, 1 << 20, 1 << 22):
        for rows in (1, 2, 100, 5000, 100_000):
            a = array(class_stride=rows, row_stride=1, classes=classes, rows=rows) if by_class else array(class_stride=1, row_stride=classes, classes=classes, rows=rows)
            for k in (1, 10, 128):
                size = lib.tgbm_scores_top_workspace(C.byref(a), k)
                # (two parts of a row at least, each with its lists and its sum)
                assert size == 0 or size >= rows * 2 * (8 * k + 8)
                assert size > 0 or classes <= 1 << 16
                assert classes > 32 or size == 0
                assert lib.tgbm_scores_top_workspace(C.byref(a), 0) == lib.tgbm_scores_top_workspace(C.byref(a), 129) == 0


@pytest.mark.parametrize("last", [1, 2, 7, 40, 1000])
@pytest.mark.parametrize("classes", [33, 700, 1600, 2100, 5000, 40_000])
def test_workspace_of_rows_beyond_a_launch(lib, classes, last):
    """Rows go by slices of 2^22: the few of the last one are shared out over the chip, and their parts have room too."""
    rows = (1 << 22) + last
    for class_stride, row_stride in ((rows, 1), (1, classes)):
        many, few = (array(class_stride=class_stride, row_stride=row_stride, classes=classes, rows=n) for n in (rows, last))
        for k in (1, 20, 128):
            assert lib.tgbm_scores_top_workspace(C.byref(many), k) >= lib.tgbm_scores_top_workspace(C.byref(few), k)
    many, few = (array(class_stride=rows, classes=classes, rows=n) for n in (rows, last))
    for entries in (1, 32, 128):
        assert lib.tgbm_scores_distill_workspace(C.byref(many), entries) >= lib.tgbm_scores_distill_workspace(C.byref(few), entries)


def test_distill_refuses(lib, capfd):
    def call(a=array(), teacher=True, classes=ADDRESS, scores=ADDRESS, kind=0, entries=3, labels=ADDRESS, temperature=1.0, weight=0.5, loss=ADDRESS, pairs=ADDRESS,
             stride=10, room=ADDRESS, size=1 << 20):
        t = S._Teacher(classes, scores, None, kind, entries)
        return lib.tgbm_scores_distill(C.byref(a), C.byref(t) if teacher else None, labels, temperature, weight, loss, pairs, stride, room, size, None)

    for fields, msg in BAD_ARRAYS:
        assert call(a=array(**fields)) == 1 and msg in capfd.readouterr().err
    large = array(class_stride=100, classes=100_000, rows=100)
    needed = lib.tgbm_scores_distill_workspace(C.byref(large), 3)
    assert needed > 0
    for more, msg in ((dict(a=array(kind=1)), "float scores"), (dict(a=array(class_stride=1, row_stride=4)), "side by side"), (dict(teacher=False), "teacher"),
                      (dict(kind=7), "unknown type"), (dict(entries=0), "0 entries"), (dict(entries=129), "129 entries"), (dict(classes=None), "null"),
                      (dict(scores=None), "null"), (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                      (dict(weight=-0.1), "weight"), (dict(weight=float("nan")), "weight"), (dict(labels=None), "labels"), (dict(stride=9), "pair_stride"),
                      (dict(loss=None, pairs=None), "no output"), (dict(a=large, stride=100, size=needed - 1), "workspace"),
                      (dict(a=large, stride=100, room=None), "workspace")):
        assert call(**more) == 1 and msg in capfd.readouterr().err, more
    assert call(a=array(rows=0)) == 0
    assert lib.tgbm_scores_distill_workspace(C.byref(large), 0) == lib.tgbm_scores_distill_workspace(C.byref(large), 129) == 0


@pytest.mark.parametrize("rules", [dict(repetition=1e-60), dict(repetition=1e60), dict(repetition=-1.0), dict(frequency=1e300), dict(presence=float("nan"))])
def test_estimator_refuses_numbers_that_32_bits_do_not_hold(rules):
    """Before the library sees them, which ends the process."""
    clf = T.TGBMClassifier(objective="multi:softprob", num_class=3)
    clf.model, clf.tree_per_iter, clf.group_label = C.c_void_p(ADDRESS), 3, [0.0, 1.0, 2.0]
    try:
        with pytest.raises(ValueError, match="above 0"):
            clf._class_rules(2, None, None, [[1.0], [2.0]], **dict(dict(repetition=1.0, frequency=0.0, presence=0.0), **rules))
        clf._class_rules(2, None, None, [[1.0], [2.0]], 1.5, 0.1, -0.1)
    finally:
        clf.model = None
