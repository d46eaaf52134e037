"""The workspace of `sample`: what it is for, and that less of it is refused. Nothing is launched, so no GPU is needed."""
import ctypes as C

import pytest

import thundergbm_amd as T
from test_class_scores_cpu import ADDRESS, array, rules
from thundergbm_amd import scores as S

BUCKETS, LISTED, PARTS = 2048, 2048, 64
SPLIT_ROW = 8 * BUCKETS + 8 * LISTED + 4 * BUCKETS + 4 * PARTS + 16  # sums, listed scores and counts of a row that goes by parts, and a few numbers
SPLIT_ROWS, SPLIT_LEAST, LAID_BYTES = 384, 65_536, 128 << 20


@pytest.fixture(scope="module")
def lib():
    return T.load()


def how(**fields):
    h = S._Sampling(temperature_all=1.0, p_all=1.0)
    for k, v in fields.items():
        setattr(h, k, v)
    return h


def by_row(classes, rows):  # the classes of a row side by side
    return array(classes=classes, rows=rows, class_stride=1, row_stride=classes)


def by_class(classes, rows):
    return array(classes=classes, rows=rows, class_stride=rows, row_stride=1)


def workspace(lib, a, h=how(), r=rules()):
    return lib.tgbm_scores_sample_workspace(C.byref(a), C.byref(r), C.byref(h))


def test_long_rows(lib):
    """Few of them go by parts, with room for each row; more of them by whole rows, which want none."""
    for classes in (SPLIT_LEAST, 70_000, 1 << 22):
        for rows in (1, 2, 383, SPLIT_ROWS):
            assert workspace(lib, by_row(classes, rows)) == SPLIT_ROW * rows
        for rows in (SPLIT_ROWS + 1, 1000, 100_000):
            assert workspace(lib, by_row(classes, rows)) == 0
    assert workspace(lib, by_row(SPLIT_LEAST - 1, 5)) == 0
    # beyond 2^22 rows a call goes by slices, of which the last one may have few
    assert workspace(lib, by_row(70_000, (1 << 22) + 7)) == SPLIT_ROW * 7
    assert workspace(lib, by_row(70_000, (1 << 22) + 385)) == 0


@pytest.mark.parametrize("classes,rows", [(3000, 100), (9000, 4), (20_000, 3), (20_000, 1677), (20_000, 1678), (20_001, 5000), (1 << 20, 31), (1 << 20, 32), (1 << 20, 33), (1 << 22, 9), (40_000, 838 * 3 + 385), (70_000, 383), (70_000, 479), (70_000, 479 + 384), (70_000, 479 + 385), (65_535, 100)])
def test_rows_that_are_laid_out(lib, classes, rows):
    """As many as fit into 128 MB at a time, and room for parts where those, or what is left of them, are few and long."""
    pitch = (classes + 3) // 4 * 4
    most = max(1, min(rows, LAID_BYTES // 4 // pitch))
    sizes = {most, rows % most} - {0}
    parts = max((SPLIT_ROW * n for n in sizes if n <= SPLIT_ROWS and classes >= SPLIT_LEAST), default=0)
    assert workspace(lib, by_class(classes, rows)) == 4 * most * pitch + parts
    assert workspace(lib, by_row(classes, rows), r=rules(shown=ADDRESS, shown_begin=ADDRESS, n_shown=10 * rows, repetition=1.0)) == 4 * most * pitch + parts


WANTED = [(by_class(3000, 10), how(p_all=0.5), rules()), (by_class(3000, 10), how(k_all=5), rules()), (by_row(3000, 10), how(k_all=60), rules()), (by_row(70_000, 3), how(), rules()),
          (by_class(40_000, 7), how(min_p_all=0.1), rules()), (by_row(40_000, 700), how(), rules(shown=ADDRESS, shown_begin=ADDRESS, n_shown=9, repetition=1.0)), (by_class(100, 100_000), how(k_all=5), rules())]


@pytest.mark.parametrize("a,h,r", WANTED)
def test_less_than_is_needed_is_refused(lib, capfd, a, h, r):
    need = workspace(lib, a, h, r)
    assert need > 0
    call = lambda room, size: lib.tgbm_scores_sample(C.byref(a), C.byref(r), C.byref(h), ADDRESS, ADDRESS, ADDRESS, room, size, None)
    for room, size, msg in ((ADDRESS, need - 1, "%d bytes of workspace, %d are needed" % (need - 1, need)), (ADDRESS, 0, "0 bytes of workspace"), (None, need, "are needed"),
                            (None, 0, "are needed"), (ADDRESS + 8, need, "16 bytes"), (ADDRESS + 1, 2 * need, "16 bytes")):
        assert call(room, size) == 1
        err = capfd.readouterr().err
        assert err.startswith("tgbm_scores_sample: ") and msg in err
