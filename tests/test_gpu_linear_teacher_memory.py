"""What a linear layer as a teacher holds on the device: slices of its rows, however wide they are."""
import ctypes as C

import numpy as np
import pytest

import datasets as D
import thundergbm_amd as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device_memory():
    """Free memory, once the library has given back what it keeps."""
    D.warm_up(T)
    hip = C.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))

    def free():
        f, t = C.c_size_t(), C.c_size_t()
        assert hip.hipMemGetInfo(C.byref(f), C.byref(t)) == 0
        return f.value

    return free


def held(free, call):
    """The result, and the blocks that the call left to be kept: the most that it held at a time, by size."""
    T.release_memory()
    before = free()
    out = call()
    return out, before - free()


def whole_numbers(rows, width, shift):
    """Rows with whole numbers up to 127 in magnitude, 127 among them: 8 bits hold them as they are, and sums of their products are exact."""
    at = np.arange(rows, dtype=np.int64)[:, None] * (13 + shift) + np.arange(width, dtype=np.int64) * 7
    x = (at % 11 - 5).astype(np.float32)
    x[:, 0] = 127
    return x


def test_wide_rows_go_by_slices(device_memory):
    """2.5 slices of 256 MB: features of 8 bits beside one of them, few scores."""
    n, F, C_, k = 10_240, 16_384, 4, 2
    x, w = whole_numbers(n, F, 0), whole_numbers(C_, F, 3)
    teacher, bytes_held = held(device_memory, lambda: T.Teacher.linear(x, w, np.arange(C_), k=k))
    assert bytes_held < (1 << 28) + (1 << 26) + (1 << 25), bytes_held  # (a slice's features in 32 and in 8 bits, all else)
    scores = (x @ w.T).astype(np.float64)  # (whole numbers below 2^24)
    order = np.argsort(-scores, 1, kind="stable")[:, :k]
    np.testing.assert_array_equal(teacher.labels, order.astype(np.float32))
    np.testing.assert_array_equal(teacher.scores, np.take_along_axis(scores, order, 1))


def test_weights_go_by_slices(device_memory):
    """Weights of 1.5 slices: what stays of them is their 8 bits."""
    n, F, C_, k = 4096, 4096, 24_576, 5
    x, w = whole_numbers(n, F, 0), whole_numbers(C_, F, 3)
    bias = (np.arange(C_) % 5).astype(np.float32)
    teacher, bytes_held = held(device_memory, lambda: T.Teacher.linear(x, w, np.arange(C_), bias=bias, k=k))
    # the slice that either of them comes through, the weights in 8 bits, 2730 rows' scores, their features in 8 bits; lists, what top wants beside them and the like
    assert bytes_held < (1 << 28) + C_ * F + (1 << 28) + (1 << 24) + (1 << 25), bytes_held
    some = np.array([0, 1, 2729, 2730, 2731, n - 1])
    scores = (x[some] @ w.T + bias).astype(np.float64)
    order = np.argsort(-scores, 1, kind="stable")[:, :k]
    np.testing.assert_array_equal(teacher.labels[some], order.astype(np.float32))
    np.testing.assert_array_equal(teacher.scores[some], np.take_along_axis(scores, order, 1))
