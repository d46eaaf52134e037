"""Inputs of the tests of the operators on class scores."""
import numpy as np


def bits_of(table):
    """[sets, words] of int32 from truth values [sets, classes]."""
    sets, C = table.shape
    padded = np.zeros((sets, (C + 31) // 32 * 32), np.uint64)
    padded[:, :C] = table
    words = (padded.reshape(sets, -1, 32) << np.arange(32, dtype=np.uint64)).sum(2)
    return words.astype(np.uint32).view(np.int32)


def scores(rng, C, n, special=0.0):
    """Scores of trees and the odd ones among them: equal ones, zeros of both signs, infinities, NaNs, the lowest number."""
    z = rng.standard_normal((C, n)).astype(np.float32) * 3
    z = np.where(rng.random((C, n)) < 0.3, np.round(z), z).astype(np.float32)
    if special:
        odd = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -3.4028235e38, 3.4028235e38, 1e-42], np.float32)
        z = np.where(rng.random((C, n)) < special, odd[rng.integers(0, len(odd), (C, n))], z)
    return z


def rules(rng, C, n, bias=True, sets="each", shown=True, longest=9):
    """sets: "one", "each", "some" (with rows that allow everything, rows whose number is no set's) or "none"."""
    r = {}
    if bias:
        r["bias"] = (np.round(rng.standard_normal(C) * 16) / 16).astype(np.float32)
    if sets != "none":
        count = {"one": 1, "each": n, "some": 5}[sets]
        table = rng.random((count, C)) < rng.choice([0.05, 0.5, 0.95], (count, 1))
        if sets != "one":
            table[count // 2] = False  # a row that nothing is left of
        r["allowed"] = bits_of(table)
        if sets == "some":
            r["allowed_set"] = rng.integers(-2, 7, n).astype(np.int32)
    if shown:
        lengths = rng.integers(0, longest + 1, n)
        lengths[rng.random(n) < 0.2] = 0
        begin = np.zeros(n + 1, np.int64)
        begin[1:] = np.cumsum(lengths)
        lists = (rng.random(begin[-1]) ** 3 * C).astype(np.int32)
        lists[rng.random(begin[-1]) < 0.05] = C  # no class
        lists[rng.random(begin[-1]) < 0.05] = -1
        if begin[-1]:
            r.update(shown=lists, shown_begin=begin, repetition=1.3, frequency=0.2, presence=0.4)
    return r


def teacher(rng, C, n, K, dtype=None, short=True, repeated=False):
    """(classes [n, K], scores [n, K], the log-sum-exp of a teacher over all classes at a temperature of one): lists that end early, entries that are no
    class, rows without entries, and on demand classes that several entries name."""
    full = rng.standard_normal((n, C)).astype(np.float32) * 2.5
    k = min(K, C)
    at = np.argsort(-full, axis=1, kind="stable")[:, :k].astype(np.int32)
    t = np.take_along_axis(full, at, 1)
    if k < K:
        at = np.concatenate([at, np.full((n, K - k), -1, np.int32)], 1)
        t = np.concatenate([t, np.zeros((n, K - k), np.float32)], 1)
    if short:
        at[rng.random((n, K)) < 0.1] = -1
        at[rng.random((n, K)) < 0.05] = C
        t[rng.random((n, K)) < 0.05] = -np.inf
        at[::7] = -1
    if repeated:
        from_ = rng.integers(0, K, (n, K))
        at = np.where(rng.random((n, K)) < 0.5, np.take_along_axis(at, from_, 1), at)
    shuffled = rng.permuted(np.broadcast_to(np.arange(K), (n, K)), axis=1)
    of = lambda x: np.ascontiguousarray(np.take_along_axis(x, shuffled, 1))
    return of(at), of(t), full
