"""Operators on class scores, restated with numpy: one class and one row at a time where that is plainest. Scores become
32-bit numbers first and every step of an adjustment is rounded to 32 bits, as the operators are defined; sums and
exponentials are in 64 bits."""
import numpy as np


def is_allowed(allowed, allowed_set, row, rows, c):
    if allowed is None:
        return True
    sets = allowed.shape[0]
    s = (0 if sets == 1 else row) if allowed_set is None else int(allowed_set[row])
    if s < 0:
        return True
    if s >= sets:
        return False
    return bool(int(allowed[s, c // 32]) >> (c % 32) & 1)


def allowed_table(allowed, allowed_set, C, n):
    """[classes, rows] of truth values."""
    if allowed is None:
        return np.ones((C, n), bool)
    bits = ((allowed.astype(np.int64)[:, :, None] >> np.arange(32)) & 1).astype(bool).reshape(allowed.shape[0], -1)[:, :C]
    sets = allowed.shape[0]
    of = (np.zeros(n, np.int64) if sets == 1 else np.arange(n)) if allowed_set is None else allowed_set.astype(np.int64)
    table = np.zeros((n, C), bool)
    known = (of >= 0) & (of < sets)
    table[known] = bits[of[known]]
    table[of < 0] = True
    return table.T


def times_shown(shown, begin, C, n):
    m = np.zeros((C, n), np.int64)
    if shown is not None:
        for i in range(n):
            b, e = max(0, int(begin[i])), min(len(shown), int(begin[i + 1]))
            for c in shown[b:max(b, e)]:
                if 0 <= c < C:
                    m[c, i] += 1
    return m


def adjusted(z, bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None, repetition=1.0, frequency=0.0, presence=0.0):
    """z: float32 [classes, rows]; so is the result."""
    C, n = z.shape
    f = np.float32
    with np.errstate(all="ignore"):
        s = z.astype(f)
        if bias is not None:
            s = s + bias.astype(f)[:, None]
        m = times_shown(shown, shown_begin, C, n)
        less = np.where(s > 0, s / f(repetition), s * f(repetition)) - f(frequency) * m.astype(f) - f(presence)
        s = np.where(m > 0, less, s)
        assert s.dtype == f
        return np.where(allowed_table(allowed, allowed_set, C, n), s, f(-np.inf))


def top(x, k, temperature=1.0):
    """x: adjusted scores, float32 [classes, rows]. The k best of every row and the log-sum-exp."""
    C, n = x.shape
    values = np.full((n, k), -np.inf, np.float32)
    classes = np.full((n, k), -1, np.int32)
    lse = np.zeros(n)
    for i in range(n):
        s = x[:, i]
        listed = np.flatnonzero(s > -np.inf)  # (no NaN either)
        best = listed[np.argsort(-s[listed].astype(np.float64), kind="stable")][:k]
        values[i, :len(best)], classes[i, :len(best)] = s[best], best
        t = s.astype(np.float64) / temperature
        m = t.max() if not np.isnan(t).any() else np.nan
        with np.errstate(all="ignore"):
            lse[i] = m if not np.isfinite(m) else m + np.log(np.exp(t - m).sum())
    return values, classes, lse
