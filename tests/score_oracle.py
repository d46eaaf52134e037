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


def log_softmax(z):
    """Down the columns; a column of -inf alone stays one."""
    m = z.max(0)
    with np.errstate(all="ignore"):
        lse = np.where(np.isneginf(m), 0.0, m + np.log(np.exp(z - m).sum(0)))
        return z - lse


def distill(z, classes, teacher, labels=None, lse=None, temperature=1.0, weight=1.0):
    """z: [classes, rows]. loss [rows] and pairs [classes, rows, 2], in 64 bits, and how far off 32 bits may be (of each).

    The room: u = 2^-24 for a rounding. An exponential of -x has three in its argument and two in its value: (3 x + 2) u. A
    sum has one for every addition in a row, `adds`: at most 76 within a thread, 10 over the threads and 50 over chunks
    (fewer where a row has few classes), and the errors of its terms, 3 u times their mean x, which is at most ln C. Products and quotients
    have one each. In what the entries give: the quotient by the temperature, the sum's logarithm (four), the additions."""
    T, u = float(temperature), 2.0**-24
    C, n = z.shape
    z = z.astype(np.float64)
    loss, pairs = np.zeros(n), np.zeros((C, n, 2))
    loss_room, pairs_room = np.zeros(n), np.zeros((C, n, 2))
    logp, log1 = log_softmax(z / T), log_softmax(z)
    adds = min(C, 76 + 10 + 50)
    w = float(np.float32(weight))
    for i in range(n):
        finite = z[np.isfinite(z[:, i]), i]
        spread = np.ptp(finite) if finite.size else 0.0
        q, named, norm, sum_dq = np.zeros(C), np.zeros(C, bool), 0.0, 0.0
        dq = np.zeros(C)
        entries = [(int(c), float(t) / T) for c, t in zip(classes[i], teacher[i]) if 0 <= c < C and t != -np.inf]
        with np.errstate(all="ignore"):
            if entries:
                ts = np.array([t for _, t in entries])
                norm = float(lse[i]) if lse is not None else ts.max() + np.log(np.exp(ts - ts.max()).sum())
                for c, t in entries:
                    e = np.exp(t - norm)
                    named[c] = True
                    q[c] += e
                    d = e * u * (4 * abs(t) + 2 * abs(norm) + len(entries) + 20)
                    dq[c] += d
                    sum_dq += d
            p = np.exp(logp[:, i])
            x = np.where(p > 0, -logp[:, i], 0)
            dp = p * u * (3 * x + 2 * adds + 6 * np.log(C) + 16)
            mass = sum(np.exp(t - norm) for _, t in entries)
            r = 0.0
            target, dtarget = q.copy(), dq.copy()
            takes_rest = bool(entries) and lse is not None and not named.all() and bool(np.any(logp[~named, i] > -np.inf))
            if takes_rest:
                r = max(0.0, 1.0 - mass)
                dr = sum_dq + u * (len(entries) + 2)
                log_R = np.log(p[~named].sum()) if p[~named].sum() > 1e-280 else log_sum(logp[~named, i])
                share = np.exp(np.where(named, -np.inf, logp[:, i] - log_R))
                target = np.where(named, q, r * share)
                xs = np.where(share > 0, -np.log(np.where(share > 0, share, 1)), 0)
                dtarget = np.where(named, dq, dr * share + r * share * u * (3 * xs + 2 * adds + 6 * np.log(C) + 16))
            a = w if entries else 0.0
            soft = soft_room = 0.0
            if entries:
                for c in np.flatnonzero(q > 0):
                    soft += q[c] * (np.log(q[c]) - logp[c, i])
                    soft_room += dq[c] * (abs(np.log(q[c]) - logp[c, i]) + 1)
                    soft_room += q[c] * u * (6 * abs(np.log(q[c])) + 8 * abs(logp[c, i]) + 2 * adds + 6 * np.log(C) + 30 + 4 * spread / T)
                if r > 0:
                    soft += r * (np.log(r) - log_R)
                if takes_rest:
                    soft_room += dr * (abs(np.log(max(r, dr))) + abs(log_R) + 2) if np.isfinite(log_R) else 0
                    soft_room += r * u * (6 * abs(np.log(r)) if r > 0 else 0) + r * u * (8 * abs(log_R) + 2 * adds + 6 * np.log(C) + 30 + 4 * spread / T)
                soft_room += 4 * u * abs(soft)
            value, room = a * T * T * soft if a else 0.0, a * T * T * soft_room
            g = a * T * (p - target) if a else np.zeros(C)
            dg = a * T * (dp + dtarget + 3 * u * (p + target))
            h, dh = a * p * (1 - p), a * (dp + 3 * u * p)
            if labels is not None and weight < 1:
                y = labels[i]
                if 0 <= y < C and y == np.floor(y):
                    y, b = int(y), 1 - w
                    p1 = np.exp(log1[:, i])
                    x1 = np.where(p1 > 0, -log1[:, i], 0)
                    dp1 = p1 * u * (3 * x1 + 2 * adds + 6 * np.log(C) + 16)
                    value = value - b * log1[y, i]
                    room += b * u * (8 * abs(log1[y, i]) + 2 * adds + 6 * np.log(C) + 30 + 4 * spread) + 4 * u * abs(value)
                    hot = np.arange(C) == y
                    g = g + b * (p1 - hot)
                    dg = dg + b * (dp1 + 3 * u * (p1 + hot))
                    h, dh = h + b * p1 * (1 - p1), dh + b * (dp1 + 3 * u * p1)
            loss[i], loss_room[i] = value, room + 1e-37
            pairs[:, i, 0], pairs[:, i, 1] = g, np.maximum(2 * h, 1e-16)
            pairs_room[:, i, 0], pairs_room[:, i, 1] = dg + 4 * u * np.abs(g) + 1e-37, 2 * dh + 4 * u * 2 * h + 1e-22
    return loss, pairs, loss_room, pairs_room


def log_sum(x):
    m = x.max()
    return m + np.log(np.exp(x - m).sum())
