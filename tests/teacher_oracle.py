"""The loss against a teacher and its gradient pairs, from the definition in 64 bits, with how far off 32 bits may be.

Apart from score_oracle.distill in two things. Where the teacher's masses M = sum(q) + r are not one - all that is left over has no class to go to, or the
entries have more than one together - the gradient is M p - q, the loss's own. And what may be off hangs on how far an entry lies below the
row's best one, not on how large the scores are: what all of them have in common falls out of q.

u = 2^-24 is half a step of a 32-bit number near one. An exponential of -x has four in its argument (the difference, the factor log2(e) / T, which has two
itself, the product) times x, and two in its value; a logarithm three times its value and two. A sum of positive terms has one for each addition in a row."""
import numpy as np

U, LEAST = 2.0**-24, 2.0**-126


def softmax(x, adds):
    """Of x, which may hold -inf: the logarithms, the values, how far off those may be (relative), and that of their sum."""
    top = x.max() if x.size else -np.inf
    if not np.isfinite(top):
        return np.full(x.shape, -np.inf), np.zeros(x.shape), np.zeros(x.shape), 0.0, 0.0
    below = top - x
    e = np.exp(-below)
    total = e.sum()
    below = np.where(e > 0, below, 0.0)
    off_sum = U * (4 * (e * below).sum() / total + 8 + adds)
    return -(top - x) - np.log(total), e / total, U * (4 * below + 14) + off_sum, off_sum, np.log(total)


def row(z, classes, teacher, y, lse, T, w):
    C, K = len(z), len(classes)
    adds = min(C, 136)
    x = z / T
    logp, p, off_p, off_Z, log_Z = softmax(x, adds)
    dp = p * off_p + LEAST
    there = (classes >= 0) & (classes < C) & (teacher != -np.inf)
    c, t = classes[there], teacher[there]
    q, dq, named = np.zeros(C), np.zeros(C), np.zeros(C, bool)
    given = d_given = 0.0
    if len(c):
        top = t.max()
        below = (top - t) / T
        if lse is None:
            e = np.exp(-below)
            scale = 1 / e.sum()
            off = U * (4 * below + 4 + K + 12 + (e * (4 * below + 2)).sum() * scale)
        else:
            scale = np.exp(top / T - lse)
            e = np.exp(-below)
            off = U * (4 * below + abs(top / T) + 3 * abs(top / T - lse) + 8)
        qe = e * scale
        dqe = qe * off + LEAST * (1 + scale)
        np.add.at(q, c, qe)
        np.add.at(dq, c, dqe + qe * U * K)
        named[c] = True
        given, d_given = qe.sum(), dqe.sum() + qe.sum() * U * (K + 12)
    takes = len(c) > 0 and lse is not None and bool(np.any(logp[~named] > -np.inf))  # whether there is a class for the rest
    r, dr, M, dM = 0.0, 0.0, 1.0, 0.0
    target, d_target = q.copy(), dq.copy()
    if lse is not None:
        M = max(given, 1.0) if takes else given
        dM = 0.0 if takes and given < 1 - d_given - U else d_given + U
    if takes:
        r, dr = max(0.0, 1.0 - given), d_given + U
        log_share, share, off_share, off_R, log_R_ = softmax(np.where(named, -np.inf, x), adds)
        log_R = x[~named].max() + log_R_ - (x.max() + log_Z)
        target = np.where(named, q, r * share)
        d_target = np.where(named, dq, dr * share + r * share * (off_share + 3 * U) + LEAST)
    a = w if len(c) else 0.0
    soft = room = 0.0
    if len(c):
        with np.errstate(all="ignore"):
            some = np.flatnonzero(q > 0)
            far = x[named].max() - x[named]
            far = np.where(np.isfinite(far), far, 0).max()
            higher = abs(x.max() - x[named].max())
            terms = np.log(q[some]) - logp[some]
            soft = (q[some] * terms).sum()
            # the sum of q (log q - d / T), d below the highest of the named, and the mass times (log Z + what lies between); classes whose q is no
            # normal number may be left out
            size = q[some] * (np.abs(np.log(q[some])) + np.where(np.isfinite(x[some]), x[named].max() - x[some], 0))
            room = (dq[some] * (np.abs(terms) + 1)).sum() + U * ((K + 24) * size.sum() + 2 * q.sum() + 4 * q.sum() * far)
            room += LEAST * (90 + np.abs(terms)).sum()
            level = abs(log_Z) + higher
            room += q.sum() * (off_Z + U * (3 * abs(log_Z) + 2 + 3 * higher + (K + 16) * level))
        if takes:
            between = abs(x[~named].max() - x.max())
            if r > 0:
                soft += r * (np.log(r) - log_R)
            room += dr * (abs(np.log(max(r, dr))) + abs(log_R) + 2)
            room += r * (off_R + off_Z + U * ((4 * abs(np.log(r)) if r > 0 else 0) + 6 * abs(log_R_) + 6 * abs(log_Z) + 6 * between + 8))
        room += 6 * U * abs(soft)
    with np.errstate(all="ignore"):
        loss, room = (a * T * T * soft, a * T * T * room) if a else (0.0, 0.0)
        g, dg = a * T * (M * p - target), a * T * (M * dp + dM * p + d_target + 6 * U * (M * p + target))
        h, dh = a * M * p * (1 - p), a * (M * dp + dM * p + 4 * U * M * p)
    if y is not None and w < 1 and 0 <= y < C and y == np.floor(y):
        y, b = int(y), 1 - w
        log1, p1, off1, off_Z1, log_Z1 = softmax(z, adds)
        hot = np.arange(C) == y
        loss = loss - b * log1[y]
        room += b * (off_Z1 + U * (3 * abs(log_Z1) + 2 + 3 * abs(z.max() - z[y]) + 4 * abs(log1[y]))) + 4 * U * abs(loss)
        d1 = p1 * off1 + LEAST
        g, dg = g + b * (p1 - hot), dg + b * (d1 + 4 * U * (p1 + hot))
        h, dh = h + b * p1 * (1 - p1), dh + b * (d1 + 4 * U * p1)
    pairs = np.stack([g, np.maximum(2 * h, 1e-16)], 1)
    return loss, pairs, room + 1e-37, np.stack([dg + 4 * U * np.abs(g) + 1e-37, 2 * dh + 4 * U * 2 * h + 1e-22], 1)


def distill(z, classes, teacher, labels=None, lse=None, temperature=1.0, weight=1.0):
    """z: [classes, rows]. loss [rows] and pairs [classes, rows, 2], and how far off each may be, laid out the same."""
    T, w = float(np.float32(temperature)), float(np.float32(weight))
    z, teacher = z.astype(np.float64), teacher.astype(np.float64)
    with np.errstate(all="ignore"):
        rows = [row(z[:, i], classes[i], teacher[i], None if labels is None else labels[i], None if lse is None else float(lse[i]), T, w) for i in range(z.shape[1])]
    loss, pairs, loss_room, pairs_room = zip(*rows)
    return np.array(loss), np.stack(pairs, 1), np.array(loss_room), np.stack(pairs_room, 1)
