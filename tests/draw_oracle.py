"""`sample`, `quantise` and `linear`, restated with numpy in 64 bits, a row at a time where that is plainest."""
import numpy as np

LARGEST_BELOW_ONE = 1 - 2.0**-24


def of_row(v, i):
    v = v[i] if isinstance(v, np.ndarray) else v
    return v if isinstance(v, (int, np.integer)) else float(np.float32(v))


def sample(x, u, k=0, p=1.0, min_p=0.0, temperature=1.0):
    """x: adjusted scores, float32 [classes, rows]. (classes, logp); every setting a number or an array of one for each row."""
    C, n = x.shape
    classes, logp = np.full(n, -1, np.int32), np.full(n, -np.inf)
    for i in range(n):
        T, pi, mi, ki, ui = (of_row(v, i) for v in (temperature, p, min_p, k, u))
        if any(np.isnan(v) for v in (T, pi, mi, ui)):
            logp[i] = np.nan
            continue
        s = x[:, i].astype(np.float64)
        listed = np.flatnonzero(s > -np.inf)
        if not len(listed):
            continue
        order = listed[np.argsort(-s[listed], kind="stable")]
        if T < np.float32(1e-6):
            classes[i], logp[i] = order[0], 0.0
            continue
        z = s[order]
        with np.errstate(all="ignore"):
            w = np.where(z == z[0], 1.0, np.exp((z - z[0]) / min(T, 1e6)))
        kept = w >= min(max(mi, 0.0), 1.0)
        if ki > 0:
            kept &= np.arange(len(z)) < ki
        w = np.where(kept, w, 0.0)
        if pi < 1:
            front = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            stays = front < max(pi, 0.0) * w.sum()
            stays[0] = True
            w = np.where(stays, w, 0.0)
        upto = np.cumsum(w)
        at = int(np.searchsorted(upto, min(max(ui, 0.0), LARGEST_BELOW_ONE) * upto[-1], side="right"))
        at = min(at, int(np.flatnonzero(w > 0)[-1]))
        classes[i], logp[i] = order[at], np.log(w[at] / upto[-1])
    return classes, logp


def quantise(x):
    """x: float32 [rows, features]. A scale and what is rounded are 32-bit numbers, as the operator is defined."""
    with np.errstate(all="ignore"):
        most = np.abs(x).max(1)
        fine = np.isfinite(x).all(1)
        scale = np.where(fine, most / np.float32(127), np.float32(np.nan)).astype(np.float32)
        q = np.clip(np.rint(np.where(scale[:, None] > 0, x / scale[:, None], np.float32(0))), -127, 127)
    return np.where(fine[:, None], np.nan_to_num(q), 0).astype(np.int8), scale


def linear(q, scale, w, w_scale, bias=None):
    """Whole numbers and their scales: the scores in 64 bits, [classes, rows], and how far off 32 bits may be."""
    total = w.astype(np.int64) @ q.astype(np.int64).T
    assert np.abs(total).max(initial=0) < 2**31
    with np.errstate(all="ignore"):
        z = total * scale.astype(np.float64)[None] * w_scale.astype(np.float64)[:, None]
    # the sum as a 32-bit number, two products, an addition: half a step of each, of what they give
    room = 3 * 2.0**-24 * np.abs(z)
    if bias is not None:
        z = z + bias.astype(np.float64)[:, None]
        room = room + 2.0**-24 * np.abs(z)
    return z, room * 1.01 + 1e-44
