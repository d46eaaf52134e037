"""The restatement of the loss against a teacher, held against differences of its own loss and against the other restatement."""
import numpy as np
import pytest

import class_scores as D
import score_oracle as O
import teacher_oracle as N


def left_over(form, C=6, n=9, K=3):
    """Rows whose teacher's masses do not come to one: every class named and some left over, the others ruled out by the student, entries that have more
    than one together, or none of these."""
    rng = np.random.default_rng(12)
    z = rng.standard_normal((C, n))
    if form == "all_named":
        K = C
    classes, t, full = D.teacher(rng, C, n, K, short=form == "plain", repeated=form == "more_than_one")
    lse = np.log(np.exp(full.astype(np.float64) / 2).sum(1))
    if form == "all_named":
        lse += 0.4
    if form == "more_than_one":
        lse -= 1.5
    if form == "others_out":
        for i in range(n):
            z[np.setdiff1d(np.arange(C), classes[i]), i] = -np.inf
    return z, classes, t, rng.integers(0, C, n).astype(np.float32), lse.astype(np.float32)


@pytest.mark.parametrize("form", ["plain", "all_named", "others_out", "more_than_one"])
@pytest.mark.parametrize("weight", [1.0, 0.75])
def test_gradient_is_the_loss_s(form, weight):
    z, classes, t, y, lse = left_over(form)
    if form == "others_out":
        y = classes[:, 0].astype(np.float32)  # (a label that the student rules out has an infinite loss)
    args = (classes, t, y, lse, 2.0, weight)
    pairs, step = N.distill(z, *args)[1], 1e-5
    for c in range(len(z)):
        up, down = z.copy(), z.copy()
        up[c] += step
        down[c] -= step
        slope = (N.distill(up, *args)[0] - N.distill(down, *args)[0]) / (2 * step)
        # (a third derivative of at most about T^-1 = 0.5 times step^2 / 6, and 2^-52 of the loss over the step)
        np.testing.assert_allclose(pairs[c, :, 0], slope, rtol=0, atol=1e-9)
    # a shift of all scores moves no probability, and so no loss: the gradient adds up to nothing
    np.testing.assert_allclose(pairs[..., 0].sum(0), 0, atol=1e-12)
    assert np.isfinite(pairs).all()


@pytest.mark.parametrize("C,n,K,T,rest", [(8, 50, 5, 1.0, False), (8, 50, 5, 2.0, True), (100, 30, 10, 0.5, True), (300, 20, 128, 2.0, False)])
def test_restatements_agree(C, n, K, T, rest):
    """Where the masses come to one."""
    rng = np.random.default_rng(C)
    z = (rng.standard_normal((C, n)) * 2).astype(np.float32)
    classes, t, full = D.teacher(rng, C, n, K)
    lse = (np.log(np.exp(full.astype(np.float64) / T).sum(1)) + 1e-6).astype(np.float32) if rest else None
    y = rng.integers(0, C, n).astype(np.float32)
    for weight in (1.0, 0.5):
        a, b = O.distill(z, classes, t, y, lse, T, weight), N.distill(z, classes, t, y, lse, T, weight)
        np.testing.assert_allclose(a[0], b[0], rtol=0, atol=1e-12)
        np.testing.assert_allclose(a[1], b[1], rtol=0, atol=1e-12)


@pytest.mark.parametrize("oracle", [O, N])
def test_rows_whose_others_are_all_out(oracle):
    """A row's numbers do not hang on the rows before it, and the first row may be one whose classes that are not named are all at -inf."""
    z, classes, t, _, lse = left_over("others_out")
    z[:, 4] = np.random.default_rng(1).standard_normal(len(z))
    together = oracle.distill(z, classes, t, None, lse, 2.0)
    for i in range(z.shape[1]):
        alone = oracle.distill(z[:, i:i + 1], classes[i:i + 1], t[i:i + 1], None, lse[i:i + 1], 2.0)
        for a, b in zip(together, alone):
            np.testing.assert_array_equal(a[i:i + 1] if a.ndim == 1 else a[:, i:i + 1], b)
        assert np.isfinite(alone[0]).all()
