"""The best classes and their log-sum-exp at the ends of the temperatures that are taken, with scores of all sizes."""
import numpy as np
import pytest
import torch

import class_scores as D
import score_oracle as O
from test_gpu_class_scores import check_top, on_gpu, place, rounded
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu

# (sizes of every way that a call can go: few classes, one to eight wavefronts to a row, tiles of rows, parts that are joined once and twice)
SIZES = [(9, 70, 3), (32, 60, 40), (100, 40, 20), (700, 40, 5), (1000, 40, 64), (1500, 40, 40), (1500, 40, 100), (5000, 5, 7), (6000, 520, 2), (12_000, 520, 50), (20_000, 520, 3),
         (70_000, 3, 128), (300_000, 2, 128)]


@pytest.mark.parametrize("order", ["class", "row"])
@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.02, 1e3, 1e6])
@pytest.mark.parametrize("C,n,k", SIZES)
def test_ends_of_the_temperatures(C, n, k, T, order):
    rng = np.random.default_rng(C + n)
    # scores of every row about a number of its own, 20 to 100 000 away from zero on either side, as far apart as the temperature makes them count or as trees' are
    middle = np.exp(rng.uniform(np.log(20), np.log(1e5), n)) * rng.choice([-1, 1], n)
    spread = rng.choice([T, 3.0], n)
    z = (middle + spread * rng.standard_normal((C, n))).astype(np.float32)
    rows = np.r_[0:min(n, 20), max(n - 20, 0):n] if n > 100 else np.arange(n)
    T32 = float(np.float32(T))
    got = S.top(place(z, order), k, temperature=T)
    check_top([x[torch.from_numpy(rows).cuda()] for x in got], z[:, rows], k, T32)
    assert bool((torch.isfinite(got[2]) == (got[1][:, 0] >= 0)).all())
    if C < 6000:
        z = rounded(z, torch.bfloat16)
        r = D.rules(rng, C, n, sets="some")
        got = S.top(place(z, order, torch.bfloat16), k, temperature=T, **on_gpu(r))
        check_top(got, O.adjusted(z, **r), k, T32)


def test_length_of_the_lists_as_numpy_s_integer():
    x = place(np.random.default_rng(1).standard_normal((50, 9)).astype(np.float32), "class")
    for a, b in zip(S.top(x, np.int64(3)), S.top(x, 3)):
        assert torch.equal(a, b)
