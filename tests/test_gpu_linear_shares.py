"""Products of many features by few classes: the wavefronts of a workgroup share the features, four, eight or sixteen of them."""
import numpy as np
import pytest

import test_gpu_linear as L
from thundergbm_amd import scores as S

pytestmark = L.pytestmark


@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("n,F,C", [(3, 2049, 17), (9, 65_536, 40), (17, 2100, 70), (24, 8192, 1000), (32, 20_001, 130), (20, 65_536, 100), (33, 2049, 5), (64, 8192, 65), (100, 8192, 500), (500, 2300, 9)])
def test_shared_features(n, F, C, order):
    rng = np.random.default_rng(n + F * 3 + C)
    q, scale, w, w_scale, bias = L.case(rng, n, F, C)
    for j, dtype in enumerate(L.TYPES):
        pad_w = (-F % 128, 3, -F % 16)[j]
        got = S.linear(L.strided(q, (0, 5, -F % 128)[j]), L.strided(w, pad_w, shift=16 * (j != 1)), w_scale.cuda(), bias=bias.cuda(), x_scale=scale.cuda(), order=order, dtype=dtype)
        L.check(got, q, scale, w, w_scale, bias, dtype)
