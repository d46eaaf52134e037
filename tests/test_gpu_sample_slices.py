"""Draws from rows that are laid out slice by slice: many to a slice, few and long ones at the end, which go by parts of a row."""
import numpy as np
import pytest
import torch

import draw_oracle as R
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C,n", [(20_000, 1677 + 3), (70_000, 479 + 3), (70_000, 479 + 385), (65_536, 512 + 384)])
def test_what_is_left_of_the_slices(C, n):
    gen = torch.Generator("cuda").manual_seed(n)
    z = torch.randn(C, n, device="cuda", generator=gen) * 3
    u = torch.rand(n, device="cuda", generator=gen)
    some = np.array([0, 1, n // 2, n - 386, n - 385, n - 384, n - 4, n - 3, n - 2, n - 1])
    for how in (dict(), dict(p=0.9, temperature=0.7), dict(k=500, min_p=0.001)):
        got = S.sample(z, u, **how)
        # the same rows with their classes side by side, which are not laid out
        by_row = S.sample(z.t().contiguous().t(), u, **how)
        assert torch.equal(got[0], by_row[0])
        # (each is rounded once to 32 bits, and off by 1e-11 at most before)
        torch.testing.assert_close(got[1], by_row[1], rtol=2.0**-23 * 1.01, atol=2e-11)
        want, logp = R.sample(z[:, some].cpu().numpy(), u.cpu().numpy()[some], **how)
        np.testing.assert_array_equal(got[0].cpu().numpy()[some], want)
        np.testing.assert_allclose(got[1].cpu().numpy()[some], logp, rtol=2.0**-24 * 1.01, atol=1e-11)
