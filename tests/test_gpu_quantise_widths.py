"""Widths of quantised rows, which the caller of tgbm_rows_quantise chooses: zeros behind the features up to there, nothing written beyond."""
import ctypes as C

import numpy as np
import pytest
import torch

import draw_oracle as R
import thundergbm_amd as T
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu


def quantise(x, q, pitch, width, scale):
    rows = S._Rows(x.data_ptr(), None, x.stride(0), 0, x.shape[0], x.shape[1], 0)
    rc = T.load().tgbm_rows_quantise(C.byref(rows), q.data_ptr(), pitch, width, scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc


@pytest.mark.parametrize("n,F", [(3, 5), (4, 128), (3, 1000), (2, 4100), (2, 16_384), (2, 20_000)])
def test_wide_rows(n, F):
    """A padding longer than the rows themselves, and a pitch that goes beyond it."""
    x = np.random.default_rng(F).standard_normal((n, F)).astype(np.float32)
    want, want_scale = R.quantise(x)
    for width, pitch in ((F, F), (F, F + 3), (F + 1, F + 9), (70_001, 70_004), (1 << 20, 1 << 20)):
        q, scale = torch.full((n * pitch + 64,), 77, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
        assert quantise(torch.from_numpy(x).cuda(), q, pitch, width, scale) == 0
        got = q[:n * pitch].view(n, pitch)
        np.testing.assert_array_equal(got[:, :F].cpu().numpy(), want)
        np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
        assert not torch.count_nonzero(got[:, F:width]) and bool((got[:, width:] == 77).all()) and bool((q[n * pitch:] == 77).all())


@pytest.mark.parametrize("F", [16_384, 65_536])
def test_the_widest_row(F):
    """2^31 - 1 bytes: the step that leaves the padding is beyond what an int holds."""
    width = (1 << 31) - 1
    x = np.random.default_rng(F).standard_normal((1, F)).astype(np.float32)
    want, want_scale = R.quantise(x)
    q, scale = torch.full((width + 4097,), 77, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    assert quantise(torch.from_numpy(x).cuda(), q, width, width, scale) == 0
    np.testing.assert_array_equal(q[:F].cpu().numpy(), want[0])
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
    for at in range(F, width, 1 << 28):
        assert not bool(q[at:min(at + (1 << 28), width)].any())
    assert bool((q[width:] == 77).all())
