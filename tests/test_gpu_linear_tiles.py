"""The product by large tiles: types of the scores, features that are no whole chunks, lines behind the last whole tile in either order, and scores with a pitch of their own."""
import ctypes as C

import pytest
import torch

import thundergbm_amd as T
from thundergbm_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def whole(gen, rows, F, pitch, spare):
    """Rows of whole numbers at a pitch; behind the last one's features lies nothing unless there is something to spare, and all padding is 77."""
    memory = torch.full(((rows - 1) * pitch + F + (pitch - F if spare else 0),), 77, dtype=torch.int8, device="cuda")
    view = memory.as_strided((rows, F), (pitch, 1))
    view.copy_(torch.randint(-127, 128, (rows, F), device="cuda", generator=gen, dtype=torch.int32))
    return view


def layer(n, C_, F, w_pitch, spare, x_pitch=None):
    gen = torch.Generator("cuda").manual_seed(n + F)
    q, w = whole(gen, n, F, x_pitch or (F + 127) // 128 * 128, True), whole(gen, C_, F, w_pitch, spare)
    # (scores of about 1, which 16 bits hold)
    scale, w_scale = (torch.rand(r, device="cuda", generator=gen) / 128 + 2.0**-8 for r in (n, C_))
    bias = torch.randn(C_, device="cuda", generator=gen)
    total = w.double() @ q.double().t().contiguous()
    return q, scale, w, w_scale, bias, total.float() * scale * w_scale[:, None] + bias[:, None]


# (640: five whole chunks; 600 and 650 with rows that can be read beyond them; 656: weights that end where their features do)
FEATURES = [(640, 640, False), (600, 608, True), (650, 656, True), (656, 656, False), (656, 768, True), (650, 650, False)]


@pytest.mark.parametrize("F,w_pitch,spare", FEATURES)
@pytest.mark.parametrize("n,C_", [(1024, 32_769), (1000, 32_768 + 130), (32_769, 1024), (33_000, 1000)])
def test_types_and_features(n, C_, F, w_pitch, spare):
    q, scale, w, w_scale, bias, want = layer(n, C_, F, w_pitch, spare)
    for dtype in TYPES:
        for order in ("row", "class"):
            z = S.linear(q, w, w_scale, bias=bias, x_scale=scale, order=order, dtype=dtype)
            assert torch.equal(z, want.to(dtype))
            del z
    plain = S.linear(q, w, w_scale, x_scale=scale, order="class")  # (without a bias)
    assert torch.equal(plain, S.linear(q, w, w_scale, bias=torch.zeros_like(bias), x_scale=scale, order="row"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("n,C_,F", [(1, 700, 256), (16, 333, 2304), (30, 130, 100), (64, 100, 640), (300, 500, 130), (3000, 129, 28), (1025, 32_769, 650), (32_769, 1025, 650)])
def test_scores_with_a_pitch(n, C_, F, order, dtype):
    """What lies between the lines of the scores stays what it was."""
    q, scale, w, w_scale, bias, want = layer(n, C_, F, (F + 15) // 16 * 16, True)
    lines, width = (n, C_) if order == "row" else (C_, n)
    pitch = width + 3
    out = torch.full((lines * pitch + 5,), 7, dtype=dtype, device="cuda")
    rows = lambda x, s: S._rows(torch, "x", x, s, whole=True, floating=False)
    a, b = rows(q, scale), rows(w, w_scale)
    kind = TYPES.index(dtype)
    o = S._Scores(out.data_ptr() + 2 * out.element_size(), 1 if order == "row" else pitch, pitch if order == "row" else 1, kind, C_, n)
    lib = T.load()
    size = lib.tgbm_scores_linear_workspace(C.byref(a), C.byref(b))
    room = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    assert lib.tgbm_scores_linear(C.byref(a), C.byref(b), bias.data_ptr(), C.byref(o), room.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    got = out[2:2 + lines * pitch].view(lines, pitch)
    assert torch.equal(got[:, :width], (want.t() if order == "row" else want).to(dtype))
    assert bool((got[:, width:] == 7).all()) and bool((out[:2] == 7).all()) and bool((out[2 + lines * pitch:] == 7).all())
