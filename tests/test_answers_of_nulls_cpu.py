"""Null arrays at the entry points that answer from host arrays: refused before anything is on its way to a GPU. Such a refusal ends the process, so each call has one
of its own."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SAMPLE = r"""
import ctypes as C, sys
sys.path.insert(0, %r)
import thundergbm_amd as T
from thundergbm_amd.scores import _Rules, _Sampling
room = (C.c_float * 16)()
u, classes, logp = %s
T.load().tgbm_predict_sample(1, room, room, room, None, 1, 3, 1.0, C.byref(_Rules(repetition=1.0)), C.byref(_Sampling(temperature_all=1.0, p_all=1.0)), u, classes, logp)
"""


def refusal(code):
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert out.returncode != 0
    return out.stderr


@pytest.mark.parametrize("arrays,msg", [("None, room, room", "u is null"), ("room, None, room", "an output is null"), ("room, room, None", "an output is null")])
def test_drawn_answers(arrays, msg):
    assert "tgbm_predict_sample: " + msg in refusal(SAMPLE % (ROOT, arrays))


LINEAR = r"""
import ctypes as C, sys
sys.path.insert(0, %r)
import thundergbm_amd as T
room = (C.c_float * 64)()
x, weights, values, classes, lse = %s
T.load().tgbm_linear_top(2, 4, x, 3, weights, None, 2, 1.0, values, classes, lse)
"""


@pytest.mark.parametrize("arrays,msg", [("None, room, room, room, room", "x: null data"), ("room, None, room, room, room", "weights: null data"),
                                        ("room, room, None, room, room", "an output is null"), ("room, room, room, None, room", "an output is null"),
                                        ("room, room, room, room, None", "an output is null")])
def test_a_linear_layer_as_a_teacher(arrays, msg):
    assert "tgbm_linear_top: " + msg in refusal(LINEAR % (ROOT, arrays))
