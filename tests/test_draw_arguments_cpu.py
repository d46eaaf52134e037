"""Refusals of `sample`, `quantise` and `linear`: nothing is launched, so no GPU is needed."""
import ctypes as C

import numpy as np
import pytest
import torch

import thundergbm_amd as T
from test_class_scores_cpu import ADDRESS, BAD_ARRAYS, BAD_RULES, array, rules
from thundergbm_amd import scores as S


@pytest.fixture(scope="module")
def lib():
    return T.load()


def how(**fields):
    h = S._Sampling(temperature_all=1.0, p_all=1.0)
    for k, v in fields.items():
        setattr(h, k, v)
    return h


def rows(data=ADDRESS, scale=ADDRESS, pitch=128, kind=3, n=10, features=100, padded=1):
    return S._Rows(data, scale, pitch, kind, n, features, padded)


def ref(x):
    return None if x is None else C.byref(x)


def sample(lib, a=array(), r=rules(), h=how(), u=ADDRESS, outs=(ADDRESS, ADDRESS), room=ADDRESS, size=1 << 20):
    return lib.tgbm_scores_sample(ref(a), ref(r), ref(h), u, *outs, room, size, None)


@pytest.mark.parametrize("fields,msg", BAD_ARRAYS)
def test_sample_refuses_arrays(lib, capfd, fields, msg):
    assert sample(lib, a=array(**fields)) == 1
    err = capfd.readouterr().err
    assert err.startswith("tgbm_scores_sample: ") and msg in err


@pytest.mark.parametrize("fields,msg", BAD_RULES)
def test_sample_refuses_rules(lib, capfd, fields, msg):
    assert sample(lib, r=rules(**fields)) == 1
    assert msg in capfd.readouterr().err


NAN, INF = float("nan"), float("inf")
BAD_SETTINGS = [(dict(temperature_all=t), "temperature") for t in (-1.0, 1e-7, 2e6, NAN, INF)] + [(dict(p_all=p), "p is") for p in (0.0, -0.5, 1.5, NAN)] + \
    [(dict(min_p_all=m), "min_p") for m in (-0.1, 1.1, NAN)] + [(dict(k_all=-1), "k is -1")]


@pytest.mark.parametrize("fields,msg", BAD_SETTINGS)
def test_sample_refuses_settings(lib, capfd, fields, msg):
    assert sample(lib, h=how(**fields)) == 1
    assert msg in capfd.readouterr().err
    assert lib.tgbm_scores_sample_workspace(ref(array()), ref(rules()), ref(how(**fields))) == 0


def test_sample_refuses_nulls_and_small_workspaces(lib, capfd):
    for args in (dict(a=None), dict(r=None), dict(h=None), dict(u=None), dict(outs=(None, ADDRESS)), dict(outs=(ADDRESS, None))):
        assert sample(lib, **args) == 1
        assert capfd.readouterr().err.startswith("tgbm_scores_sample: ")
    for a, h in ((array(classes=100), how(k_all=5)), (array(classes=100), how(p_all=0.5))):
        need = lib.tgbm_scores_sample_workspace(ref(a), ref(rules()), ref(h))
        if need:
            assert sample(lib, a=a, h=h, size=need - 1) == 1 and sample(lib, a=a, h=h, room=None) == 1
            assert "workspace" in capfd.readouterr().err
    assert sample(lib, a=array(rows=0, data=None)) == 0


BAD_ROWS = [(dict(kind=4), "type 4"), (dict(kind=-1), "type -1"), (dict(n=-1), "-1 rows"), (dict(features=0), "0 features"), (dict(features=65_537, pitch=1 << 17), "65537 features"),
            (dict(pitch=99), "pitch of 99"), (dict(pitch=-128), "pitch of -128"), (dict(data=None), "null data")]


@pytest.mark.parametrize("fields,msg", BAD_ROWS)
def test_rows_are_refused(lib, capfd, fields, msg):
    quantise = lambda **f: lib.tgbm_rows_quantise(ref(rows(**{"kind": 0, **f})), ADDRESS, 1 << 18, 1 << 17, ADDRESS, None)
    assert quantise(**fields) == 1 and msg in capfd.readouterr().err
    good, out = rows(), array(classes=10)
    for x, w in ((rows(**fields), good), (good, rows(**fields))):
        assert lib.tgbm_scores_linear(ref(x), ref(w), None, ref(out), ADDRESS, 1 << 20, None) == 1
        err = capfd.readouterr().err
        assert err.startswith("tgbm_scores_linear: ") and msg in err
        assert lib.tgbm_scores_linear_workspace(ref(x), ref(w)) == 0
        capfd.readouterr()


def test_quantise_refuses(lib, capfd):
    call = lambda x=rows(kind=0), q=ADDRESS, pitch=128, width=128, scale=ADDRESS: lib.tgbm_rows_quantise(ref(x), q, pitch, width, scale, None)
    for args in (dict(x=None), dict(x=rows(kind=3)), dict(q=None), dict(scale=None), dict(width=99), dict(pitch=127)):
        assert call(**args) == 1
        assert capfd.readouterr().err.startswith("tgbm_rows_quantise: ")
    assert call(x=rows(kind=0, n=0, data=None)) == 0


def test_linear_refuses(lib, capfd):
    def call(x=rows(), w=rows(n=4), out=array(), room=ADDRESS, size=1 << 20):
        return lib.tgbm_scores_linear(ref(x), ref(w), None, ref(out), room, size, None)

    for args, msg in ((dict(x=None), "x is null"), (dict(w=None), "weights is null"), (dict(out=None), "out is null"), (dict(w=rows(n=4, kind=0)), "weights: type 0"),
                      (dict(x=rows(scale=None)), "no scales"), (dict(w=rows(n=4, scale=None)), "no scales"), (dict(x=rows(features=99)), "99 features"),
                      (dict(out=array(classes=5)), "5 classes"), (dict(out=array(rows=9)), "9 rows"), (dict(out=array(kind=3)), "unknown type"),
                      (dict(size=3), "bytes of workspace"), (dict(room=None), "bytes of workspace"), (dict(room=ADDRESS + 8), "16 bytes")):
        assert call(**args) == 1
        assert msg in capfd.readouterr().err
    # rows that can be taken as they lie want no workspace
    assert lib.tgbm_scores_linear_workspace(ref(rows(features=128)), ref(rows(features=128))) == 0
    assert lib.tgbm_scores_linear_workspace(ref(rows(features=128)), ref(rows(features=128, data=ADDRESS + 8))) > 0
    assert lib.tgbm_scores_linear_workspace(ref(rows(features=100, padded=0)), ref(rows(features=100, padded=0))) > 0


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(3, 5)
    for call in (lambda: S.sample(x, torch.zeros(5)), lambda: S.quantise(x), lambda: S.linear(x, x, x)):
        with pytest.raises(ValueError, match="on the GPU"):
            call()
    with pytest.raises(ValueError, match="torch tensor"):
        S.quantise(np.zeros((3, 5), np.float32))


@pytest.mark.parametrize("name,v", [("k", -1), ("k", 1.5), ("k", None), ("k", "3"), ("p", 0.0), ("p", 1.0001), ("p", NAN), ("p", None), ("min_p", -0.1), ("min_p", 2), ("temperature", -1.0),
                                    ("temperature", 1e-7), ("temperature", NAN), ("temperature", "hot")])
def test_settings_that_are_no_numbers_of_theirs(name, v):
    fine = {"k": (torch.int32, lambda x: x >= 0), "p": (torch.float32, lambda x: 1e-37 <= x <= 1), "min_p": (torch.float32, lambda x: 0 <= x <= 1),
            "temperature": (torch.float32, lambda x: x == 0 or 1e-6 <= x <= 1e6)}[name]
    with pytest.raises(ValueError, match=name + " is"):
        S._setting(torch, name, v, torch.zeros(3, 5), *fine, "something else")
