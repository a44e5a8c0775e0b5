"""Refusals of the training entry points (sc_lr_*, sc_sample): every argument
is checked on the host before anything is launched.  CPU only: the operands'
checks come before the trainer's, so a NULL trainer is what a good call is
refused for."""
import ctypes

import pytest

import surfcascade_amd as sc
from surfcascade_amd.train import _Samples, _SampleParams, _WeakBank

INVALID = -1


@pytest.fixture(scope="module")
def L():
    return sc.load_library()


def _x(**kw):
    d = dict(data=4096, dtype=0, n_patches=608, n=10, ld=608 * 32, rows=None, n_rows=0)
    d.update(kw)
    return _Samples(**d)


def _k(**kw):
    d = dict(m=608, h=1, patch=None, w=4096, b=None)
    d.update(kw)
    return _WeakBank(**d)


def _msg(L):
    return L.sc_last_error().decode()


def _response(L, x, k, act=1, res=None, kind=0, res_ld=0, y_ld=None):
    y_ld = k.m * k.h if y_ld is None else y_ld
    return L.sc_lr_response(None, ctypes.byref(x), ctypes.byref(k), act, 1.0, res, kind, res_ld, 1.0, 8192, y_ld)


def _grad(L, x, k, act=1, kind=0, dres=None, dres_ld=0, dy_ld=None):
    dy_ld = k.m * k.h if dy_ld is None else dy_ld
    return L.sc_lr_response_grad(None, ctypes.byref(x), ctypes.byref(k), act, 1.0, 8192, dy_ld, 4096, 4096, kind,
                                 1.0, dres, dres_ld, None, 0)


def _loss(L, x, k):
    return L.sc_lr_loss(None, ctypes.byref(x), ctypes.byref(k), 4096, None, 4096, 4096, 4096, None, 0)


def test_good_operands_get_to_the_trainer(L):
    assert _response(L, _x(), _k()) == INVALID and "null trainer" in _msg(L)
    assert _grad(L, _x(), _k()) == INVALID and "null trainer" in _msg(L)
    assert _loss(L, _x(), _k()) == INVALID and "null trainer" in _msg(L)
    assert _sample(L) == INVALID and "null trainer" in _msg(L)


BAD_SAMPLES = [(dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(n=-1), "samples"),
               (dict(n=2**30 + 1), "samples"), (dict(n_patches=0), "patches"), (dict(ld=608 * 32 - 1), "overlap"),
               (dict(ld=2**41), "stride"), (dict(rows=4096, n_rows=-1), "rows"),
               (dict(rows=4096, n_rows=2**30 + 1), "rows")]
BAD_BANKS = [(dict(m=-1), "weak"), (dict(h=-1), "weak"), (dict(h=1025), "weak"), (dict(m=609), "patch"),
             (dict(m=2**25, h=2, patch=4096), "too many")]


@pytest.mark.parametrize("call", [_response, _grad, _loss])
@pytest.mark.parametrize("kw,word", BAD_SAMPLES)
def test_bad_samples(L, call, kw, word):
    assert call(L, _x(**kw), _k()) == INVALID and word in _msg(L)


@pytest.mark.parametrize("call", [_response, _grad, _loss])
@pytest.mark.parametrize("kw,word", BAD_BANKS)
def test_bad_banks(L, call, kw, word):
    assert call(L, _x(), _k(**kw)) == INVALID and word in _msg(L)


def test_null_operands(L):
    assert L.sc_lr_response(None, None, None, 0, 1.0, None, 0, 0, 1.0, None, 0) == INVALID
    assert L.sc_lr_loss(None, None, None, None, None, None, None, None, None, 0) == INVALID
    assert L.sc_lr_workspace(None, None, None) == INVALID
    assert L.sc_sample_workspace(1, 1, 1, None) == INVALID
    assert L.sc_trainer_create(0, None) == INVALID
    assert L.sc_trainer_synchronize(None) == INVALID
    assert L.sc_trainer_wait_stream(None, None) == INVALID
    assert L.sc_stream_wait_trainer(None, None) == INVALID
    assert L.sc_trainer_set_stream(None, None, 1) == INVALID
    assert L.sc_trainer_stream(None) is None
    L.sc_trainer_destroy(None)


def test_response_arguments(L):
    x, k = _x(), _k()
    assert _response(L, x, k, act=2) == INVALID and "activation" in _msg(L)
    assert _response(L, x, k, kind=3, res=4096) == INVALID and "residual" in _msg(L)
    assert _response(L, x, k, kind=1) == INVALID and "residual" in _msg(L)
    assert _response(L, x, k, res=4096) == INVALID and "residual" in _msg(L)
    assert _response(L, x, k, kind=2, res=4096, res_ld=607) == INVALID and "res_ld" in _msg(L)
    assert _response(L, x, k, kind=1, res=4096, res_ld=0) == INVALID and "res_ld" in _msg(L)
    assert _response(L, x, k, y_ld=607) == INVALID and "y_ld" in _msg(L)


def test_grad_arguments(L):
    x, k = _x(), _k()
    assert _grad(L, x, k, act=-1) == INVALID and "activation" in _msg(L)
    assert _grad(L, x, k, kind=2) == INVALID and "dres" in _msg(L)
    assert _grad(L, x, k, dres=4096) == INVALID and "dres" in _msg(L)
    assert _grad(L, x, k, kind=2, dres=4096, dres_ld=607) == INVALID and "dres_ld" in _msg(L)
    assert _grad(L, x, k, dy_ld=607) == INVALID and "dy_ld" in _msg(L)
    # learners that do not exist leave a row residual's gradient to be written
    assert _grad(L, x, _k(m=0), kind=1) == INVALID and "dres" in _msg(L)


def _sample(L, dtype=0, b=2, v=10, ld=10, s=3, u_ld=3, index_ld=3, prm=None):
    return L.sc_sample(None, 4096, dtype, b, v, ld, None, ctypes.byref(prm) if prm else None, 4096, s, u_ld, 4096,
                       index_ld, None, None, 0)


@pytest.mark.parametrize("kw,word", [(dict(dtype=7), "type"), (dict(b=-1), "negative"), (dict(v=-1), "negative"),
                                     (dict(s=-1), "negative"), (dict(v=2**26 + 1, ld=2**27), "2^26"),
                                     (dict(ld=9), "overlap"), (dict(u_ld=2), "overlap"),
                                     (dict(index_ld=2), "overlap")])
def test_sample_sizes(L, kw, word):
    assert _sample(L, **kw) == INVALID and word in _msg(L)


@pytest.mark.parametrize("prm,word", [((-1.0, 0, 1.0, 0.0), "temperature"), ((float("nan"), 0, 1.0, 0.0), "temperature"),
                                      ((float("inf"), 0, 1.0, 0.0), "temperature"), ((1.0, -1, 1.0, 0.0), "top_k"),
                                      ((1.0, 0, -0.1, 0.0), "top_p"), ((1.0, 0, float("nan"), 0.0), "top_p"),
                                      ((1.0, 0, 1.0, 1.5), "min_p"), ((1.0, 0, 1.0, float("nan")), "min_p")])
def test_sample_parameters(L, prm, word):
    assert _sample(L, prm=_SampleParams(*prm)) == INVALID and word in _msg(L)


def test_sample_defaults(L):
    p = _SampleParams(9, 9, 9, 9)
    L.sc_sample_params_default(ctypes.byref(p))
    assert (p.temperature, p.top_k, p.top_p, p.min_p) == (1.0, 0, 1.0, 0.0)
    L.sc_sample_params_default(None)


def test_workspace_sizes(L):
    n = ctypes.c_size_t(99)
    for x, k in ((_x(n=0), _k()), (_x(), _k(m=0)), (_x(rows=4096, n_rows=0), _k())):
        assert L.sc_lr_workspace(ctypes.byref(x), ctypes.byref(k), ctypes.byref(n)) == 0 and n.value == 0
    x = _x(n=100000)
    assert L.sc_lr_workspace(ctypes.byref(x), ctypes.byref(_k()), ctypes.byref(n)) == 0
    assert n.value % (608 * 34 * 4) == 0
    assert L.sc_sample_workspace(-1, 1, 1, ctypes.byref(n)) == INVALID
    assert L.sc_sample_workspace(0, 0, 0, ctypes.byref(n)) == 0


def test_no_gpu_is_a_device_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(sc.SurfCascadeError) as e:
        sc.Trainer()
    assert e.value.code == -5


@pytest.mark.parametrize("kw", [dict(b=2**30 + 1), dict(s=2**30 + 1, u_ld=2**31, index_ld=2**31)])
def test_too_many_rows_or_draws(L, kw):
    assert _sample(L, **kw) == INVALID and "2^30" in _msg(L)
    size = ctypes.c_size_t()
    assert L.sc_sample_workspace(kw.get("b", 1), 10, kw.get("s", 1), ctypes.byref(size)) == INVALID
