"""Refusals of the sampler: nothing is launched."""
import ctypes as C

import pytest
import torch


def test_c_entry_refuses(cuda_lib):
    from lloom_b200 import _lib

    L = cuda_lib
    buf = (C.c_uint8 * 4096)()
    p = (C.addressof(buf) + 15) & ~15

    def call(x=p, type=0, b=1, v=8, ld=8, u=p, t=None, ta=1.0, k=None, ka=0, tp=None, tpa=1.0, mp=None, mpa=0.0, ids=p, probs=p):
        return L.lloom_b200_sample(x, type, b, v, ld, u, t, ta, k, ka, tp, tpa, mp, mpa, ids, probs, None)

    assert call(type=8) == _lib.ERR_DTYPE
    for bad in ({"b": 0}, {"v": 0}, {"ld": 7}, {"v": 327681, "ld": 400000}):
        assert call(**bad) == _lib.ERR_SHAPE, bad
    for bad in ({"x": None}, {"u": None}, {"ids": None}):
        assert call(**bad) == _lib.ERR_NULL, bad
    for bad in ({"x": p + 2}, {"u": p + 1}, {"ids": p + 4}, {"probs": p + 2}, {"t": p + 2}, {"k": p + 1}, {"tp": p + 2}, {"mp": p + 3}):
        assert call(**bad) == _lib.ERR_ALIGN, bad
    nan = float("nan")
    for bad in ({"ta": -0.1}, {"ta": nan}, {"ka": -1}, {"tpa": 1.1}, {"tpa": -0.1}, {"tpa": nan}, {"mpa": 1.5}, {"mpa": nan}):
        assert call(**bad) == _lib.ERR_VALUE, bad
    assert b"setting" in L.lloom_b200_error_string(_lib.ERR_VALUE)


def test_python_refuses(cuda_lib):
    from lloom_b200 import LloomError, _lib, sample, sampling

    x, u = torch.zeros(2, 8), torch.zeros(2)

    def status(*a, **kw):
        with pytest.raises(LloomError) as e:
            sample(*a, **kw)
        return e.value.status

    assert status(x, u) == _lib.ERR_DEVICE
    assert status(x.int(), u) == _lib.ERR_DTYPE
    assert status(x, u.double()) == _lib.ERR_DTYPE
    with pytest.raises((TypeError, LloomError)):
        sample(x, u, temperature="hot")
    assert sampling.MAX_VOCAB == 327680
