"""What Model.sample_tokens hands to the library (no GPU: the call is a fake that keeps its numbers)."""
import ctypes as C

import numpy as np
import pytest

from ai00_server_b200 import capi, runtime


@pytest.fixture
def model(monkeypatch):
    class Lib:
        def b200rwkv_sample_tokens(self, h, n, q, d, tokens, probs):
            self.uniform = np.ctypeslib.as_array(C.cast(d._obj.uniform, C.POINTER(C.c_float)), (n,)).copy()
            return 0

    lib = Lib()
    monkeypatch.setattr(capi, "lib", lambda: lib)
    m = runtime.Model.__new__(runtime.Model)
    m.info, m._h, m.fake = {"num_vocab": 100}, None, lib
    monkeypatch.setattr(runtime.Model, "__del__", lambda self: None, raising=False)
    return m


BELOW_ONE = float(np.nextafter(np.float32(1), np.float32(0)))


@pytest.mark.parametrize("x", [[1 - 2.0 ** -25, 0.5], [1 - 2.0 ** -53, 0.0], np.array([1 - 2.0 ** -30, 1 - 2.0 ** -26])])
def test_doubles_below_one_stay_below_one(model, x):
    """(One in some 33 million of a program's doubles would round to 1.)"""
    model.sample_tokens([0, 1], x)
    want = [min(float(np.float32(v)), BELOW_ONE) for v in np.asarray(x)]
    assert model.fake.uniform.tolist() == want


def test_what_is_no_number_in_the_range_is_left_to_the_library(model):
    for x in ([1.0, 0.5], np.float32([1.0, 0.25]), [-0.25, 2.0], [float("nan"), 0.5]):
        model.sample_tokens([0, 1], x)
        assert np.array_equal(model.fake.uniform, np.asarray(x, np.float32), equal_nan=True)
    model.sample_tokens([0, 1], np.float32([0.1, BELOW_ONE]))
    assert model.fake.uniform.tolist() == [float(np.float32(0.1)), BELOW_ONE]
