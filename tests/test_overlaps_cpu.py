"""Outputs that lie in what a call reads, or in one another: a list or a row without gaps beside rows that have some (no GPU needed: a call that is taken fails for want of a device)."""
import ctypes as C

import pytest

from ai00_server_b200 import capi
from tests.test_token_ops_cpu import CALLS, made

WIDE = dict(x=1 << 20, x_stride=200)                 # 4 rows of 100 f16: bytes 0 to 200 of every 400


def code(call, change):
    cls, fields = CALLS[call]
    return getattr(capi.lib(), "b200rwkv_" + call)(0, None, C.byref(made(cls, fields, change)))


@pytest.mark.parametrize("call", ["op_norm", "op_e4m3"])
@pytest.mark.parametrize("at", [-12, 0, 100, 196, 388, 400, 596, 800, 1196, 1396])
def test_scales_in_rows_with_gaps(call, at):
    """Sixteen bytes of scales that reach into a row."""
    assert code(call, {**WIDE, "scale": (1 << 20) + at}) == capi.ERR_INVALID


@pytest.mark.parametrize("call", ["op_norm", "op_e4m3"])
@pytest.mark.parametrize("at", [-16, 200, 300, 384, 600, 784, 1000, 1400])
def test_scales_in_gaps(call, at):
    """And that do not: as far as the device."""
    assert code(call, {**WIDE, "scale": (1 << 20) + at}) not in (capi.ERR_INVALID, capi.ERR_UNSUPPORTED)


def test_tokens_in_rows_with_gaps():
    wide = dict(logits=1 << 20, logits_stride=200)   # 4 rows of 100 f32: bytes 0 to 400 of every 800
    for at, refused in ((0, True), (396, True), (400, False), (784, False), (788, True), (1200, False), (2396, True), (2796, True), (2800, False), (-12, True), (-16, False)):
        for name in ("tokens", "probs"):
            got = code("op_sample", {**wide, name: (1 << 20) + at})
            assert (got == capi.ERR_INVALID) == refused, (at, name, got)


def test_weights_and_rows_of_outputs_with_gaps():
    """A weight, or scales of products, under rows of outputs that lie apart."""
    out = dict(out=4 << 20, out_stride=200)          # 4 rows of 100 bytes of 8 bits
    assert code("op_norm", {**out, "weight": (4 << 20) + 300}) == capi.ERR_INVALID           # (400 bytes: over a gap and the rows beside it)
    rows = dict(out=6 << 20, out_stride=400)         # 4 rows of 100 bf16: bytes 0 to 200 of every 800
    assert code("op_linear_e4m3", {**rows, "x_scale": (6 << 20) + 180}) == capi.ERR_INVALID   # (32 bytes)
    assert code("op_linear_e4m3", {**rows, "x_scale": (6 << 20) + 200}) not in (capi.ERR_INVALID, capi.ERR_UNSUPPORTED)
    assert code("op_linear_e4m3", {**rows, "x_scale": (6 << 20) + 780}) == capi.ERR_INVALID
