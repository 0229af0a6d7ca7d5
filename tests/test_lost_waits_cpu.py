"""b200rwkv_op_lost_waits: what the host can see is refused (no GPU needed)."""
import ctypes as C

import pytest

from ai00_server_b200 import capi


def test_null_and_no_device():
    assert capi.lib().b200rwkv_op_lost_waits(0, None) == capi.ERR_INVALID
    total = C.c_int64(-5)
    with pytest.raises(capi.B200Error):
        capi.check(capi.lib().b200rwkv_op_lost_waits(1 << 20, C.byref(total)))
    assert total.value == -5
