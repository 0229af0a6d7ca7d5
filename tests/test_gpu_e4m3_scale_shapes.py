"""Scales of another shape are refused, whose elements are as many: their rows would be taken for other blocks, and products be wrong without an error."""
import pytest
import torch

from ai00_server_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


def test_scales_of_other_shapes(ops):
    n, w, outs = 4, 1024, 512                       # 8 blocks of inputs, 4 of outputs
    f = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731
    x, wide = f(n, w), f(outs, w)
    q, s = ops.to_e4m3(x)
    wq, ws = ops.to_e4m3(wide, rows=128)
    for g in (lambda: ops.linear_e4m3(q, f(8, n), wq, ws), lambda: ops.linear_e4m3(q, s, wq, f(8, 4)), lambda: ops.linear_e4m3(q, s.view(-1), wq, ws), lambda: ops.linear_e4m3(q, s, wq, ws.view(2, 16)),
              lambda: ops.linear_e4m3(q, s, wq, ws.view(4, 8, 1)), lambda: ops.linear_e4m3(q, s.t().contiguous().t(), wq, ws),
              lambda: ops.to_e4m3(x, scale=f(8, n)), lambda: ops.to_e4m3(x, scale=f(n * 8)), lambda: ops.to_e4m3(wide, rows=128, scale=f(8, 4)),
              lambda: ops.rms_norm(x, scale=f(8, n)), lambda: ops.rms_norm(x, scale=f(n * 8))):
        with pytest.raises(capi.B200Error) as ei:
            g()
        assert ei.value.code == capi.ERR_INVALID and "scale must be" in str(ei.value)


def test_scales_of_their_shape(ops):
    """Given ones are written to and handed back; one row or one block in any stride that leaves them in a row."""
    x, w = torch.randn(3, 300, device="cuda"), torch.randn(200, 300, device="cuda")
    s, ws = torch.empty(3, 3, device="cuda"), torch.empty(2, 3, device="cuda")
    q, got = ops.to_e4m3(x, scale=s)
    assert got is s
    wq, got = ops.to_e4m3(w, rows=128, scale=ws)
    assert got is ws
    k = 288                                          # (products take multiples of 16)
    qk, wk = q[:, :k].contiguous(), wq[:, :k].contiguous()
    y = ops.linear_e4m3(qk, s, wk, ws, out_dtype=torch.float32)
    one = ops.linear_e4m3(qk[:1], s[:1], wk, ws, out_dtype=torch.float32)
    strided = torch.empty(1, 40, device="cuda")[:, :3].copy_(s[:1])
    assert torch.equal(ops.linear_e4m3(qk[:1], strided, wk, ws, out_dtype=torch.float32), one)
    want = (qk.double() * s.double().repeat_interleave(128, 1)[:, :k]) @ (wk.double() * ws.double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :k]).T
    assert float((y.double() - want).abs().max()) <= 2.0 ** -16 * float(want.abs().max())
    z, got, _ = ops.rms_norm(x, scale=s)
    assert got is s and z.shape == x.shape
