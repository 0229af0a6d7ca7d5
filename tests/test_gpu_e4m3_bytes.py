"""8-bit numbers byte for byte: those of a division by the scale in f32 and a conversion to float8_e4m3fn, which any other program makes of the same values (on the CPU here)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


def rnd(*shape, std=1.0, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def check_bytes(q, scale, y, rows):
    """q and scale are those of the f32 values y."""
    y, q, scale = y.float().cpu(), q.cpu(), scale.cpu()
    n, w = y.shape
    pad = torch.nn.functional.pad(torch.where(y.isnan(), 0.0, y).abs(), (0, -w % 128, 0, -n % rows))
    assert torch.equal(scale, pad.view(-1, rows, pad.shape[1] // 128, 128).amax((1, 3)).clamp(min=2.0 ** -100) / 448)
    want = (y / scale.repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :w]).clamp(-448, 448).to(E4M3)      # (a hair above 448 is 448)
    nan = want.float().isnan()
    assert torch.equal(q.float().isnan(), nan)
    off = (q.view(torch.uint8) != want.view(torch.uint8)) & ~nan
    assert not bool(off.any()), (int(off.sum()), y[off][:4], q.float()[off][:4], want.float()[off][:4])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("n,w", [(1, 1), (131, 1000), (333, 8960), (700, 1027), (1400, 512)])
def test_rows_and_blocks(ops, dtype, rows, n, w):
    """Values of 16 bits often lie on the ties of their group."""
    for x in (rnd(n, w, dtype=dtype, seed=n), rnd(n, w, seed=n + 1).square().to(dtype)):
        check_bytes(*ops.to_e4m3(x, rows=rows), x, rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("w", [512, 513])
def test_every_tie(ops, rows, w):
    """Groups whose largest makes every number and every tie between two of them a value, at the smallest and the largest scales too."""
    numbers = torch.arange(0x7F, dtype=torch.uint8).view(E4M3).float()                  # 0 .. 448
    ties = (numbers[1:] + numbers[:-1]) / 2
    x = torch.zeros(rows * 8, w)
    for i, unit in enumerate((1.0, 2.0 ** -110, 2.0 ** -72, 2.0 ** -70, 2.0 ** 119, 3 * 2.0 ** -120, 5 * 2.0 ** -73, 7 * 2.0 ** 3)):
        r = i * rows
        x[r, :127], x[r, 128:254], x[r, 256:382] = numbers * unit, ties * unit, -ties * unit
        x[r, 254] = x[r, 382] = 448 * unit
        x[r, 384:510] = torch.nextafter(ties, torch.zeros(())) * unit
        x[r, 510] = -448 * unit
    x = x.cuda()
    check_bytes(*ops.to_e4m3(x, rows=rows), x, rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("w", [256, 301])
def test_zeros_infinities_and_scales_of_all_sizes(ops, rows, w):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(rows * 40, w)
    for i in range(36):
        x[i * rows] = torch.randn(w, generator=torch.Generator().manual_seed(i)) * 2.0 ** (-143 + 7.5 * i)
    x[:, 3] = -0.0
    x[36 * rows, :6] = torch.tensor([inf, -2.0, -0.0, 0.0, 3.0, -inf])
    x[37 * rows, :4] = torch.tensor([nan, 2.0, -0.0, -1e-30])
    x[38 * rows] = -0.0
    x[39 * rows, :3] = torch.tensor([3.4e38, -3.4e38, 1e-45])
    x = x.cuda()
    check_bytes(*ops.to_e4m3(x, rows=rows), x, rows)


@pytest.mark.parametrize("n,w", [(1, 2560), (5, 8201), (700, 4096), (1300, 1001)])
@pytest.mark.parametrize("weight", [F32, BF16])
def test_norm(ops, n, w, weight):
    """What the norm makes 8 bits of are the rows that it hands out in f32."""
    x, g = rnd(n, w, std=2.0, seed=w), (1 + rnd(w, std=0.3, seed=2)).to(weight)
    y, _, _ = ops.rms_norm(x, g, offset=0.25, out_dtype=F32)
    q, s, _ = ops.rms_norm(x, g, offset=0.25)
    check_bytes(q, s, y, 1)
