"""Operators from the residual rows of a step to its tokens (ai00_server_b200.device_ops: rms_norm, to_e4m3, linear_e4m3, sample) against their definitions in 64
bits, at the sizes, masks and layouts where they can go wrong.

Tolerances.  An e4m3 number is off by half a step: 2^-4 of the value, or 2^-10 below the smallest normal number.  A scale is one f32 division: 2^-24, and 2^-23 more once it is a
reciprocal and multiplied.  Norms: a thread adds up to 64 squares in a row and the block some 12 sums more, each off by 2^-24 of a sum of positive terms: 2^-17 of the mean at
most, half of it in its root; rsqrtf and three products add 2^-22 each at most: 2^-17 altogether.  Products: those of two e4m3 numbers are exact; a step of 32 of them with its running sum is off by
2^-22 of the magnitudes at most, four steps to a block, and a block's factor and multiply-add by 2^-23 more, for every block in turn and up to eight parts.  Tokens are equal: sums are exact
in units of 2^-40, 64-bit ones off by 2^-53 a term, and none of the fixed inputs here has a border between."""
import numpy as np
import pytest
import torch

from ai00_server_b200 import capi

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


def rnd(*shape, std=1.0, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def spread(scale, rows, shape):
    """A scale for every value."""
    return scale.double().repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def check_e4m3(q, scale, y, rows, off=0.0):
    """q and scale stand for y [64 bits], of which every value may be off by `off` of itself beforehand."""
    n, w = y.shape
    assert q.dtype == E4M3 and q.shape == y.shape and scale.dtype == F32
    pad = torch.nn.functional.pad(y.abs(), (0, -w % 128, 0, -n % rows))
    want = pad.view(-1, rows, pad.shape[1] // 128, 128).amax((1, 3)).clamp(min=2.0 ** -100) / 448
    assert bool(((scale.double() - want).abs() <= want * (2.0 ** -24 + off)).all())
    s = spread(scale, rows, y.shape)
    bad = (q.double() * s - y).abs() > torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20) + y.abs() * (2.0 ** -22 + 2 * off)
    assert not bool(bad.any()), int(bad.sum())


# ---- to_e4m3 --------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,w", [(1, 1), (1, 8), (3, 127), (2, 128), (5, 129), (128, 136), (127, 1000), (129, 264), (300, 513), (17, 8960), (1000, 40)])
@pytest.mark.parametrize("rows", [1, 128])
def test_rows_in_8_bits(ops, dtype, n, w, rows):
    x = rnd(n, w, std=3.0, dtype=dtype, seed=n + w)
    q, s = ops.to_e4m3(x, rows=rows)
    check_e4m3(q, s, x.double(), rows)
    again = ops.to_e4m3(x, rows=rows)
    assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1], s)


@pytest.mark.parametrize("rows", [1, 128])
def test_rows_in_8_bits_zeros_and_extremes(ops, rows):
    x = torch.zeros(rows * 4, 512, device="cuda")
    r = slice(0, rows)
    x[r, 130], x[r, 131] = 3e38, -3e38
    x[rows:2 * rows, 0], x[rows:2 * rows, 200], x[rows:2 * rows, 300] = 1e-38, 1e-30, 1e-45
    x[2 * rows, 5], x[2 * rows, 6] = float("nan"), 2.0
    x[3 * rows, 300], x[3 * rows, 301] = float("inf"), 2.0
    q, s = ops.to_e4m3(x, rows=rows)
    v = q.float() * spread(s, rows, x.shape).float()
    assert not v[:rows, :128].any() and not v[:rows, 256:].any()
    assert bool(((v[:rows, 130:132] - x[:rows, 130:132]).abs() <= 2.0 ** -4 * 3e38).all())
    assert bool((s >= 2.0 ** -100 / 448 * (1 - 2.0 ** -23)).all()) and bool(v[rows:2 * rows].isfinite().all())
    # (each off by half a step: of its own size, or of the smallest numbers of the least scale)
    off, least = (v[rows:2 * rows] - x[rows:2 * rows]).abs(), 2.0 ** -100 / 448 * 2.0 ** -10
    fine = off <= (x[rows:2 * rows] * 2.0 ** -4).clamp(min=least) * (1 + 1e-6)
    assert bool(fine.all())
    nan = q[2 * rows].float().isnan()
    assert bool(nan[5]) and int(nan.sum()) == 1 and abs(float(v[2 * rows, 6]) - 2.0) <= 2.0 * 2.0 ** -4
    assert bool(q[3 * rows, 300].float().isnan()) and bool(s[3, 2].isinf()) and float(q[3 * rows, 301].float()) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 128])
def test_rows_in_8_bits_strides_and_rows_behind(ops, dtype, rows):
    n, w = 131, 200
    for at, gap in ((0, 24), (3, 5), (8, 8)):
        wide = rnd(n + 1, w + at + gap, dtype=dtype, seed=at)
        out = torch.full((n + 2, w + at + gap), 7.0, device="cuda").to(E4M3)
        q, s = ops.to_e4m3(wide[:n, at:at + w], rows=rows, out=out[:n, at:at + w])
        check_e4m3(q, s, wide[:n, at:at + w].double(), rows)
        keep = torch.ones(out.shape, dtype=torch.bool, device="cuda")
        keep[:n, at:at + w] = False
        assert bool((out.float()[keep] == 7.0).all())


def test_rows_in_8_bits_many_and_none(ops):
    for n, w, rows in ((0, 100, 1), (0, 100, 128), (1 << 18, 9, 1), (1 << 18, 9, 128)):
        x = rnd(n, w, dtype=F16, seed=3)
        q, s = ops.to_e4m3(x, rows=rows)
        assert q.shape == (n, w) and s.shape == (-(-n // rows), 1)
        if n:
            check_e4m3(q, s, x.double(), rows)


# ---- rms_norm -------------------------------------------------------------------------------------------------------------------------------
def norm_want(x, weight, residual, eps, offset):
    h = x.double() + (residual.double() if residual is not None else 0)
    w = weight.double() if weight is not None else torch.ones(x.shape[1], dtype=torch.float64, device="cuda")
    return h / (h.square().mean(1, keepdim=True) + eps).sqrt() * (offset + w)


# f32: h itself is off by 2^-24 of the larger summand where its two cancel
def norm_off(x, residual, y, weight, offset):
    if residual is None:
        return 0.0
    h = x.double() + residual.double()
    big = torch.maximum(x.double().abs(), residual.double().abs())
    return 2.0 ** -24 * big / h.square().mean(1, keepdim=True).sqrt() * (offset + weight.double()).abs()


def check_norm(ops, x, weight, residual, eps, offset, out_dtype, got):
    out, scale, total = got
    y = norm_want(x, weight, residual, eps, offset)
    if residual is not None:
        assert torch.equal(total, (x.float() + residual.float()).to(residual.dtype))
    slack = norm_off(x, residual, y, weight, offset) if weight is not None else 0.0
    if out_dtype is E4M3:
        s = spread(scale, 1, y.shape)
        want = torch.nn.functional.pad(y.abs(), (0, -y.shape[1] % 128)).view(y.shape[0], -1, 128).amax(2).clamp(min=2.0 ** -100) / 448
        most = float(slack.max()) / 448 if residual is not None and weight is not None else 0.0
        assert bool(((scale.double() - want).abs() <= want * 2.0 ** -16 + most).all())
        err = (out.double() * s - y).abs()
        bound = torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -14) + y.abs() * 2.0 ** -16 + 2 * slack
    else:
        assert scale is None and out.dtype == out_dtype
        err = (out.double() - y).abs()
        bound = y.abs() * (torch.finfo(out_dtype).eps / 2 + 2.0 ** -17) + 2 * slack + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
    assert bool((err <= bound).all()), float((err / (bound + 1e-300)).max())


@pytest.mark.parametrize("dtype,res,weight,out", [
    (F32, F32, F32, E4M3), (F32, None, None, F32), (F16, F16, F32, E4M3), (F16, F32, F16, F16), (F16, None, F16, E4M3), (BF16, BF16, BF16, E4M3), (BF16, F32, F32, E4M3),
    (BF16, None, F32, BF16), (F16, F32, BF16, E4M3)])
@pytest.mark.parametrize("n,w", [(1, 1), (2, 7), (3, 128), (4, 255), (1, 2560), (333, 1000), (400, 2056), (310, 4096), (2, 8192), (5, 8201), (300, 8960), (3, 16384), (2, 20000), (3, 32768)])
def test_norm_against_64_bits(ops, dtype, res, weight, out, n, w):
    x = rnd(n, w, std=2.0, dtype=dtype, seed=w)
    r = rnd(n, w, std=5.0, dtype=res, seed=w + 1) if res else None
    g = (1 + rnd(w, std=0.3, seed=2)).to(weight) if weight else None
    got = ops.rms_norm(x, g, residual=r, eps=1e-5, out_dtype=out)
    check_norm(ops, x, g, r, 1e-5, 0.0, out, got)
    again = ops.rms_norm(x, g, residual=r, eps=1e-5, out_dtype=out)
    assert all(a is b or torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("n", [3, 700])
def test_norm_offset_in_place_and_strides(ops, dtype, res, n):
    """Weights stored as offsets from one; the sum over the residual, and over x; rows of wider buffers, on and off boundaries, of which nothing else changes."""
    w = 520
    for at, gap in ((0, 8), (16, 0), (5, 2)):
        wide_x = rnd(n + 1, w + at + gap, dtype=dtype, seed=1)
        wide_r = rnd(n + 1, w + at + gap, std=4.0, dtype=res, seed=2)
        wide_o = torch.full((n + 1, w + at + gap), 5.0, device="cuda").to(E4M3)
        x, r, o = (t[:n, at:at + w] for t in (wide_x, wide_r, wide_o))
        g = rnd(w, std=0.2, seed=3)
        before_x, before_r = wide_x.clone(), wide_r.clone()
        got = ops.rms_norm(x, g, residual=r, eps=1e-3, offset=1.0, out=o, residual_out=r)
        check_norm(ops, before_x[:n, at:at + w], g, before_r[:n, at:at + w], 1e-3, 1.0, E4M3, got)
        assert got[2] is r and torch.equal(wide_x, before_x)
        keep = torch.ones(wide_r.shape, dtype=torch.bool, device="cuda")
        keep[:n, at:at + w] = False
        assert torch.equal(wide_r[keep], before_r[keep]) and bool((wide_o.float()[keep] == 5.0).all())
        if dtype == res:
            y = before_r[:n, at:at + w]
            got = ops.rms_norm(x, g, residual=y, eps=1e-3, offset=1.0, residual_out=x)
            check_norm(ops, before_x[:n, at:at + w], g, y, 1e-3, 1.0, E4M3, got)
            assert torch.equal(wide_x[keep], before_x[keep])


@pytest.mark.parametrize("dtype,res,weight,out", [(F32, F32, F32, E4M3), (F32, None, None, F32), (F16, F32, F16, F16), (BF16, BF16, BF16, E4M3), (BF16, None, F32, E4M3), (F16, F32, BF16, E4M3)])
@pytest.mark.parametrize("n,w", [(7301, 8), (5000, 136), (4000, 1000), (2001, 2560), (1100, 4096), (7301, 3), (3700, 1001), (1100, 4095)])
def test_norm_of_more_rows_than_stay_on_the_gpu(ops, dtype, res, weight, out, n, w):
    """CTAs take several rows one after another: each row as if it were alone, its residual in place."""
    x = rnd(n, w, std=2.0, dtype=dtype, seed=w)
    r = rnd(n, w, std=5.0, dtype=res, seed=w + 1) if res else None
    g = (1 + rnd(w, std=0.3, seed=2)).to(weight) if weight else None
    got = ops.rms_norm(x, g, residual=r, eps=1e-5, offset=0.25, out_dtype=out)
    check_norm(ops, x, g, r, 1e-5, 0.25, out, got)
    few = ops.rms_norm(x[-3:], g, residual=None if r is None else r[-3:], eps=1e-5, offset=0.25, out_dtype=out)
    if r is not None:
        assert torch.equal(few[2], got[2][-3:])
        again = r.clone()
        ops.rms_norm(x, g, residual=again, eps=1e-5, offset=0.25, out_dtype=out, residual_out=again)
        assert torch.equal(again, got[2])


def test_norm_rows_that_are_zero_or_no_number(ops):
    x = rnd(4, 300, seed=1)
    x[1] = 0.0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    clean = ops.rms_norm(x[:1].contiguous(), torch.ones(300, device="cuda"))
    q, s, _ = ops.rms_norm(x, torch.ones(300, device="cuda"))
    assert torch.equal(q[0].view(torch.uint8), clean[0][0].view(torch.uint8))
    assert not q[1].float().any() and bool(s[1].isfinite().all())
    assert bool(q[2].float().isnan().all())
    assert bool(q[3, 9].float().isnan())
    y, _, _ = ops.rms_norm(x, torch.ones(300, device="cuda"), out_dtype=F32)
    assert not y[1].any() and bool(y[2].isnan().all()) and bool(y[3, 9].isnan()) and bool((y[3, 10:] == 0).all())
    assert ops.rms_norm(x[:0], None)[0].shape == (0, 300)


# ---- linear_e4m3 ----------------------------------------------------------------------------------------------------------------------------
def e4m3_of(x, rows):
    """(numbers, scales) by torch alone."""
    n, w = x.shape
    g = torch.nn.functional.pad(x, (0, -w % 128, 0, -n % rows)).view(-(-n // rows), rows, -(-w // 128), 128)
    s = g.abs().amax((1, 3)).clamp(min=2.0 ** -100) / 448
    return (g / s[:, None, :, None]).reshape(-1, g.shape[2] * 128)[:n, :w].to(E4M3).contiguous(), s


def make_linear(T, K, N, seed=0):
    # (columns of one block in a few are far larger: blocks that weigh much beside ones that do not)
    x, xs = e4m3_of(rnd(T, K, seed=seed) * (1 + 30 * (torch.arange(K, device="cuda") // 128 % 5 == 2)), 1)
    w, ws = e4m3_of(rnd(N, K, std=K ** -0.5, seed=seed + 1), 128)
    return x, xs, w, ws


def check_linear(out, x, xs, w, ws, base):
    xd, wd = x.double() * spread(xs, 1, x.shape), w.double() * spread(ws, 128, w.shape)
    y = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    blocks = xs.shape[1]
    err = mag * (4 * 2.0 ** -22 + (blocks + 16) * 2.0 ** -23)
    if base is not None:
        y = y + base.double()
        err = err + 2.0 ** -24 * y.abs()
    err = err * (1 + 2.0 ** -8) + torch.finfo(out.dtype).eps / 2 * y.abs() + 1e-30
    if out.dtype == F16:
        err = err + 2.0 ** -25
    bad = (out.double() - y).abs() > err
    assert not bool(bad.any()), (int(bad.sum()), float(((out.double() - y).abs() / err).max()))


LINEAR = [(1, 16, 1), (1, 2560, 2560), (2, 144, 5), (7, 272, 130), (16, 128, 128), (16, 4096, 640), (17, 1040, 257), (32, 256, 384), (33, 512, 129), (64, 1024, 300), (65, 400, 64),
          (100, 2048, 1000), (128, 384, 200), (129, 640, 256), (200, 272, 700), (300, 4096, 130), (333, 8960, 96), (600, 512, 5000), (1021, 1040, 2570), (513, 144, 10250)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,K,N", LINEAR)
def test_linear_against_64_bits(ops, dtype, T, K, N):
    x, xs, w, ws = make_linear(T, K, N, seed=T + K)
    out = ops.linear_e4m3(x, xs, w, ws, out_dtype=dtype)
    check_linear(out, x, xs, w, ws, None)
    assert torch.equal(out, ops.linear_e4m3(x, xs, w, ws, out_dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,N", [(1, 1024, 640), (5, 272, 130), (40, 512, 257), (100, 1024, 384), (333, 1040, 2570), (1030, 512, 5001), (1500, 256, 2560)])
def test_linear_with_a_base_and_in_place(ops, dtype, T, K, N):
    x, xs, w, ws = make_linear(T, K, N, seed=T)
    base = rnd(T, N, dtype=dtype, seed=5)
    out = ops.linear_e4m3(x, xs, w, ws, base=base)
    check_linear(out, x, xs, w, ws, base)
    here = base.clone()
    assert ops.linear_e4m3(x, xs, w, ws, base=here, out=here) is here
    assert torch.equal(here, out)


@pytest.mark.parametrize("T", [1, 20, 130, 700])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_linear_strides_and_rows_behind(ops, dtype, T):
    """x, base and out as columns of wider tensors; what lies beside and behind stays as it was, and what lies behind x and its rows is not read."""
    K, N = 272, 2567
    x, xs, w, ws = make_linear(T, K, N, seed=T)
    for at, gap in ((0, 0), (5, 4), (8, 9)):
        wide_x = torch.full((T + 2, K + 48), 0x7F, dtype=torch.uint8, device="cuda").view(E4M3)          # NaN
        wide_x[:T, 16:16 + K] = x
        wide_b = rnd(T + 1, N + at + gap, dtype=dtype, seed=9)
        wide_o = torch.full((T + 3, N + at + gap), 7.0, dtype=dtype, device="cuda")
        ops.linear_e4m3(wide_x[:T, 16:16 + K], xs, w, ws, base=wide_b[:T, at:at + N], out=wide_o[:T, at:at + N])
        check_linear(wide_o[:T, at:at + N], x, xs, w, ws, wide_b[:T, at:at + N])
        keep = torch.ones_like(wide_o, dtype=torch.bool)
        keep[:T, at:at + N] = False
        assert bool((wide_o[keep] == 7.0).all())


@pytest.mark.parametrize("T", [3, 300, 900])
def test_linear_bad_values_stay_with_their_token(ops, T):
    x, xs, w, ws = make_linear(T, 1040, 3000, seed=1)
    clean = ops.linear_e4m3(x, xs, w, ws, out_dtype=F32)
    dirty, scales = x.clone(), xs.clone()
    dirty.view(torch.uint8)[1, 700] = 0x7F
    scales[2, 8] = float("inf")
    out = ops.linear_e4m3(dirty, scales, w, ws, out_dtype=F32)
    assert bool(out[1].isnan().all()) and not bool(out[2].isfinite().any())
    others = torch.ones(T, dtype=torch.bool, device="cuda")
    others[1:3] = False
    assert torch.equal(out[others], clean[others])


def test_linear_no_tokens_and_far_rows(ops):
    x, xs, w, ws = make_linear(4, 64, 40)
    assert ops.linear_e4m3(x[:0], xs[:0], w, ws).shape == (0, 40)
    step = ((1 << 32) // 3 + 4096) & ~15
    far = torch.empty(3 * step + 64, dtype=torch.uint8, device="cuda").view(E4M3).as_strided((4, 64), (step, 1))
    far.copy_(x)
    out = torch.empty(3 * step + 64, dtype=F16, device="cuda").as_strided((4, 40), (step, 1))
    ops.linear_e4m3(far, xs, w, ws, out=out)
    check_linear(out.contiguous(), x, xs, w, ws, None)


@pytest.mark.parametrize("T,K,N,out", [(133, 192, 61143, BF16), (128, 144, 75777, F16), (300, 272, 20001, F32), (257, 128, 19009, BF16), (700, 1040, 9999, F16)])
def test_linear_of_many_outputs_and_few_inputs(ops, T, K, N, out):
    """Tiles whose ends cost more than their products: rows of base and out that start off boundaries, the base in place, part of a wider buffer."""
    x, xs = e4m3_of(rnd(T, K, seed=1), 1)
    w, ws = e4m3_of(rnd(N, K, std=K ** -0.5, seed=2), 128)
    wide = rnd(T + 1, N + 3, dtype=out, seed=3)
    before, part = wide.clone(), wide[:T, 1:1 + N]
    exact = (x.double() * spread(xs, 1, x.shape)) @ (w.double() * spread(ws, 128, w.shape)).T
    most = (x.double() * spread(xs, 1, x.shape)).abs() @ (w.double() * spread(ws, 128, w.shape)).abs().T
    ops.linear_e4m3(x, xs, w, ws, base=part, out=part)
    want = exact + before[:T, 1:1 + N].double()
    # (the steps' bound of the head of this file for up to nine blocks of inputs, the addition of the base, the rounding of what comes out)
    bound = most * 9 * 2.0 ** -20 + want.abs() * (2.0 ** -23 + torch.finfo(out).eps / 2) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
    assert bool(((part.double() - want).abs() <= bound).all())
    wide[:T, 1:1 + N] = before[:T, 1:1 + N]
    assert torch.equal(wide, before)
    plain = ops.linear_e4m3(x, xs, w, ws, out_dtype=out)
    assert bool(((plain.double() - exact).abs() <= most * 9 * 2.0 ** -20 + exact.abs() * torch.finfo(out).eps / 2 + torch.finfo(out).smallest_normal * torch.finfo(out).eps).all())


# ---- sample ---------------------------------------------------------------------------------------------------------------------------------
def draw_want(logits, u, temperature, top_k, top_p, min_p):
    """(token, share) of a row, from the definition."""
    l = np.asarray(logits, np.float64)
    top = l.max()
    if np.isnan(l).any() or np.isnan([u, temperature, top_p, min_p]).any() or not 0 <= temperature < np.inf:
        return -1, np.nan
    if top == -np.inf:
        return -1, 0.0
    order = np.lexsort((np.arange(l.size), -l))
    if temperature == 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.where(l == top, 1.0, np.exp((l - top) / temperature))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        s = np.cumsum(w[order])
        order = order[:max(1, int((s < max(top_p, 0) * s[-1]).sum()) + 1)]
    order = np.concatenate([order[:1], order[1:][w[order[1:]] >= min(min_p, 1.0)]])
    ids = np.sort(order)
    s = np.cumsum(w[ids])
    j = min(int((s <= max(u, 0.0) * s[-1]).sum()), np.flatnonzero(w[ids])[-1])
    return int(ids[j]), w[ids[j]] / s[-1]


def check_draws(tokens, probs, rows, u, temperature=None, top_k=None, top_p=None, min_p=None):
    n = rows.shape[0]
    l = rows.double().cpu().numpy()
    at = lambda x, i, none: none if x is None else x[i].item()  # noqa: E731
    want = [draw_want(l[i], u[i].item(), at(temperature, i, 1.0), at(top_k, i, 0), at(top_p, i, 1.0), at(min_p, i, 0.0)) for i in range(n)]
    assert tokens.tolist() == [t for t, _ in want]
    p = np.array([x for _, x in want])
    got = probs.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(p))
    fine = ~np.isnan(p)
    assert (np.abs(got - p)[fine] <= 2.0 ** -23 * p[fine] + rows.shape[1] * 2.0 ** -40).all()


def limits(n, seed, ks=(1, 2, 40, 300), k=True, p=True, m=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.rand(n, generator=g)  # noqa: E731
    t = 0.3 + 1.5 * r()
    t[::7] = 0.0
    top_k = torch.tensor([0, *ks])[(r() * (len(ks) + 1)).long()].to(torch.int32)
    top_p = torch.where(r() < 0.3, 1.0, r())
    min_p = torch.where(r() < 0.4, 0.0, 0.3 * r() ** 3)
    give = lambda x, want: x.cuda() if want else None  # noqa: E731
    return dict(temperature=t.cuda(), top_k=give(top_k, k), top_p=give(top_p, p), min_p=give(min_p, m)), r().cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,V,std", [(1, 1, 1.0), (5, 2, 1.0), (9, 31, 2.0), (20, 257, 1.0), (16, 1000, 3.0), (33, 2048, 1.0), (17, 4099, 2.0), (12, 32000, 2.5), (16, 65536, 3.0), (40, 65536, 1.0),
                                     (6, 100003, 2.0), (3, 262147, 1.5), (2, 524288, 2.0), (130, 5001, 4.0)])
def test_tokens_against_64_bits(ops, dtype, n, V, std):
    rows = rnd(n, V, std=std, dtype=dtype, seed=V + n)
    kw, u = limits(n, V)
    tokens, probs = ops.sample(rows, u, **kw)
    check_draws(tokens, probs, rows, u, **kw)
    again = ops.sample(rows, u, **kw)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], probs)


@pytest.mark.parametrize("which", ["", "k", "p", "m", "kp", "pm", "km"])
@pytest.mark.parametrize("n,V", [(8, 65536), (200, 9000)])
def test_tokens_limits_alone(ops, which, n, V):
    rows = rnd(n, V, std=2.0, seed=3)
    kw, u = limits(n, 5, k="k" in which, p="p" in which, m="m" in which)
    if which == "":
        kw["temperature"] = None
    tokens, probs = ops.sample(rows, u, **kw)
    check_draws(tokens, probs, rows, u, **kw)


def test_tokens_follow_the_distribution(ops):
    """Every border of a small row: u from just below to just above the sums."""
    V = 37
    row = rnd(1, V, std=1.5, seed=4)
    w = torch.softmax(row.double(), 1).cumsum(1)[0].cpu().numpy()
    u = np.unique(np.concatenate([[0.0, 1 - 2.0 ** -24], np.float32(w[:-1]) - 2.0 ** -20, np.float32(w[:-1]) + 2.0 ** -20, np.linspace(0, 1, 501)[:-1]]).clip(0, 1 - 2.0 ** -24).astype(np.float32))
    rows = row.expand(len(u), V).contiguous()
    u = torch.from_numpy(u).cuda()
    tokens, probs = ops.sample(rows, u)
    check_draws(tokens, probs, rows, u)
    assert tokens.unique().numel() == V


@pytest.mark.parametrize("V", [5, 600, 3000, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tokens_that_are_equal(ops, V, dtype):
    """All logits alike, or of a few values only: the lower ids come first in what is kept, however many there are."""
    n = 24
    for values in (1, 3):
        rows = (torch.randint(0, values, (n, V), generator=torch.Generator().manual_seed(V)).cuda() * 0.5 - 20).to(dtype)
        kw, u = limits(n, V + values, ks=(2, max(1, V // 3), max(1, V - 1), V, V + 5))
        kw["temperature"] = None
        tokens, probs = ops.sample(rows, u, **kw)
        check_draws(tokens, probs, rows, u, **kw)
    best = ops.sample(torch.zeros(3, V, dtype=dtype, device="cuda"), torch.tensor([0.0, 0.5, 0.999], device="cuda"), temperature=torch.zeros(3, device="cuda"))
    assert best[0].tolist() == [0, 0, 0] and best[1].tolist() == [1.0, 1.0, 1.0]


@pytest.mark.parametrize("n,V", [(150, 70001), (80, 200003), (76, 300001)])
def test_tokens_of_wide_rows_that_are_equal(ops, n, V):
    """More rows than pairs of SMs, so that a row is one CTA's: tens of thousands of equal tokens, in front of the end of top-p and at it."""
    rows = (torch.randint(0, 3, (5, V), generator=torch.Generator().manual_seed(V)).cuda() * 0.5).float()
    rows[3] = 2.0
    rows[4] = rows[4] * 1e-3
    rows = rows.repeat(-(-n // 5), 1)[:n].contiguous()
    g = torch.Generator().manual_seed(n)
    u, p, k = (torch.rand(n, generator=g) for _ in range(3))
    kw = dict(top_p=(0.02 + 0.98 * p).cuda(), top_k=torch.where(k < 0.5, 0, (k * V).int()).to(torch.int32).cuda())
    tokens, probs = ops.sample(rows, u.cuda(), **kw)
    check_draws(tokens, probs, rows, u, **kw)


@pytest.mark.parametrize("n,V", [(2, 9001), (24, 70001), (150, 20010), (80, 60000)])
def test_tokens_where_half_are_masked(ops, n, V):
    """Every other token, or all of a stretch, is -inf: nothing of these may reach a sum, whichever way a step takes the tokens."""
    rows = rnd(n, V, std=1.5, seed=V)
    rows[rnd(n, V, seed=V + 1) > 0] = -float("inf")
    rows[:, V // 3:V // 2] = -float("inf")
    rows[1::2, V // 4:] = torch.finfo(F32).min
    g = torch.Generator().manual_seed(n)
    u, p = torch.rand(n, generator=g), torch.rand(n, generator=g)
    for kw in ({}, {"top_p": 0.5 + 0.5 * p}, {"top_p": 1 - 0.01 * p}, {"top_k": (p * V * 0.3).int() + 600}, {"top_k": (p * V * 0.3).int() + 600, "top_p": 1 - 0.1 * p}, {"min_p": 0.3 * p, "top_p": 0.9 + 0 * p}):
        kw = {name: x.cuda() for name, x in kw.items()}
        tokens, probs = ops.sample(rows, u.cuda(), **kw)
        check_draws(tokens, probs, rows, u, **kw)


@pytest.mark.parametrize("n,V", [(3, 30000), (100, 50001)])
def test_tokens_where_the_nucleus_ends_in_the_tail(ops, n, V):
    """top-p of nearly one, where what is behind the end is counted instead of what is in front, and flat or steep rows, where thousands of tokens lie beside it."""
    g = torch.Generator().manual_seed(n)
    u, p = torch.rand(n, generator=g), torch.rand(n, generator=g)
    for std, t in ((1.0, 1.0), (3.0, 0.5), (6.0, 0.4), (0.001, 1.0), (2.0, 30.0)):
        rows = rnd(n, V, std=std, seed=V)
        for top_p in (1 - 10 ** -(1 + 6 * p), 0.5 + 1e-3 * (p - 0.5)):
            kw = dict(top_p=top_p.float().cuda(), temperature=torch.full((n,), t).cuda())
            tokens, probs = ops.sample(rows, u.cuda(), **kw)
            check_draws(tokens, probs, rows, u, **kw)


def test_tokens_of_rows_with_nothing_or_no_number(ops):
    V = 5000
    inf, nan = float("inf"), float("nan")
    rows = rnd(8, V, seed=2)
    rows[0] = -inf
    rows[1, 4000] = nan
    rows[2] = -inf
    rows[2, 77] = -3.0                              # one token left
    rows[3, 100] = rows[3, 4999] = inf               # two that are everything
    rows[4, ::2] = torch.finfo(F32).min              # masked by the lowest value
    rows[5, 1:] = -inf
    u = torch.full((8,), 0.7, device="cuda")
    kw = dict(top_k=torch.full((8,), 50, dtype=torch.int32, device="cuda"), top_p=torch.full((8,), 0.9, device="cuda"), min_p=torch.full((8,), 0.001, device="cuda"))
    for lim in ({}, kw, {"top_p": kw["top_p"]}, {"top_k": kw["top_k"]}):
        tokens, probs = ops.sample(rows, u, **lim)
        check_draws(tokens, probs, rows, u, **lim)
        assert tokens[:4].tolist() == [-1, -1, 77, 4999] and tokens[5].item() == 0
    bad = torch.tensor([nan, -1.0, inf, 1.0, 1.0, 1.0, 1.0, 1.0], device="cuda")
    fine = rnd(8, V, seed=3)
    tokens, probs = ops.sample(fine, u, temperature=bad)
    assert tokens[:3].tolist() == [-1, -1, -1] and bool(probs[:3].isnan().all()) and bool((tokens[3:] >= 0).all())
    u2 = torch.tensor([nan, -0.5, 1.0, 7.0, inf, 0.0, 0.25, 1 - 2.0 ** -24], device="cuda")
    tokens, probs = ops.sample(fine, u2)
    assert tokens[0].item() == -1 and tokens[1].item() == 0 and tokens[2:5].tolist() == [V - 1] * 3 and tokens[5].item() == 0
    for name in ("top_p", "min_p"):
        x = torch.full((8,), 0.5, device="cuda")
        x[3] = nan
        tokens, probs = ops.sample(fine, u, **{name: x})
        assert tokens[3].item() == -1 and bool(probs[3].isnan()) and bool((tokens[[0, 1, 2, 4, 5, 6, 7]] >= 0).all())


def test_tokens_limits_at_their_ends(ops):
    n, V = 12, 3001
    rows = rnd(n, V, std=2.0, seed=8)
    u = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda()
    one = torch.ones(n, device="cuda")
    for kw in ({"top_p": 0 * one}, {"top_p": -one}, {"top_p": 1e-30 * one}, {"top_p": 2 * one}, {"min_p": one}, {"min_p": 3 * one}, {"min_p": -one}, {"min_p": 1e-30 * one},
               {"top_k": torch.full((n,), -5, dtype=torch.int32, device="cuda")}, {"top_k": torch.full((n,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")},
               {"temperature": 1e-30 * one}, {"temperature": 1e-44 * one}, {"temperature": 1e30 * one}, {"temperature": 3e38 * one, "top_p": 0.5 * one},
               {"top_p": (1 - 2.0 ** -24) * one}, {"top_k": torch.full((n,), V, dtype=torch.int32, device="cuda"), "top_p": 0.999 * one}):
        tokens, probs = ops.sample(rows, u, **kw)
        check_draws(tokens, probs, rows, u, **kw)
    huge = rows * 1e37
    check_draws(*ops.sample(huge, u), huge, u)
    tiny = rows * 1e-42
    check_draws(*ops.sample(tiny, u, top_k=torch.full((n,), 700, dtype=torch.int32, device="cuda")), tiny, u, top_k=torch.full((n,), 700, dtype=torch.int32))


@pytest.mark.parametrize("V", [1000, 65536, 524285])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_tokens_strides_and_places_behind(ops, V, dtype):
    """Rows of a wider tensor on and off boundaries, with NaN beside them; tokens and probs behind the last row stay as they were."""
    n = 5
    for at, gap in ((0, 3), (4, 4), (3, 2)):
        wide = torch.full((n + 1, V + at + gap), float("nan"), dtype=dtype, device="cuda")
        rows = wide[:n, at:at + V]
        rows.copy_(rnd(n, V, std=2.0, dtype=dtype, seed=at))
        kw, u = limits(n, V + at)
        tokens = torch.full((n + 3,), -7, dtype=torch.int32, device="cuda")
        probs = torch.full((n + 3,), -7.0, device="cuda")
        ops.sample(rows, u, **kw, tokens=tokens[:n], probs=probs[:n])
        check_draws(tokens[:n], probs[:n], rows, u, **kw)
        assert tokens[n:].tolist() == [-7] * 3 and probs[n:].tolist() == [-7.0] * 3
    assert ops.sample(rows[:0], u[:0])[0].shape == (0,)


# ---- all of them ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 16, 300])
def test_from_residual_rows_to_tokens(ops, T):
    """The end of a step as a program runs it: norm in 8 bits, the head's product, adjusted logits, tokens; then the whole captured and replayed on other rows."""
    W, V, R = 1024, 5003, 16
    head, hs = ops.to_e4m3(rnd(V, W, std=4 * W ** -0.5, dtype=F16, seed=1), rows=128)
    gain = (1 + rnd(W, std=0.2, seed=2)).to(F16)
    a, b, scale = rnd(2, R, W, std=W ** -0.5, dtype=F16, seed=3), rnd(2, V, R, std=0.2, dtype=F16, seed=4), torch.ones(2, device="cuda")
    index = (torch.arange(T, device="cuda") % 3 - 1).to(torch.int32)
    x, r = rnd(T, W, dtype=F16, seed=5), rnd(T, W, std=3.0, seed=6)
    controls = torch.tensor([[1.1, 0.2, 0.3, 0.99, 1.0]], device="cuda").expand(T, 5).contiguous()
    history, offset = torch.randint(0, V, (T * 4,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda(), (4 * torch.arange(T + 1)).to(torch.int32).cuda()
    kw, u = limits(T, 9)
    logits, total = torch.empty(T, V, device="cuda"), torch.empty_like(r)
    tokens, probs = torch.empty(T, dtype=torch.int32, device="cuda"), torch.empty(T, device="cuda")
    plain = torch.empty(T, W, dtype=F16, device="cuda")

    def step():
        q, s, _ = ops.rms_norm(x, gain, residual=r, out_dtype=E4M3, residual_out=total)
        ops.rms_norm(x, gain, residual=r, out=plain, residual_out=total)
        y = ops.linear_e4m3(q, s, head, hs, out=logits)
        ops.low_rank(plain, a, b, index, scale, base=y, out=y)
        ops.logits(y, "logits", controls=controls, history=history, history_offset=offset, out=y)
        ops.sample(y, u, **kw, tokens=tokens, probs=probs)
        return q, s

    def check(q, s):
        check_norm(ops, x, gain, r, 1e-5, 0.0, E4M3, (q, s, total))
        y = (q.double() * spread(s, 1, q.shape)) @ (head.double() * spread(hs, 128, head.shape)).t()
        for i in range(2):
            y[index == i] += (plain[index == i].double() @ a[i].double().t()) @ b[i].double().t()
        seen = torch.zeros(T, V, dtype=torch.float64, device="cuda")
        weight = seen.clone()
        for j in range(4):
            at = history.view(T, 4)[:, j].long()
            rows = torch.arange(T, device="cuda")
            seen[rows, at] = 1
            weight[rows, at] += controls[0, 3].double() ** (3 - j)
        rep = controls[0, 0].double()
        y = torch.where(seen > 0, torch.where(y > 0, y / rep, y * rep) - controls[0, 1].double() - controls[0, 2].double() * weight, y)
        # (f32 sums of a thousand products of unit size, and adapters whose S is carried in 22 bits)
        assert float((logits.double() - y).abs().max()) <= 2e-4
        check_draws(tokens, probs, logits, u, **kw)

    check(*step())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, s = step()
    x.copy_(rnd(T, W, dtype=F16, seed=15)), r.copy_(rnd(T, W, std=3.0, seed=16)), u.copy_(limits(T, 19)[1])
    for _ in range(2):
        g.replay()
    check(q, s)
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    was = tokens.clone()
    with torch.cuda.stream(s2):
        step()
    s2.synchronize()
    assert torch.equal(tokens, was)


def test_two_streams_at_once(ops):
    """Products, norms and draws of other inputs on two streams side by side have the values of calls alone."""
    T, K, N = 700, 1024, 4000
    made = [make_linear(T, K, N, seed=s) for s in (0, 50)]
    rows = [rnd(64, 40000, std=2.0, seed=s) for s in (1, 2)]
    lim = [limits(64, s) for s in (3, 4)]
    alone = [(ops.linear_e4m3(*m), ops.sample(r, u, **kw), ops.rms_norm(r[:, :5000], None)) for m, r, (kw, u) in zip(made, rows, lim)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                (kw, u) = lim[i]
                got[i].append((ops.linear_e4m3(*made[i]), ops.sample(rows[i], u, **kw), ops.rms_norm(rows[i][:, :5000], None)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, t, q in got[i]:
            assert torch.equal(y, alone[i][0]) and torch.equal(t[0], alone[i][1][0]) and torch.equal(q[0].view(torch.uint8), alone[i][2][0].view(torch.uint8))


def test_tensors_that_do_not_fit(ops):
    x, xs, w, ws = make_linear(4, 64, 40)
    grad = torch.zeros(2, 8, device="cuda", requires_grad=True)
    bad = [
        lambda: ops.to_e4m3(grad), lambda: ops.rms_norm(grad), lambda: ops.sample(grad, torch.zeros(2, device="cuda")),
        lambda: ops.to_e4m3(x), lambda: ops.to_e4m3(torch.zeros(2, 8, device="cuda"), rows=64), lambda: ops.to_e4m3(torch.zeros(2, 8, device="cuda").t()),
        lambda: ops.to_e4m3(torch.zeros(2, 8, device="cuda"), scale=torch.zeros(3, device="cuda")), lambda: ops.to_e4m3(torch.zeros(2, 8, dtype=torch.int32, device="cuda")),
        lambda: ops.rms_norm(torch.zeros(2, 8, device="cuda"), torch.ones(9, device="cuda")), lambda: ops.rms_norm(torch.zeros(2, 8, device="cuda"), torch.ones(8)),
        lambda: ops.rms_norm(torch.zeros(2, 8, dtype=F16, device="cuda"), residual=torch.zeros(2, 8, dtype=BF16, device="cuda")),
        lambda: ops.rms_norm(torch.zeros(2, 8, dtype=F16, device="cuda"), out_dtype=F32), lambda: ops.rms_norm(torch.zeros(2, 32769, device="cuda")),
        lambda: ops.rms_norm(torch.zeros(2, 8, device="cuda"), residual_out=torch.zeros(2, 8, device="cuda")),
        lambda: ops.rms_norm(torch.zeros(2, 8, device="cuda"), out_dtype=F32, scale=torch.zeros(2, device="cuda")),
        lambda: ops.linear_e4m3(x, xs, w[:, :48], ws), lambda: ops.linear_e4m3(x, xs[:3], w, ws), lambda: ops.linear_e4m3(x, xs, w, ws[:0]), lambda: ops.linear_e4m3(x.float(), xs, w, ws),
        lambda: ops.linear_e4m3(x, xs, w, ws, out_dtype=E4M3), lambda: ops.linear_e4m3(x[:, :40], xs, w[:, :40].contiguous(), ws), lambda: ops.linear_e4m3(x[:, 8:], xs, w[:, 8:].contiguous(), ws),
        lambda: ops.linear_e4m3(x, xs, w, ws, base=torch.zeros(4, 40, device="cuda"), out=torch.zeros(4, 40, dtype=F16, device="cuda")),
        lambda: ops.sample(torch.zeros(2, 8, device="cuda"), torch.zeros(3, device="cuda")), lambda: ops.sample(torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.float64)),
        lambda: ops.sample(torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda"), top_k=torch.zeros(2, device="cuda")),
        lambda: ops.sample(torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda"), temperature=torch.ones(2)), lambda: ops.sample(x, torch.zeros(4, device="cuda"))]
    for i, f in enumerate(bad):
        with pytest.raises(capi.B200Error):
            f()
            pytest.fail(f"call {i} was taken")
