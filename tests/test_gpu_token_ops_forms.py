"""Forms of the operators from residual rows to tokens that smaller shapes do not reach: scales of products that come in several pieces, rows far apart, rows one after another in a CTA, draws of a
served model at real width.  Definitions and tolerances are those of test_gpu_token_ops.py."""
import numpy as np
import pytest
import torch

from ai00_server_b200 import capi, runtime, synth
from tests.test_gpu_sample_tokens import check as check_slots
from tests.test_gpu_token_ops import BF16, E4M3, F16, F32, check_draws, check_e4m3, check_linear, check_norm, limits, make_linear, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


# ---- products: scales lie in shared memory for 16 blocks of inputs at a time (32 in the form for 16 tokens) ----
def form(T, K, N, sms):
    """(tokens of the few-token form, or 0 for pairs of SMs; CTAs of a cluster, or tiles; the most blocks of inputs that one CTA adds up), as the call chooses."""
    blocks, tiles = -(-K // 128), lambda t: -(-N // 128) * -(-T // t)

    def split(t, per_sm):
        s = 1
        while s < 8 and tiles(t) * s * 2 <= per_sm * sms and blocks >= s * 8:
            s *= 2
        return s
    for t, per_sm in ((16, 4), (32, 4), (64, 2)):
        if T <= t:
            return t, split(t, per_sm), -(-blocks // split(t, per_sm))
    s, pairs = split(128, 1), -(-T // 256) * -(-N // 256)
    few = -(-tiles(128) * s // sms) * (-(-blocks // s) * 47 + 700)
    return (0, pairs, blocks) if -(-pairs // (sms // 2)) * (blocks * 45 + 270) + 460 < few else (128, s, -(-blocks // s))


def uneven(s, seed):
    """Scales that differ by up to 2^8 from block to block: one that is left from another shows."""
    g = torch.Generator().manual_seed(seed)
    return s * (2.0 ** torch.randint(-4, 5, s.shape, generator=g)).cuda()


@pytest.mark.parametrize("dtype,base", [(F32, False), (BF16, True), (F16, False)])
@pytest.mark.parametrize("T,K,N,want", [
    (5, 34832, 300, 16), (16, 4352, 38020, 16), (20, 17424, 260, 32), (50, 20000, 130, 64), (333, 8960, 2560, 128), (128, 16400, 512, 128),
    (700, 2048, 9999, 0), (600, 2064, 5000, 0), (1024, 2176, 6000, 0), (300, 4096, 12800, 0), (2048, 4224, 10250, 0), (513, 6144, 5122, 0)])
def test_products_of_many_blocks(ops, T, K, N, want, dtype, base):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    took, _, blocks = form(T, K, N, sms)
    if sms == 148:                                   # (the shapes are for that many)
        assert took == want and blocks > (32 if want == 16 else 15)
    x, xs, w, ws = make_linear(T, K, N, seed=T + K)
    xs, ws = uneven(xs, 1), uneven(ws, 2)
    b = rnd(T, N, dtype=dtype, seed=5) if base else None
    out = ops.linear_e4m3(x, xs, w, ws, base=b, out_dtype=None if base else dtype)
    check_linear(out, x, xs, w, ws, b)
    if base:
        assert torch.equal(ops.linear_e4m3(x, xs, w, ws, base=b, out=b), out)


# ---- norms: rows one after another ----
@pytest.mark.parametrize("dtype,res,out", [(BF16, BF16, E4M3), (F32, F32, E4M3), (F16, F32, F16), (BF16, None, E4M3), (F16, F16, E4M3)])
@pytest.mark.parametrize("n,w", [(7301, 8), (2001, 2560), (1100, 4096), (3700, 1001), (1100, 4095)])
def test_norm_of_many_rows_in_place(ops, dtype, res, out, n, w):
    """The sum in place of the residual, and of x, while the next row is on its way: outputs, scales and sums are those of separate buffers, and the last rows' those of a call of their own."""
    x, g = rnd(n, w, std=2.0, dtype=dtype, seed=w), 1 + rnd(w, std=0.3, seed=2)
    r = rnd(n, w, std=5.0, dtype=res, seed=w + 1) if res else None
    same = lambda a, b: all(p is q or torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))  # noqa: E731
    got = ops.rms_norm(x, g, residual=r, out_dtype=out)
    check_norm(ops, x, g, r, 1e-5, 0.0, out, got)
    few = ops.rms_norm(x[-3:], g, residual=None if r is None else r[-3:], out_dtype=out)
    check_norm(ops, x[-3:], g, None if r is None else r[-3:], 1e-5, 0.0, out, few)
    if r is None:
        return
    again = r.clone()
    assert same(ops.rms_norm(x, g, residual=again, out_dtype=out, residual_out=again), got)
    if dtype == res:
        over = x.clone()
        assert same(ops.rms_norm(over, g, residual=r, out_dtype=out, residual_out=over), got)


# ---- rows further apart than 32 bits count ----
STEP = ((1 << 32) // 3 + 4096) & ~15                 # elements between four rows


def far(n, w, dtype, step=STEP, shift=0):
    size = torch.empty((), dtype=dtype).element_size()
    room = torch.empty(((n - 1) * step + w + 64 + shift) * size, dtype=torch.uint8, device="cuda")
    return room.view(dtype)[shift:].as_strided((n, w), (step, 1))


@pytest.mark.parametrize("w,shift", [(256, 0), (301, 3)])
def test_norm_of_far_rows(ops, w, shift):
    x, r = rnd(4, w, dtype=F16, seed=1), rnd(4, w, std=3.0, dtype=F16, seed=2)
    g = 1 + rnd(w, std=0.2, seed=3)
    fx, fr, fo = far(4, w, F16, shift=shift), far(4, w, F16, shift=shift), far(4, w, E4M3, shift=shift)
    fx.copy_(x), fr.copy_(r)
    got = ops.rms_norm(fx, g, residual=fr, out=fo, residual_out=fr)
    check_norm(ops, x, g, r, 1e-5, 0.0, E4M3, (fo.contiguous(), got[1], fr.contiguous()))
    assert torch.equal(fx, x)


@pytest.mark.parametrize("w,shift", [(256, 0), (301, 3)])
def test_8_bits_of_far_rows(ops, w, shift):
    for rows, n, step in ((1, 4, STEP), (128, 130, (1 << 25) + 4096)):
        x = rnd(n, w, dtype=F16, seed=4)
        fx, fo = far(n, w, F16, step, shift), far(n, w, E4M3, step, shift)
        fx.copy_(x)
        _, s = ops.to_e4m3(fx, rows=rows, out=fo)
        check_e4m3(fo.contiguous(), s, x.double(), rows)
        del fx, fo


@pytest.mark.parametrize("shift", [0, 1])
def test_draws_of_far_rows(ops, shift):
    V = 5003
    rows = rnd(4, V, std=2.0, dtype=F16, seed=6)
    fr = far(4, V, F16, shift=shift)
    fr.copy_(rows)
    kw, u = limits(4, 7)
    check_draws(*ops.sample(fr, u, **kw), rows, u, **kw)


# ---- tokens of a served model at real width ----
@pytest.fixture(scope="module")
def model():
    m = runtime.Model(synth.make_st(synth.Shape(6, 1, 256, 896, V=65536, Dm=32, Dd=64), 0), max_batch=16, token_chunk_size=32)
    for s in range(16):
        m.state.load(m.state.init(), s)
    m.rows = np.concatenate(m.infer_raw(list(range(16)), [1] * 16, [17 * s + 1 for s in range(16)], [capi.OPTION_LAST] * 16))
    yield m
    m.close()


@pytest.mark.parametrize("n", [1, 16, 100, 400])
def test_tokens_of_slots_at_real_width(model, n):
    """A cluster a row, a CTA a row, and two CTAs to an SM; slots in any order, several times each."""
    rng = np.random.default_rng(n)
    slots = rng.integers(0, 16, n) if n > 16 else rng.permutation(16)[:n]
    u, t = rng.random(n).astype(np.float32), (0.5 + rng.random(n)).astype(np.float32)
    k, p = (rng.integers(0, 3, n) * 600).astype(np.int32), np.where(rng.random(n) < 0.5, 1.0, rng.random(n)).astype(np.float32)
    t[::5] = 0.0
    rows = model.rows[slots]
    check_slots(model.sample_tokens(slots.tolist(), u, temperature=t, top_k=k, top_p=p), rows, u, t, k, p)
    if n == 16:
        history = [[int(x) for x in rng.integers(0, 65536, 9)] for _ in range(n)]
        controls = np.float32([[1.2, 0.4, 0.3, 0.99, 0.8]] * n)
        adjusted = model.sample_rows(slots.tolist(), "logits", controls=controls, history=history)
        check_slots(model.sample_tokens(slots.tolist(), u, top_k=k, top_p=p, controls=controls, history=history), adjusted, u, 1.0, k, p)
