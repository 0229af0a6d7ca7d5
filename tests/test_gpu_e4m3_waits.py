"""Waits of the 8-bit products' kernels that run out: what the wait was for must not leave the kernels as if it were right, everything else must, and the kernels end.  They are compiled for
the test with waits that end and are then told to some threads as lost (e4m3_waits.cu)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ai00_server_b200 import build

pytestmark = pytest.mark.gpu

K = 2048                                          # 16 blocks of inputs: more than any ring of operands has
FEW, MANY, PAIR = 192, 320, 384                   # threads of the kernel for 16 tokens, for 128, and of the pairs


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("waits") / "waits.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "e4m3_waits.cu")
    subprocess.check_call([os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), *build.NVCC_FLAGS, "-shared", src, "-o", so])
    lib = C.CDLL(so)
    lib.waits_run.argtypes = [C.c_int] * 8 + [C.c_void_p] * 5
    return lib


def run(lib, form, split, T, N, kernel=0, block=-1, thread=-1):
    """Which outputs are NaN; the others are right."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = n(T, K).to(torch.float8_e4m3fn), n(N, K).to(torch.float8_e4m3fn)
    xs, ws = 0.5 + torch.rand(T, K // 128, generator=g, device="cuda"), 0.5 + torch.rand(-(-N // 128), K // 128, generator=g, device="cuda")
    out = torch.zeros(T, N, device="cuda")
    torch.cuda.synchronize()
    assert lib.waits_run(kernel, block, thread, form, split, T, K, N, *(t.data_ptr() for t in (x, xs, w, ws, out))) == 0
    xd, wd = x.double() * xs.double().repeat_interleave(128, 1), w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    nan = out.isnan()
    # (a block of inputs that is missing is off by more than one of some 11; sums of 2048 products of unit size in f32 by 2^-11)
    bound = (4 * 2.0 ** -22 + 32 * 2.0 ** -23) * (xd.abs() @ wd.abs().T)
    assert bool(((out.double() - xd @ wd.T).abs() <= bound)[~nan].all())
    return nan


def columns(nan, at, n):
    """All outputs of these columns are NaN, and no others."""
    want = torch.zeros_like(nan)
    want[:, at:at + n] = True
    return torch.equal(nan, want)


@pytest.mark.parametrize("form,split,T,N", [(16, 4, 10, 300), (16, 1, 16, 128), (128, 1, 100, 300), (128, 2, 128, 260), (256, 2, 300, 600), (256, 1, 256, 256)])
def test_no_wait_lost(lib, form, split, T, N):
    assert not run(lib, form, split, T, N).any()


# of the kernel for 16 tokens: warps 0 to 3 add up, 4 loads, 5 multiplies
@pytest.mark.parametrize("thread", [-1, 0, 77, 127, 128, 141, 160, 191])
@pytest.mark.parametrize("block", [0, 2, 7, 11])
def test_few_tokens(lib, block, thread):
    """Three tiles of 128 outputs, a cluster of four CTAs each: the tile of a CTA with a lost wait."""
    tile = block // 4
    assert columns(run(lib, 16, 4, 10, 300, FEW, block, thread), tile * 128, 128)


# of the kernel for 128: warps 0 to 7 add up, 8 loads, 9 multiplies
@pytest.mark.parametrize("thread", [-1, 5, 255, 256, 270, 288, 300])
@pytest.mark.parametrize("block,split", [(0, 1), (2, 1), (3, 2)])
def test_more_tokens(lib, block, split, thread):
    assert columns(run(lib, 128, split, 100, 300, MANY, block, thread), block // split * 128, 128)


# of the pairs: warps 0 to 7 add up, 8 multiplies (the first CTA's), 9 loads, 10 and 11 load scales.  Two clusters, of which each has three of six tiles: two of tokens by three of outputs
def tiles_of(cluster, shape):
    want = torch.zeros(shape, dtype=torch.bool, device="cuda")
    for u in range(cluster, 6, 2):
        want[u % 2 * 256:u % 2 * 256 + 256, u // 2 * 256:u // 2 * 256 + 256] = True
    return want


@pytest.mark.parametrize("block,thread", [(0, 256), (0, 283), (2, 256), (0, 288), (1, 288), (2, 288), (3, 288), (0, 0), (1, 32), (3, 224), (0, -1), (1, -1), (3, -1)])
def test_pairs(lib, block, thread):
    """The thread that loads or one that multiplies, or one that releases the accumulators of its warp: everything of the cluster from there on, which is all of it."""
    nan = run(lib, 256, 2, 300, 600, PAIR, block, thread)
    assert torch.equal(nan, tiles_of(block // 2, nan.shape))


@pytest.mark.parametrize("block,thread", [(0, 1), (1, 37), (2, 131), (3, 255)])
def test_pairs_one_that_adds_up(lib, block, thread):
    """Its token and half of the columns in every tile of its cluster."""
    nan = run(lib, 256, 2, 300, 600, PAIR, block, thread)
    want = torch.zeros_like(nan)
    row, half = block % 2 * 128 + thread % 128, thread // 128
    for u in range(block // 2, 6, 2):
        want[u % 2 * 256 + row:u % 2 * 256 + row + 1, u // 2 * 256 + half * 128:u // 2 * 256 + half * 128 + 128] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("block,thread", [(0, 320), (1, 340), (2, 383), (3, 352)])
def test_pairs_scales(lib, block, thread):
    """Scales of a tile are a piece of memory of two: the first wait is for the third tile, of which nothing is right any more."""
    nan = run(lib, 256, 2, 300, 600, PAIR, block, thread)
    want = torch.zeros_like(nan)
    u = block // 2 + 4
    want[u % 2 * 256:u % 2 * 256 + 256, u // 2 * 256:u // 2 * 256 + 256] = True
    assert torch.equal(nan, want)


def test_lost_waits_are_counted(lib):
    """One for each thread that lost one, in every kernel; none without."""
    lib.waits_lost.restype = C.c_uint
    before = lib.waits_lost()
    for form, split, T, N, threads, thread in ((16, 4, 10, 300, FEW, 77), (128, 1, 100, 300, MANY, 5), (256, 2, 300, 600, PAIR, 131)):
        run(lib, form, split, T, N)
        assert lib.waits_lost() == before
        run(lib, form, split, T, N, threads, 0, thread)
        assert lib.waits_lost() >= before + 1
        before = lib.waits_lost()


def test_none_in_the_library():
    from ai00_server_b200 import device_ops
    x, w = torch.randn(300, 256, device="cuda"), torch.randn(400, 256, device="cuda")
    device_ops.linear_e4m3(*device_ops.to_e4m3(x), *device_ops.to_e4m3(w, rows=128))
    torch.cuda.synchronize()
    assert device_ops.lost_waits() == 0 and device_ops.lost_waits(0) == 0
