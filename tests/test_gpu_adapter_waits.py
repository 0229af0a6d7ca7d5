"""Waits of the adapters' tile kernels that run out: what the wait was for must not leave the kernels as if it were right.  The kernels are compiled for the
test with waits that end and are then told to some threads as lost (adapter_waits.cu)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ai00_server_b200 import build

pytestmark = pytest.mark.gpu

T, N, R = 300, 200, 16                   # 128, 128 and 44 tokens of one adapter; an output of 128 columns and one of 72
LOW, OUT, PRODUCTS = 288, 256, 256       # threads of the two kernels; the thread of the first that issues the products


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("waits") / "waits.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "adapter_waits.cu")
    subprocess.check_call([os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), *build.NVCC_FLAGS, "-shared", src, "-o", so])
    lib = C.CDLL(so)
    lib.waits_workspace.restype = C.c_longlong
    lib.waits_run.argtypes = [C.c_int] * 8 + [C.c_void_p] * 8 + [C.c_int]
    return lib


def run(lib, kernel=0, block=-1, thread=-1, K=512, ctas=4):
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, a, b, base = n(T, K).half(), (n(1, R, K) * K ** -0.5).half(), n(1, N, R).half(), n(T, N)
    index, scale = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda")
    out = torch.zeros(T, N, device="cuda")
    work = torch.empty(lib.waits_workspace(T, 1, R), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.waits_run(kernel, block, thread, T, 1, K, N, R, *(t.data_ptr() for t in (x, a, b, index, scale, base, out, work)), ctas) == 0
    want = base.double() + (x.double() @ a[0].double().T) @ b[0].double().T
    fine = ~out.isnan()
    assert bool(((out.double() - want).abs() <= 1e-3)[fine].all())          # (an eighth of S missing is off by a third: sums of 16 products of unit size)
    return out.isnan()


def test_no_wait_lost(lib):
    assert not run(lib).any()


@pytest.mark.parametrize("thread", [-1, PRODUCTS])
@pytest.mark.parametrize("block", [0, 3, 15, 17])
def test_sums_of_a_tile_with_a_lost_wait(lib, block, thread):
    """All tokens of the tile, whichever of the cluster's CTAs it was: with all of its threads, and with the one that issues the products."""
    nan = run(lib, LOW, block, thread)
    rows = nan.any(1)
    assert torch.equal(rows, nan.all(1))
    assert int(rows.sum()) == (128, 128, 44)[block // 8]


def test_slab_that_waits_for_its_place(lib):
    """A thread that loads the fifth slab of its CTA (40 slabs of 64 over eight) loses the wait for the place of the first: the products of the CTA do not end."""
    nan = run(lib, LOW, 10, 5, K=2560)
    assert torch.equal(nan.any(1), nan.all(1)) and int(nan.any(1).sum()) == 128


@pytest.mark.parametrize("thread", [0, 37, PRODUCTS - 1])
@pytest.mark.parametrize("block", [0, 3, 15, 17])
def test_sums_of_a_thread_with_a_lost_wait(lib, block, thread):
    """The products have ended for all others: the token that the thread hands on (ranks 0 to 15: the first 128 threads one each), and no other."""
    nan = run(lib, LOW, block, thread)
    assert torch.equal(nan.any(1), nan.all(1))
    assert int(nan.any(1).sum()) == (1 if thread < 128 else 0)


@pytest.mark.parametrize("thread", [-1, 0, 5, 255])
@pytest.mark.parametrize("block", [0, 1, 3])
def test_outputs_of_a_cta_with_a_lost_wait(lib, block, thread):
    """All units of the CTA from there on (four CTAs, six units: token tiles by outputs)."""
    nan = run(lib, OUT, block, thread)
    units = [u for u in range(6) if u % 4 == block]
    assert int(nan[:, :128].sum()) == sum((128, 128, 44)[u // 2] * 128 for u in units if u % 2 == 0)
    assert int(nan[:, 128:].sum()) == sum((128, 128, 44)[u // 2] * 72 for u in units if u % 2 == 1)
