"""Limits that end among hundreds of equal logits (device_ops.sample): the end is one of them, found by its id, and every warp of the row has to take the same one before any goes on to
sum up what is kept.  Draws are the definition's, and the same in every run."""
import pytest
import torch

from tests.test_gpu_token_ops import check_draws

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


def flat_rows(n, V, seed):
    """A tenth of the tokens above a level that a third is on; of the rest half are masked.  Of neighbouring 128, mostly fewer than 64 are kept."""
    g = torch.Generator().manual_seed(seed)
    kind = torch.rand(n, V, generator=g)
    rows = torch.full((n, V), -7.0)
    rows[kind < 0.4] = 0.25
    rows[kind < 0.1] = 1.0
    rows[kind > 0.7] = -float("inf")
    return rows.cuda(), torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g)


@pytest.mark.parametrize("n,V", [(1, 9000), (5, 30000), (40, 20011), (160, 9001), (300, 40000)])
@pytest.mark.parametrize("limit", ["k", "p", "kp", "km"])
def test_the_end_is_one_of_many(ops, n, V, limit):
    rows, u, r = flat_rows(n, V, n + V)
    # the level is between a tenth and four of the tokens, and between 41 and 99 hundredths of the weights
    kw = {}
    if "k" in limit:
        kw["top_k"] = ((0.12 + 0.25 * r) * V).to(torch.int32).cuda()
    if "p" in limit:
        kw["top_p"] = (0.55 + 0.4 * r).cuda()
    if "m" in limit:
        kw["min_p"] = torch.full((n,), 0.01, device="cuda")
    tokens, probs = ops.sample(rows, u, **kw)
    check_draws(tokens, probs, rows, u, **kw)
    for _ in range(60):
        again = ops.sample(rows, u, **kw)
        assert torch.equal(again[0], tokens) and torch.equal(again[1], probs)
