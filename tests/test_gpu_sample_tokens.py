"""Model.sample_tokens: tokens for the slots of a model, drawn on the device from its kept logits rows, against the definition on the rows that infer hands out.  Adjusted
rows are those of sample_rows, to the bit."""
import numpy as np
import pytest

from ai00_server_b200 import capi, runtime, synth
from tests.test_gpu_token_ops import draw_want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    m = runtime.Model(synth.make_st("tiny6", 0), max_batch=4, token_chunk_size=32)
    for s in range(4):
        m.state.load(m.state.init(), s)
    m.rows = np.concatenate(m.infer_raw([0, 1, 2], [4, 1, 3], [1, 5, 9, 33, 7, 2, 7, 300], [capi.OPTION_LAST] * 3))
    yield m
    m.close()


def check(got, rows, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    n = len(rows)
    each = [np.broadcast_to(x, n) for x in (u, temperature, top_k, top_p, min_p)]
    f = lambda x: np.float32(x).item()  # noqa: E731
    want = [draw_want(r, f(each[0][i]), f(each[1][i]), int(each[2][i]), f(each[3][i]), f(each[4][i])) for i, r in enumerate(rows)]
    assert got[0].tolist() == [t for t, _ in want]
    p = np.array([x for _, x in want])
    assert (np.abs(got[1] - p) <= 2.0 ** -23 * p + rows.shape[1] * 2.0 ** -40).all()


def test_rows_as_they_are(model):
    u = np.float32([0.1, 0.5, 0.9])
    check(model.sample_tokens([0, 1, 2], u), model.rows, u)
    check(model.sample_tokens([0, 1, 2], u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.01), model.rows, u, 0.7, 40, 0.9, 0.01)
    check(model.sample_tokens([2, 0, 2, 1], [0.2, 0.3, 0.4, 0.99], temperature=[0, 1.5, 0.2, 1], top_k=[0, 3, 1, 0], top_p=[1, 0.5, 0.3, 0.8]), model.rows[[2, 0, 2, 1]],
          np.float32([0.2, 0.3, 0.4, 0.99]), [0, 1.5, 0.2, 1], [0, 3, 1, 0], [1, 0.5, 0.3, 0.8])
    greedy = model.sample_tokens([0, 1, 2], u, temperature=0.0)
    assert greedy[0].tolist() == model.rows.argmax(1).tolist() and greedy[1].tolist() == [1.0] * 3
    assert greedy[0].tolist() == model.sample_topk([0, 1, 2], top_k=1)[0][:, 0].tolist()
    assert model.sample_tokens([], [])[0].shape == (0,)


def test_rows_adjusted(model):
    V = model.info["num_vocab"]
    u = np.float32([0.3, 0.6, 0.8])
    controls = np.float32([[1.2, 0.4, 0.3, 0.99, 0.8]] * 3)
    history = [[1, 5, 9, 33], [], [7, 7, 300]]
    allow = np.random.default_rng(0).random((3, V)) < 0.4
    allow[2] = False
    allow[2, 11] = True
    bias = [{3: 2.0}, None, {11: -1.0}]
    for kw in ({"controls": controls, "history": history}, {"allow": allow}, {"bias": bias}, {"controls": controls, "history": history, "history_from": [2, 0, 1], "allow": allow, "bias": bias}):
        rows = model.sample_rows([0, 1, 2], "logits", **kw)
        got = model.sample_tokens([0, 1, 2], u, top_p=0.95, **kw)
        check(got, rows, u, top_p=np.float32(0.95))
        if "allow" in kw:
            assert got[0][2] == 11 and all(allow[i, t] for i, t in enumerate(got[0]))
    none = model.sample_tokens([0], [0.5], allow=np.zeros((1, V), bool))
    assert none[0].tolist() == [-1] and none[1].tolist() == [0.0]


def test_generation_follows_the_rows(model):
    """A few tokens of a prompt's continuation, each drawn on the device and fed back; the rows go nowhere else."""
    s = 3
    model.state.load(model.state.init(), s)
    toks, rng = [4, 8], np.random.default_rng(2)
    rows = model.infer_raw([s], [2], toks, [capi.OPTION_LAST])[0]
    for _ in range(6):
        u = np.float32(rng.random())
        t, p = model.sample_tokens([s], [u], temperature=0.9, top_k=30, top_p=0.9)
        check((t, p), rows, u, np.float32(0.9), 30, np.float32(0.9))
        rows = model.infer_raw([s], [1], [int(t[0])], [capi.OPTION_LAST])[0]
    model.state.load(model.state.init(), s)


def test_refusals(model):
    bad = [dict(uniform=[1.0]), dict(uniform=[-0.1]), dict(uniform=[float("nan")]), dict(uniform=[0.5, 0.5]), dict(uniform=0.5), dict(uniform=[0.5], temperature=-1.0),
           dict(uniform=[0.5], temperature=float("inf")), dict(uniform=[0.5], top_p=float("nan")), dict(uniform=[0.5], min_p=float("nan")), dict(uniform=[0.5], top_k=[1, 2]),
           dict(uniform=[0.5], controls=np.float32([[0, 0, 0, 1, 1]])), dict(uniform=[0.5], history=[[1], [2]])]
    for kw in bad:
        with pytest.raises(capi.B200Error) as ei:
            model.sample_tokens([0], **kw)
        assert ei.value.code == capi.ERR_INVALID
    for slot in (3 + 1, -1):
        with pytest.raises(capi.B200Error) as ei:
            model.sample_tokens([slot], [0.5])
        assert ei.value.code == capi.ERR_STATE
    fresh = runtime.Model(synth.make_st("tiny6", 0), max_batch=1, token_chunk_size=16)
    with pytest.raises(capi.B200Error) as ei:
        fresh.sample_tokens([0], [0.5])
    assert ei.value.code == capi.ERR_STATE
    fresh.close()
