"""Operators on device memory (ai00_server_b200.device_ops) against their definitions in 64 bits, at the sizes, masks and layouts where they can go
wrong.

Tolerances.  Adapters: products of two 16-bit numbers are exact in f32; a step of 16 of them and the running sum is off by at most 2^-22 of the sum of
magnitudes so far, whatever the order of the parts, and there are K / 16 steps in a row at most, and some dozens of sums over warps and CTAs.  The
second product takes S in parts that leave 2^-21 (f16) or 2^-16 (bf16, for bf16 outputs; 2^-23 for f32 ones) of a token's largest.  The result is
rounded once: half a step of its type.  Logits: an f32 operation is off by 2^-24 of its result; the exponential by 2^-22, beside the
rounding of its argument, |l - max| 2^-23."""
import numpy as np
import pytest
import torch

from ai00_server_b200 import capi

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from ai00_server_b200 import device_ops
    return device_ops


def rnd(*shape, std=1.0, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def adapter_want(x, a, b, index, scale, base, out_dtype):
    """(values in 64 bits, bound of the error) of one part."""
    T, K, R, N = x.shape[0], x.shape[1], a.shape[1], b.shape[1]
    y = base.double().clone() if base is not None else torch.zeros(T, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(y)
    part = 2.0 ** (-21 if x.dtype == F16 else (-23 if out_dtype == F32 else -16))
    for i in range(a.shape[0]):
        t = (index == i).nonzero()[:, 0]
        if not t.numel():
            continue
        xd, ad, bd, s = x[t].double(), a[i].double(), b[i].double(), abs(float(scale[i]))
        low = xd @ ad.t()
        y[t] += float(scale[i]) * (low @ bd.t())
        e_low = (K / 16 + 64) * 2.0 ** -22 * (xd.abs() @ ad.abs().t()) + part * low.abs().amax(1, keepdim=True)
        err[t] = s * (e_low @ bd.abs().t() + (R / 16 + 8) * 2.0 ** -22 * (low.abs() @ bd.abs().t()))
    half = torch.finfo(out_dtype).eps / 2
    err = err * (1 + half) + half * y.abs() * (index_served(index, a.shape[0])[:, None] | (base is None)) + 2.0 ** -24 * y.abs()
    return y, err


def index_served(index, n):
    return (index >= 0) & (index < n)


def check_adapters(out, want, err):
    bad = (out.double() - want).abs() > err + 1e-30
    assert not bool(bad.any()), (int(bad.sum()), float(((out.double() - want).abs() / (err + 1e-30)).max()))


def make(T, K, N, R, n, dtype, out_dtype, base=True, seed=0):
    x = rnd(T, K, dtype=dtype, seed=seed)
    a = rnd(n, R, K, std=K ** -0.5, dtype=dtype, seed=seed + 1)
    b = rnd(n, N, R, std=0.3, dtype=dtype, seed=seed + 2)
    scale = 0.25 + rnd(n, seed=seed + 3).abs()
    y = rnd(T, N, dtype=out_dtype, seed=seed + 4) if base else None
    return x, a, b, scale, y


def indices(T, n, how, seed=0):
    g = torch.Generator().manual_seed(seed)
    if how == "one":
        i = torch.full((T,), n - 1)
    elif how == "distinct":
        i = torch.arange(T) % n
    elif how == "runs":
        i = torch.sort(torch.randint(0, n, (T,), generator=g)).values
    elif how == "none":
        i = torch.full((T,), -1)
    else:                                        # any order, some without, some out of range
        i = torch.randint(-2, n + 2, (T,), generator=g)
    return i.to(torch.int32).cuda()


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("T,K,N,R,n,how", [
    (1, 8, 1, 8, 1, "one"), (1, 2048, 2048, 16, 4, "one"), (2, 40, 5, 8, 3, "distinct"), (7, 264, 31, 24, 2, "mixed"), (8, 64, 100, 16, 1, "one"),
    (9, 520, 513, 32, 1, "one"), (16, 2560, 640, 16, 8, "mixed"), (17, 1024, 96, 72, 17, "distinct"), (33, 136, 257, 128, 5, "mixed"),
    (64, 512, 300, 8, 64, "distinct"), (100, 96, 64, 256, 3, "runs"), (256, 256, 128, 40, 20, "mixed"), (257, 256, 130, 40, 20, "mixed"),
    (300, 72, 33, 16, 1024, "mixed"), (513, 1000, 257, 24, 3, "runs"), (1000, 320, 384, 64, 7, "mixed"), (777, 128, 64, 8, 2, "none"),
    (2048, 256, 512, 64, 4, "runs"), (3001, 64, 72, 16, 300, "mixed"), (640, 264, 1028, 200, 2, "runs")])
def test_adapters_against_64_bits(ops, dtype, out_dtype, T, K, N, R, n, how):
    x, a, b, scale, y = make(T, K, N, R, n, dtype, out_dtype)
    index = indices(T, n, how)
    out = ops.low_rank(x, a, b, index, scale, base=y)
    want, err = adapter_want(x, a, b, index, scale, y, out_dtype)
    check_adapters(out, want, err)
    plain = ~index_served(index, n)
    assert torch.equal(out[plain], y[plain])                     # tokens without an adapter: the base, to the bit
    again = ops.low_rank(x, a, b, index, scale, base=y)
    assert torch.equal(out, again)


@pytest.mark.parametrize("T,n,how", [(8193, 1024, "mixed"), (20000, 3, "mixed"), (33000, 1000, "runs"), (1 << 20, 5, "mixed")])
def test_adapters_of_very_long_calls(ops, T, n, how):
    """More tokens than the order keeps bins for, more tiles than a CTA keeps places of; the largest call."""
    x, a, b, scale, y = make(T, 8, 4, 8, n, F16, F32)
    index = indices(T, n, how)
    out = ops.low_rank(x, a, b, index, scale, base=y)
    check_adapters(out, *adapter_want(x, a, b, index, scale, y, F32))


@pytest.mark.parametrize("T", [4, 260])
def test_adapters_rows_far_apart(ops, T):
    """Rows of x, base and out further from each other than 32 bits count elements."""
    K, N, n = 64, 40, 3
    step = ((1 << 32) // (T - 1) + 4096) & ~7
    x, a, b, scale, y = make(T, K, N, 16, n, F16, F16)
    far = [torch.empty((T - 1) * step + 64, dtype=F16, device="cuda").as_strided((T, w), (step, 1)) for w in (K, N, N)]
    far[0].copy_(x)
    far[1].copy_(y)
    index = indices(T, n, "mixed")
    ops.low_rank(far[0], a, b, index, scale, base=far[1], out=far[2])
    check_adapters(far[2].contiguous(), *adapter_want(x, a, b, index, scale, y, F16))


@pytest.mark.parametrize("T,n", [(5, 3), (300, 9), (700, 2)])
def test_adapters_without_a_base_and_in_place(ops, T, n):
    x, a, b, scale, y = make(T, 200, 76, 24, n, F16, F32)
    index = indices(T, n, "mixed")
    out = ops.low_rank(x, a, b, index, scale, out_dtype=F32)
    want, err = adapter_want(x, a, b, index, scale, None, F32)
    check_adapters(out, want, err)
    assert not out[~index_served(index, n)].any()
    want, err = adapter_want(x, a, b, index, scale, y, F32)
    assert ops.low_rank(x, a, b, index, scale, base=y, out=y) is y
    check_adapters(y, want, err)


@pytest.mark.parametrize("T", [3, 40, 600])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_adapters_strides_and_rows_behind(ops, T, out_dtype):
    """x, base and out as columns of wider tensors (base and out at odd offsets); what lies beside and behind stays as it was."""
    n, K, N = 4, 136, 53
    x, a, b, scale, _ = make(T, K, N, 16, n, BF16, out_dtype)
    wide_x = torch.full((T + 2, K + 24), float("nan"), dtype=BF16, device="cuda")
    wide_x[:T, 8:8 + K] = x
    wide_y = rnd(T + 1, N + 6, dtype=out_dtype, seed=9)
    wide_o = torch.full((T + 3, N + 11), 7.0, dtype=out_dtype, device="cuda")
    index = indices(T, n, "mixed")
    ops.low_rank(wide_x[:T, 8:8 + K], a, b, index, scale, base=wide_y[:T, 3:3 + N], out=wide_o[:T, 5:5 + N])
    want, err = adapter_want(x, a, b, index, scale, wide_y[:T, 3:3 + N], out_dtype)
    check_adapters(wide_o[:T, 5:5 + N], want, err)
    keep = torch.ones_like(wide_o, dtype=torch.bool)
    keep[:T, 5:5 + N] = False
    assert bool((wide_o[keep] == 7.0).all())


@pytest.mark.parametrize("T", [1, 12, 400])
def test_adapters_several_projections_at_once(ops, T):
    """Parts of other widths and ranks in one call have the values of calls of their own."""
    n = 5
    sizes = [(256, 300, 16), (256, 64, 64), (72, 8, 8), (1000, 131, 40)]
    made = [make(T, K, N, R, n, F16, F16, seed=10 * i) for i, (K, N, R) in enumerate(sizes)]
    index, scale = indices(T, n, "mixed"), made[0][3]
    outs = ops.low_rank([m[0] for m in made], [m[1] for m in made], [m[2] for m in made], index, scale, base=[m[4] for m in made])
    for o, (x, a, b, _, y) in zip(outs, made):
        want, err = adapter_want(x, a, b, index, scale, y, F16)
        check_adapters(o, want, err)
        assert torch.equal(o, ops.low_rank(x, a, b, index, scale, base=y))


@pytest.mark.parametrize("T", [1, 12, 301])
def test_adapters_columns_of_one_buffer(ops, T):
    """x and the outputs of three projections as columns side by side of one buffer, in place: what each adds is what it adds to rows of its own."""
    n, K, widths = 5, 128, (40, 131, 64)
    made = [make(T, K, N, 16, n, F16, F16, seed=10 * i) for i, N in enumerate(widths)]
    index, scale, x = indices(T, n, "mixed"), made[0][3], made[0][0]
    wide = torch.full((T + 1, K + sum(widths) + 5), 7.0, dtype=F16, device="cuda")
    wide[:T, :K] = x
    at = K
    outs = []
    for N, m in zip(widths, made):
        outs.append(wide[:T, at:at + N])
        outs[-1].copy_(m[4])
        at += N
    ops.low_rank([wide[:T, :K]] * 3, [m[1] for m in made], [m[2] for m in made], index, scale, base=outs, out=outs)
    for o, m in zip(outs, made):
        check_adapters(o, *adapter_want(x, m[1], m[2], index, scale, m[4], F16))
    assert torch.equal(wide[:T, :K], x) and bool((wide[:T, at:] == 7.0).all()) and bool((wide[T] == 7.0).all())
    with pytest.raises(capi.B200Error):
        ops.low_rank([wide[:T, :K]] * 3, [m[1] for m in made], [m[2] for m in made], index, scale, out=[outs[0], outs[1], wide[:T, at - 65:at - 1]])


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("T,n,how", [(257, 5, "mixed"), (258, 3, "runs"), (259, 40, "tail"), (333, 4, "runs"), (1021, 70, "tail"), (1022, 6, "mixed"), (1023, 2, "one")])
def test_adapters_several_projections_of_ragged_prompts(ops, dtype, out_dtype, T, n, how):
    """Token counts that are no multiples of four or sixteen, through projections of other widths and ranks in one call: the values of calls of their own, to the
    bit.  "tail": more adapters than tokens allow tiles for all of, most tokens with one of them, the others few each."""
    sizes = [(136, 300, 16), (256, 64, 72), (72, 8, 8), (200, 131, 40)]
    if how == "tail":
        index = indices(T, n, "mixed")
        index[torch.arange(T, device="cuda") % 5 != 0] = 1
    else:
        index = indices(T, n, how)
    for base in (True, False):
        made = [make(T, K, N, R, n, dtype, out_dtype, base=base, seed=10 * i) for i, (K, N, R) in enumerate(sizes)]
        scale = made[0][3]
        outs = ops.low_rank([m[0] for m in made], [m[1] for m in made], [m[2] for m in made], index, scale, base=[m[4] for m in made] if base else None, out_dtype=out_dtype)
        for o, (x, a, b, _, y) in zip(outs, made):
            want, err = adapter_want(x, a, b, index, scale, y, out_dtype)
            check_adapters(o, want, err)
            assert torch.equal(o, ops.low_rank(x, a, b, index, scale, base=y, out_dtype=out_dtype))


def test_adapters_bad_values_stay_with_their_token(ops):
    T, n = 300, 3
    for count in (20, T):
        x, a, b, scale, y = make(count, 128, 96, 32, n, F16, F32)
        index = indices(count, n, "runs")
        clean = ops.low_rank(x, a, b, index, scale, base=y)
        x[3, 5], x[7, 100], x[11, 0] = float("nan"), float("inf"), 60000.0
        a[2, 4, 9] = 1.0
        out = ops.low_rank(x, a, b, torch.where(index == 2, -1, index).to(torch.int32), scale, base=y)
        assert bool(out[3].isnan().all()) and not bool(out[7].isfinite().any())
        others = torch.ones(count, dtype=torch.bool, device="cuda")
        others[[3, 7, 11]] = False
        others &= index != 2
        assert torch.equal(out[others], clean[others])


def test_adapters_large_and_small_magnitudes(ops):
    """S beyond f16's range and far below its smallest number."""
    T, K, N, R, n = 9, 64, 40, 8, 2
    x, a, b, scale, _ = make(T, K, N, R, n, F16, F32)
    for f in (3e3, 2e-4):
        xs, as_ = (x.float() * f).to(F16), (a.float() * f).to(F16)
        index = indices(T, n, "distinct")
        out = ops.low_rank(xs, as_, b, index, scale, out_dtype=F32)
        want, err = adapter_want(xs, as_, b, index, scale, None, F32)
        check_adapters(out, want, err)


def test_adapters_no_tokens(ops):
    x, a, b, scale, y = make(0, 64, 32, 8, 2, F16, F32)
    out = ops.low_rank(x, a, b, indices(0, 2, "one"), scale, base=y)
    assert out.shape == (0, 32)


@pytest.mark.parametrize("T", [6, 400])
def test_adapters_graph_and_stream(ops, T):
    """Captured once, replayed with other inputs and other adapters for the tokens; a call on a stream of its own."""
    n = 4
    x, a, b, scale, y = make(T, 256, 160, 16, n, F16, F32)
    index = indices(T, n, "mixed")
    out = torch.empty_like(y)
    ops.low_rank(x, a, b, index, scale, base=y, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.low_rank(x, a, b, index, scale, base=y, out=out)
    x2, _, _, _, y2 = make(T, 256, 160, 16, n, F16, F32, seed=50)
    i2 = indices(T, n, "mixed", seed=3)
    x.copy_(x2), y.copy_(y2), index.copy_(i2)
    for _ in range(2):
        g.replay()
    want, err = adapter_want(x2, a, b, i2, scale, y2, F32)
    check_adapters(out, want, err)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2 = ops.low_rank(x, a, b, index, scale, base=y)
    s.synchronize()
    assert torch.equal(o2, out)


def test_adapters_two_graphs_side_by_side(ops):
    """Two captured calls that need a plan, replayed on two streams at once."""
    T, n = 600, 6
    made = [make(T, 256, 256, 16, n, F16, F32, seed=s) for s in (0, 100)]
    idx = [indices(T, n, "mixed", seed=s) for s in (1, 2)]
    outs, graphs = [torch.empty_like(m[4]) for m in made], []
    for m, i, o in zip(made, idx, outs):
        ops.low_rank(m[0], m[1], m[2], i, m[3], base=m[4], out=o)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.low_rank(m[0], m[1], m[2], i, m[3], base=m[4], out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for m, i, o in zip(made, idx, outs):
        want, err = adapter_want(m[0], m[1], m[2], i, m[3], m[4], F32)
        check_adapters(o, want, err)


# ---------------------------------------------------------------------------------------------------------------------------------------------
def logits_want(rows, kind, controls=None, histories=None, history_from=None, biases=None, masks=None, mask_of=None):
    """(values in 64 bits, bound) row by row from the definition; histories, biases: lists of lists."""
    l = rows.detach().double().cpu().numpy().copy()
    n, V = l.shape
    err = np.zeros_like(l)
    for i in range(n):
        rep, presence, frequency, decay, temperature = controls[i].double().cpu().tolist() if controls is not None else (1, 0, 0, 1, 1)
        r, e = l[i], err[i]
        if histories is not None:
            h = [t for t in histories[i]]
            first = history_from[i] if history_from is not None else 0
            weight, w_off, said = {}, {}, set()
            for j, t in enumerate(h):
                if j >= first and 0 <= t < V:
                    said.add(t)
                    age = len(h) - 1 - j
                    w = decay ** age if age else 1.0
                    weight[t] = weight.get(t, 0.0) + w
                    # 2^(age log2 decay): the exponent is off by two steps of its size, the power by four of its own
                    w_off[t] = w_off.get(t, 0.0) + w * 2.0 ** -22 * (2 + age * abs(np.log2(decay)))
            for t in set(t for t in h if 0 <= t < V):
                r[t] = r[t] / rep if r[t] > 0 else r[t] * rep
                down = (presence + frequency * weight[t]) if t in said else 0.0
                # presence and frequency may have opposite signs: what rounds is each of the two summands, not their sum
                size = abs(presence) + abs(frequency) * weight.get(t, 0.0)
                e[t] += 2.0 ** -23 * abs(r[t]) + 2.0 ** -22 * size + abs(frequency) * w_off.get(t, 0.0) + 2.0 ** -23 * abs(r[t] - down)
                r[t] -= down
        if biases is not None:
            for t, v in dict(biases[i]).items():
                if 0 <= t < V:
                    r[t] += v
                    e[t] += 2.0 ** -23 * abs(r[t])
        m = mask_of[i] if mask_of is not None else i
        if masks is not None and 0 <= m < len(masks):
            r[~masks[m]] = -np.inf
            e[~masks[m]] = 0
        r /= temperature
        e /= temperature
        with np.errstate(invalid="ignore"):
            e += 2.0 ** -22 * np.abs(np.where(np.isfinite(r), r, 0))
        if kind != "logits":
            top = r.max()
            if top == -np.inf:
                l[i] = 0.0 if kind == "probs" else -np.inf
                continue
            with np.errstate(invalid="ignore"):
                d = r - top
                x = np.exp(d)
                z = x.sum()
                off = e + np.nanmax(np.where(np.isfinite(r), e, 0)) + 2.0 ** -22 * (1 + np.abs(np.where(np.isfinite(d), d, 0)))      # of the exponent
                z_off = float((x * off).sum() / z) + 2.0 ** -20
                if kind == "probs":
                    l[i], err[i] = x / z, (x / z) * (off + z_off) + 1e-38
                else:
                    l[i], err[i] = d - np.log(z), off + z_off + 2.0 ** -22 * np.abs(np.where(np.isfinite(d), d, 0))
    return l, err


def check_logits(out, want, err):
    o = out.double().cpu().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(o), np.isnan(want))
    assert np.array_equal(o[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(o[fine] - want[fine])
    assert (off <= err[fine]).all(), float((off / err[fine]).max())


def ragged(lists, dtype=torch.int32):
    off = np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)
    flat = [v for x in lists for v in x]
    return torch.from_numpy(off).cuda(), torch.tensor(flat, dtype=dtype).cuda()


def pack(masks):
    m, V = masks.shape
    words = (V + 31) // 32
    full = np.zeros((m, words * 32), bool)
    full[:, :V] = masks
    return torch.from_numpy(np.packbits(full.reshape(m, words, 32), axis=2, bitorder="little").view(np.int32).reshape(m, words).copy()).cuda()


def logits_case(n, V, dtype, longest, mask_share, bias, seed, std=3.0):
    r = np.random.default_rng(seed)
    rows = rnd(n, V, std=std, dtype=dtype, seed=seed)
    controls = torch.tensor(np.stack([r.uniform(0.8, 1.5, n), r.uniform(-0.3, 0.8, n), r.uniform(-0.2, 0.8, n), r.uniform(0.9, 1.0, n),
                                      r.uniform(0.5, 2.0, n)], 1), dtype=F32).cuda()
    lens = [0 if i % 4 == 3 else int(r.integers(1, longest + 1)) for i in range(n)] if longest else [0] * n
    lens[0] = longest
    # small ids come often; some tokens that the vocabulary does not have
    histories = [[int(t) if r.random() > 0.02 else int(r.choice([-1, V, V + 7, 2 ** 31 - 1])) for t in (V * r.random(m) ** 5).astype(int)] for m in lens]
    froms = [int(r.integers(0, m + 2)) for m in lens]
    biases = [[(int(t), float(np.float32(v))) for t, v in zip(r.integers(-1, V + 1, k), r.normal(0, 4, k))] for k in [bias if i % 3 else bias // 2 for i in range(n)]]
    masks = r.random((max(1, n // 2), V)) < mask_share if mask_share is not None else None
    mask_of = [int(r.integers(-1, masks.shape[0] + 1)) for _ in range(n)] if masks is not None else None
    return rows, controls, histories, froms, biases, masks, mask_of


def call(ops, rows, kind, controls, histories, froms, biases, masks, mask_of, **more):
    kw = {}
    if histories is not None:
        kw["history_offset"], kw["history"] = ragged(histories)
        kw["history_from"] = torch.tensor(froms, dtype=torch.int32).cuda() if froms is not None else None
    if biases is not None:
        kw["bias_offset"], kw["bias_token"] = ragged([[t for t, _ in b] for b in biases])
        kw["bias_value"] = torch.tensor([v for b in biases for _, v in b], dtype=F32).cuda()
    if masks is not None:
        kw["allow"] = pack(masks)
        kw["allow_row"] = torch.tensor(mask_of, dtype=torch.int32).cuda() if mask_of is not None else None
    return ops.logits(rows, kind=kind, controls=controls, **kw, **more)


@pytest.mark.parametrize("kind", ["logits", "probs", "log_probs"])
@pytest.mark.parametrize("n,V,dtype,longest,mask_share,bias", [
    (1, 1, F32, 3, None, 2), (1, 2, F32, 0, 0.5, 0), (2, 31, F16, 9, 0.5, 4), (3, 33, F32, 40, 0.3, 10), (5, 257, BF16, 300, 0.1, 40),
    (2, 1000, F32, 0, None, 0), (4, 2048, F32, 1000, 0.5, 100), (3, 4099, F16, 2500, 0.01, 3), (2, 32000, F32, 500, 0.7, 300),
    (2, 65536, F32, 4000, 0.5, 50), (1, 65536, BF16, 0, 0.001, 0), (1, 100003, F32, 9000, 0.6, 200), (1, 262147, BF16, 700, 0.5, 30)])
def test_logits_against_64_bits(ops, kind, n, V, dtype, longest, mask_share, bias):
    case = logits_case(n, V, dtype, longest, mask_share, bias, seed=V + n)
    rows, controls, histories, froms, biases, masks, mask_of = case
    out = call(ops, rows, kind, controls, histories, froms, biases, masks, mask_of)
    want, err = logits_want(rows, kind, controls, histories, froms, biases, masks, mask_of)
    check_logits(out, want, err)
    assert torch.equal(out, call(ops, rows, kind, controls, histories, froms, biases, masks, mask_of))       # the atomics' order changes nothing


def test_logits_wider_than_shared_memory(ops):
    """A vocabulary of which an eighth does not fit a CTA's shared memory."""
    V = 460001
    for kind in ("logits", "probs", "log_probs"):
        case = logits_case(2, V, F32, 3000, 0.5, 30, seed=1)
        out = call(ops, case[0], kind, *case[1:])
        want, err = logits_want(case[0], kind, *case[1:])
        check_logits(out, want, err)


@pytest.mark.parametrize("kind", ["logits", "probs", "log_probs"])
@pytest.mark.parametrize("V,stride", [(524287, 524287), (524286, 524289), (524288, 524291), (524288, 524288), (524285, 524285)])
def test_logits_widest_rows_off_boundaries(ops, kind, V, stride):
    """The widest vocabularies, rows that start up to three tokens behind a boundary: their last tokens are written, count in the sums and take their lists."""
    n = 4
    rows = torch.empty(n * stride, device="cuda").as_strided((n, V), (stride, 1))
    rows.copy_(rnd(n, V, seed=V % 97))
    rows[:, V - 3:] += 12.0                              # the last tokens are most of a row
    out = torch.full((n * stride,), float("nan"), device="cuda").as_strided((n, V), (stride, 1))
    _, controls, _, _, _, _, _ = logits_case(n, 8, F32, 0, None, 0, seed=3)
    histories = [[V - 1, 5, V - 1], [], [V - 2, V - 1], [V - 3] * 4]
    biases = [[(V - 1, 1.5)], [(V - 2, -2.0), (0, 3.0)], [], [(V - 1, 0.25), (V - 3, 4.0)]]
    call(ops, rows, kind, controls, histories, None, biases, None, None, out=out)
    want, err = logits_want(rows, kind, controls, histories, None, biases)
    check_logits(out, want, err)
    if stride > V:
        assert bool(torch.as_strided(out, (n - 1, stride - V), (stride, 1), V).isnan().all())


@pytest.mark.parametrize("kind", ["logits", "probs", "log_probs"])
def test_logits_parts_alone(ops, kind):
    """Histories, biases and masks each without the others; no controls at all."""
    rows, controls, histories, froms, biases, masks, mask_of = logits_case(4, 5000, F32, 200, 0.4, 50, seed=5)
    for args in [(None, None, None, None, None, None), (controls, None, None, None, None, None), (controls, histories, None, None, None, None),
                 (controls, histories, froms, None, None, None), (None, None, None, biases, None, None), (None, None, None, None, masks, mask_of),
                 (None, histories, froms, biases, None, None)]:
        out = call(ops, rows, kind, *args)
        want, err = logits_want(rows, kind, *args)
        check_logits(out, want, err)


@pytest.mark.parametrize("kind", ["probs", "log_probs"])
def test_logits_rows_with_nothing_left(ops, kind):
    V = 3001
    rows = rnd(4, V, seed=2)
    masks = np.zeros((4, V), bool)
    masks[1, 1500] = True                        # one token left
    masks[3] = True
    rows[3] = -float("inf")                      # allowed, but impossible
    out = ops.logits(rows, kind=kind, allow=pack(masks))
    zero, one = (0.0, 1.0) if kind == "probs" else (-float("inf"), 0.0)
    assert bool((out[0] == zero).all()) and bool((out[2] == zero).all()) and bool((out[3] == zero).all())
    assert float(out[1, 1500]) == one and bool((out[1, :1500] == zero).all()) and bool((out[1, 1501:] == zero).all())


def test_logits_masked_values_do_not_matter(ops):
    """The lowest value of the type, infinities and NaN in masked places."""
    V = 20000
    for dtype in (F32, F16, BF16):
        rows = rnd(2, V, dtype=dtype, seed=3)
        keep = np.random.default_rng(0).random((2, V)) < 0.3
        want = {k: ops.logits(rows, kind=k, allow=pack(keep)) for k in ("logits", "probs", "log_probs")}
        gone = torch.from_numpy(~keep).cuda()
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max], dtype=dtype, device="cuda")
        dirty = torch.where(gone, junk[torch.arange(2 * V, device="cuda").view(2, V) % 5], rows)
        for k, w in want.items():
            assert torch.equal(ops.logits(dirty, kind=k, allow=pack(keep)), w)
        # the lowest value itself as a mask: vanishes from the probabilities
        low = torch.where(gone, torch.finfo(dtype).min, rows)
        assert torch.equal(ops.logits(low, kind="probs"), want["probs"])
    # a NaN that is left reaches its row alone
    rows = rnd(3, V, seed=4)
    rows[1, 777] = float("nan")
    for k in ("probs", "log_probs"):
        out = ops.logits(rows, kind=k)
        assert bool(out[1].isnan().all()) and not bool(out[[0, 2]].isnan().any())


def test_logits_a_row_of_large_values(ops):
    rows = torch.full((1, 70000), 3e38, device="cuda")
    rows[0, 5] = 3.2e38
    out = ops.logits(rows, kind="probs")
    assert float(out[0, 5]) == 1.0 and float(out.sum()) == 1.0
    rows = torch.full((1, 70000), -3e38, device="cuda")
    out = ops.logits(rows, kind="probs")
    assert bool(((out - 1 / 70000).abs() <= 2.0 ** -20 / 70000).all())


def test_logits_temperature_that_is_no_number(ops):
    rows = rnd(4, 100, seed=6)
    controls = torch.tensor([[1.0, 0, 0, 1, t] for t in (0.0, -1.0, float("nan"), 1.0)]).cuda()
    for k in ("logits", "probs", "log_probs"):
        out = ops.logits(rows, kind=k, controls=controls)
        assert bool(out[:3].isnan().all()) and not bool(out[3].isnan().any())


def test_logits_temperatures_at_the_ends_of_the_type(ops):
    """Up to 2^-127 and 3e38 they are what logits are divided by; one whose reciprocal is infinite is none (zero logits would be NaN beside the infinities of
    the others)."""
    rows = torch.tensor([[0.0, 1.0, -2.0, 2.0 ** -126]] * 5, device="cuda")
    temperatures = [2.0 ** -126, 3.0e38, 2.0 ** -127, 2.0 ** -128, 2.0 ** -149]
    controls = torch.tensor([[1.0, 0, 0, 1, t] for t in temperatures]).cuda()
    out = ops.logits(rows, kind="logits", controls=controls).double().cpu().numpy()
    want = rows[0].double().cpu().numpy()
    assert np.array_equal(out[0], want * 2.0 ** 126) and np.array_equal(out[2], [0.0, 2.0 ** 127, -np.inf, 2.0])
    off = np.abs(out[1] - want / float(controls[1, 4]))
    assert (off <= 2.0 ** -149 * (1 + np.abs(want))).all()                    # (subnormal reciprocal and results: a step of those)
    for k in ("logits", "probs", "log_probs"):
        res = ops.logits(rows, kind=k, controls=controls)
        assert bool(res[3:].isnan().all()) and not bool(res[:3].isnan().any())


def test_logits_repeats_and_the_edges_of_decay(ops):
    """One token many times (a count beyond 2^16), decay 0 (the newest token alone), 1 (a count) and beyond its range; a bias listed twice."""
    V, m = 64, 70000
    rows = rnd(5, V, seed=7)
    controls = torch.tensor([[1.0, 0.25, 0.5, d, 1.0] for d in (1.0, 0.0, 0.5, 7.0, -3.0)]).cuda()
    histories = [[9] * m, [3, 9, 9], [9, 9, 9, 4], [9] * 3, [1, 9]]
    off, flat = ragged(histories)
    out = ops.logits(rows, kind="logits", controls=controls, history=flat, history_offset=off)
    down = (rows - out).double().cpu().numpy()
    assert abs(down[0, 9] - (0.25 + 0.5 * m)) <= 0.5 * m * 2.0 ** -22
    for got, want in [(down[1, 9], 0.75), (down[1, 3], 0.25), (down[2, 9], 0.25 + 0.5 * 0.875), (down[2, 4], 0.75), (down[3, 9], 1.75), (down[4, 9], 0.75), (down[4, 1], 0.25)]:
        assert abs(got - want) <= 2.0 ** -21
    off, tok = ragged([[5, 7, 5], [], [5], [], []])
    out = ops.logits(rows, kind="logits", bias_offset=off, bias_token=tok, bias_value=torch.tensor([100.0, 2.0, 1.0, 4.0]).cuda())
    assert float(out[0, 5]) == float(rows[0, 5] + 1.0) and float(out[0, 7]) == float(rows[0, 7] + 2.0) and float(out[2, 5]) == float(rows[2, 5] + 4.0)
    assert torch.equal(out[[1, 3, 4]], rows[[1, 3, 4]])


@pytest.mark.parametrize("m", [3000, 100000])
def test_logits_weights_that_decay_away(ops, m):
    """One token said over and over: what has decayed away adds nothing to its weight, and counts for presence all the same.

    An entry is kept in units of 2^-28: it is off by half a unit, or by itself where it is less.  Then as in logits_want."""
    V, decays, frequency = 50, [0.0, 0.5, 0.9, 0.99, 0.999, 0.9999], 0.5
    rows = rnd(len(decays), V, seed=31)
    controls = torch.tensor([[1.0, 0.25, frequency, d, 1.0] for d in decays]).cuda()
    history = [4] * 3 + [9] * m                          # (token 4 is the oldest)
    off, flat = ragged([history] * len(decays))
    out = ops.logits(rows, kind="logits", controls=controls, history=flat, history_offset=off).double().cpu().numpy()
    l = rows.double().cpu().numpy()
    for i, d in enumerate(controls[:, 3].double().tolist()):
        age = np.arange(m + 3)
        w = np.where(age == 0, 1.0, d ** age)
        with np.errstate(divide="ignore"):
            w_off = np.where(w > 0, w * 2.0 ** -22 * (2 + age * np.abs(np.log2(d))), 0) if d > 0 else 0 * w
        w_off = w_off + np.minimum(w, 2.0 ** -29) * (age > 0)
        for t, part in ((9, slice(0, m)), (4, slice(m, m + 3))):
            down = 0.25 + frequency * w[part].sum()
            bound = frequency * w_off[part].sum() + 2.0 ** -22 * down + 2.0 ** -23 * abs(l[i, t] - down)
            assert abs(out[i, t] - (l[i, t] - down)) <= bound, (d, t, out[i, t], l[i, t] - down, bound)


@pytest.mark.parametrize("V", [4096, 4097, 65536, 460001])
def test_logits_strides_in_place_and_rows_behind(ops, V):
    for shift in (0, 1, 4):
        wide = rnd(4, V + 12, seed=8)
        rows = wide[:3, shift:shift + V]
        want, err = logits_want(rows, "probs")
        outw = torch.full((5, V + 8), 7.0, device="cuda")
        ops.logits(rows, kind="probs", out=outw[:3, shift:shift + V])
        check_logits(outw[:3, shift:shift + V], want, err)
        keep = torch.ones_like(outw, dtype=torch.bool)
        keep[:3, shift:shift + V] = False
        assert bool((outw[keep] == 7.0).all())
        before = wide.clone()
        ops.logits(rows, kind="probs", out=rows)
        check_logits(rows, want, err)
        assert torch.equal(wide[3], before[3]) and torch.equal(wide[:, shift + V:], before[:, shift + V:])


def test_logits_graph_stream_and_no_rows(ops):
    rows, controls, histories, froms, biases, masks, mask_of = logits_case(6, 30000, F32, 400, 0.5, 20, seed=11)
    assert ops.logits(rows[:0], kind="probs").shape == (0, 30000)
    out = call(ops, rows, "probs", controls, histories, froms, biases, masks, mask_of)
    off, flat = ragged(histories)
    g, res = torch.cuda.CUDAGraph(), torch.empty_like(out)
    with torch.cuda.graph(g):
        ops.logits(rows, kind="log_probs", controls=controls, history=flat, history_offset=off, out=res)
    rows.copy_(rnd(6, 30000, seed=12))
    g.replay()
    g.replay()
    want, err = logits_want(rows, "log_probs", controls, histories)
    check_logits(res, want, err)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2 = ops.logits(rows, kind="log_probs", controls=controls, history=flat, history_offset=off)
    s.synchronize()
    assert torch.equal(o2, res)


@pytest.mark.parametrize("kind", ["logits", "probs"])
def test_logits_rows_far_apart(ops, kind):
    n, V, step = 4, 1000, (1 << 32) // 3 + 4096
    rows = rnd(n, V, seed=21)
    far = torch.empty((n - 1) * step + V, device="cuda").as_strided((n, V), (step, 1))
    out = torch.empty((n - 1) * step + V, device="cuda").as_strided((n, V), (step, 1))
    far.copy_(rows)
    ops.logits(far, kind=kind, out=out)
    assert torch.equal(out.contiguous(), ops.logits(rows, kind=kind)) if kind == "logits" else bool(((out - ops.logits(rows)).abs() <= 2.0 ** -20 * out).all())


def test_calls_from_two_threads(ops):
    """Two host threads, each on a stream of its own, at the same time: what each gets is what it gets alone."""
    import threading
    sets = []
    for i, T in enumerate((40, 700)):
        x, a, b, scale, y = make(T, 256, 96, 16, 5, F16, F32, seed=10 * i)
        index = indices(T, 5, "mixed", seed=i)
        rows = rnd(9 + i, 3000 + i, seed=30 + i)
        sets.append((x, a, b, index, scale, y, rows, ops.low_rank(x, a, b, index, scale, base=y), ops.logits(rows)))
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2, timeout=60)

    def work(s):
        x, a, b, index, scale, y, rows, want, probs = s
        stream = torch.cuda.Stream()
        gate.wait()
        with torch.cuda.stream(stream):
            got = [(ops.low_rank(x, a, b, index, scale, base=y), ops.logits(rows)) for _ in range(50)]
        stream.synchronize()
        wrong.extend(1 for o, q in got if not (torch.equal(o, want) and torch.equal(q, probs)))

    threads = [threading.Thread(target=work, args=(s,)) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_logits_history_longer_than_is_counted(ops):
    """Of a history the newest 2^17 - 1 tokens count: a token that is older than those alone is as if it had not been said."""
    V, m = 300, 140000
    most = (1 << 17) - 1
    rows = rnd(1, V, seed=13)
    history = [7] * 10 + [5] * (m - 10)
    off, flat = ragged([history])
    controls = torch.tensor([[2.0, 1.0, 0.5, 1.0, 1.0]]).cuda()
    out = ops.logits(rows, kind="logits", controls=controls, history=flat, history_offset=off)
    r = float(rows[0, 5])
    want = (r / 2 if r > 0 else r * 2) - (1.0 + 0.5 * most)
    assert abs(float(out[0, 5]) - want) <= abs(want) * 2.0 ** -22
    keep = torch.ones(V, dtype=torch.bool, device="cuda")
    keep[5] = False
    assert torch.equal(out[0, keep], rows[0, keep])


def test_tensors_that_ask_for_a_gradient_are_refused(ops):
    x, a, b, scale, y = make(3, 64, 32, 8, 2, F16, F16)
    index = indices(3, 2, "distinct")
    for t in (x, a, b, y):
        t.requires_grad_()
        with pytest.raises(capi.B200Error):
            ops.low_rank(x, a, b, index, scale, base=y)
        with torch.no_grad():
            ops.low_rank(x, a, b, index, scale, base=y)
        t.requires_grad_(False)
    rows = rnd(2, 50).requires_grad_()
    with pytest.raises(capi.B200Error):
        ops.logits(rows)


def test_the_first_call_of_a_process_can_be_captured():
    """Kernels are set up by the call that needs them first, also while a stream is captured."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from ai00_server_b200 import device_ops as d
r = lambda *s: torch.randn(*s, device="cuda")
sets = [(T, r(T, 64).half(), r(3, 16, 64).half(), r(3, 40, 16).half(), (torch.arange(T, device="cuda") % 3).int(), torch.ones(3, device="cuda")) for T in (1, 40, 300)]
rows = r(4, 500)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = [d.low_rank(x, a, b, i, s) for _, x, a, b, i, s in sets]
    probs = d.logits(rows)
g.replay()
torch.cuda.synchronize()
for (T, x, a, b, i, s), o in zip(sets, outs):
    w = torch.stack([(x[t].float() @ a[t % 3].float().T) @ b[t % 3].float().T for t in range(T)])
    assert ((o.float() - w).abs() <= 2e-2 * w.abs().max()).all()
assert ((probs - rows.softmax(1)).abs() <= 1e-6).all()
print("captured")
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_head_adapter_then_probabilities(ops):
    """A decode batch's last steps as a server runs them, captured as one graph: adapters of the vocabulary head on the head's own output, then the
    requests' penalties, masks and biases."""
    T, K, V, n = 12, 512, 8000, 3
    x, a, b, scale, y = make(T, K, V, 16, n, F16, F32)
    index = indices(T, n, "mixed")
    _, controls, histories, froms, biases, masks, mask_of = logits_case(T, V, F32, 150, 0.5, 20, seed=21)
    off, flat = ragged(histories)
    boff, btok = ragged([[t for t, _ in r] for r in biases])
    bval = torch.tensor([v for r in biases for _, v in r]).cuda()
    allow, row = pack(masks), torch.tensor(mask_of, dtype=torch.int32).cuda()
    start = torch.tensor(froms, dtype=torch.int32).cuda()
    out = torch.empty(T, V, device="cuda")
    fresh = y.clone()

    def step():
        ops.low_rank(x, a, b, index, scale, base=y, out=y)
        ops.logits(y, kind="probs", controls=controls, history=flat, history_offset=off, history_from=start, allow=allow, allow_row=row,
                   bias_offset=boff, bias_token=btok, bias_value=bval, out=out)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    y.copy_(fresh)
    g.replay()
    want_y, err_y = adapter_want(x, a, b, index, scale, fresh, F32)
    check_adapters(y, want_y, err_y)
    want, err = logits_want(y, "probs", controls, histories, froms, biases, masks, mask_of)
    check_logits(out, want, err)
