"""Adapters of slots (b200rwkv_adapter_load / b200rwkv_slot_adapter) in the steps of the RWKV models, against the oracle on weights W + alpha B A^T kept
in f32: the operands of every product are the engine's own (f16 weights, f16 low-rank factors), so the distance is that of the plain model."""
import numpy as np
import pytest

from ai00_server_b200 import capi, runtime, synth
from oracle import quant_numpy as Q
from oracle import rwkv_numpy as O

pytestmark = pytest.mark.gpu

REL_TOL = 1e-3
ALL = ("att.receptance", "att.key", "att.value", "att.gate", "att.output", "ffn.key", "ffn.value", "ffn.receptance")


def rel_err(a, b):
    return float(np.abs(a - b).max() / max(np.abs(b).max(), 1e-30))


def with_adapter(weights, lora, alpha):
    out = dict(weights)
    for name in lora:
        if name.endswith(".lora.0"):
            base = name[:-7]
            a, b = lora[name].astype(np.float32), lora[base + ".lora.1"].astype(np.float32)
            out[base + ".weight"] = weights[base + ".weight"].astype(np.float32) + np.float32(alpha) * (b @ a.T)
    return out


def moved(weights, seed):
    """Projection weights off by 2^-12 of themselves, up or down: the products of operands of which a quarter are a whole f16 step, 2^-10 at most, off."""
    rng = np.random.default_rng(seed)
    return {k: v.astype(np.float32) * (1 + np.float32(2.0 ** -12) * rng.choice(np.array([-1, 1], np.float32), size=v.shape))
            if k.endswith(".weight") and v.ndim == 2 and k != "emb.weight" else v for k, v in weights.items()}


# two files: every matrix at rank 12 (padded), some of them at rank 8
def files(preset):
    return [(synth.make_lora_st(preset, rank=12, seed=5, targets=ALL), 0.7), (synth.make_lora_st(preset, rank=8, seed=6), -0.9)]


def setup(preset, max_batch=4, chunk=32, exact=False, quant=0):
    st = synth.make_st(preset, 0)
    m = runtime.Model(st, max_batch=max_batch, token_chunk_size=chunk, exact=exact, quant=quant, quant_type="Int8" if quant else 0)
    base = O.parse_st(st)
    if quant:
        base = Q.quantize_model(base, quant, Q.QUANT_INT8)
    act = "f32" if exact else "f16"
    fs = files(preset)
    oracles = [O.Oracle(base, act)] + [O.Oracle(with_adapter(base, O.parse_st(f), alpha), act) for f, alpha in fs]
    handles = [None] + [m.load_adapter(f, alpha) for f, alpha in fs]
    for s in range(max_batch):
        m.state.load(m.state.init(), s)
    return m, oracles, handles


@pytest.mark.parametrize("preset,exact,quant", [("tiny5", False, 0), ("tiny6", False, 0), ("tiny7", False, 0), ("small6", False, 0), ("tiny6", True, 0),
                                                ("tiny7", True, 0), ("tiny6", False, 2), ("small7", False, 0)])
def test_slots_with_different_adapters(preset, exact, quant):
    m, oracles, handles = setup(preset, exact=exact, quant=quant)
    try:
        # f16 operands: a sum that lands on the other side of a rounding border moves an operand by a step of f16, and what follows need not be
        # well conditioned: the third layer of the RWKV-7 model norms a head whose values nearly cancel on its first token and hands 2.5e-4 of its input
        # on as 3.6e-2 of its output.  How far two right implementations can be apart is therefore computed for each output: the distances of the
        # oracle from itself with operands off by such steps (four draws) and from its f32 contract, which rounds none; twice the largest, 1e-3 at
        # least.  At precision 1 nothing is rounded and 1e-4 holds, for the same head too.
        near = [[O.Oracle(moved(o.w, i), "f16") for i in range(4)] + [O.Oracle(o.w, "f32")] for o in oracles] if not exact else None
        who = [1, 0, 2, 1]
        for s, w in enumerate(who):
            m.set_adapter(s, handles[w])
        rng = np.random.default_rng(3)
        states = [o.state_init() for o in (oracles[w] for w in who)]
        beside = [[x.copy() for _ in range(5)] for x in states]
        plain = oracles[0].state_init()
        change = 0.0
        for step, counts in enumerate([(9, 3, 1, 20), (1, 1, 1, 1), (1, 1, 1, 1), (2, 0, 5, 1)]):
            toks = [rng.integers(1, 500, size=n).tolist() for n in counts]
            rows = m.infer_raw([0, 1, 2, 3], [len(t) for t in toks], sum(toks, []), [capi.OPTION_LAST, capi.OPTION_FULL, capi.OPTION_LAST, capi.OPTION_FULL])
            for s, w in enumerate(who):
                if not toks[s]:
                    continue
                want, states[s] = oracles[w].run(toks[s], states[s], full=s in (1, 3))
                tol = 1e-4
                if not exact:
                    tol = REL_TOL
                    for i, o in enumerate(near[w]):
                        other, beside[s][i] = o.run(toks[s], beside[s][i], full=s in (1, 3))
                        tol = max(tol, 2 * rel_err(other, want))
                assert rows[s].shape == want.shape
                assert rel_err(rows[s], want) <= tol, (step, s, rel_err(rows[s], want), tol)
                if s == 0:
                    other, plain = oracles[0].run(toks[s], plain)
                    change = max(change, rel_err(other, want))
        for s in range(4):
            tol = 1e-4 if exact else max([2 * REL_TOL] + [2 * rel_err(x, states[s]) for x in beside[s]])
            assert rel_err(m.state.back(s), states[s]) <= tol
        assert change > 20 * REL_TOL                      # the adapters really change the model
    finally:
        m.close()


@pytest.mark.parametrize("preset,counts", [("tiny6", (40, 21, 3, 30)), ("tiny5", (130, 60, 1, 40)), ("tiny6", (300, 1, 120, 7)), ("tiny7", (290, 200, 16, 1))])
def test_prompts_with_adapters(preset, counts):
    """Steps of every form: up to 64 and 128 tokens, and several hundred, with all rows of one prompt asked for."""
    m, oracles, handles = setup(preset, chunk=128)
    try:
        who = [2, 0, 1, 2]
        for s, w in enumerate(who):
            m.set_adapter(s, handles[w])
        rng = np.random.default_rng(4)
        toks = [rng.integers(1, 500, size=n).tolist() for n in counts]
        options = [capi.OPTION_FULL, capi.OPTION_LAST, capi.OPTION_LAST, capi.OPTION_NONE]
        rows = m.infer_raw([0, 1, 2, 3], list(counts), sum(toks, []), options)
        for s, w in enumerate(who):
            want, state = oracles[w].run(toks[s], oracles[w].state_init(), full=s == 0)
            if s < 3:
                assert rel_err(rows[s], want) <= 2 * REL_TOL, (s, rel_err(rows[s], want))
            assert rel_err(m.state.back(s), state) <= 2 * REL_TOL
    finally:
        m.close()


@pytest.mark.parametrize("preset", ["tiny5", "tiny6", "tiny7"])
def test_adapters_of_one_projection_at_a_time(preset):
    """A file that has one of the matrices alone (in all layers), at precision 1, where nothing is rounded: 1e-4 of the oracle, where an adapter that is one percent too
    large in that projection is further off than four times that."""
    st = synth.make_st(preset, 0)
    base = O.parse_st(st)
    full = O.parse_st(synth.make_lora_st(preset, rank=12, seed=5, targets=ALL))
    m = runtime.Model(st, max_batch=4, token_chunk_size=32, exact=True)
    rng = np.random.default_rng(8)
    served = 0
    try:
        for target in (*ALL, "head"):
            pairs = {k: v for k, v in full.items() if target in k}
            if not pairs:
                continue
            served += 1
            handle = m.load_adapter(synth.pack_st(pairs), 1.0)
            oracle, more = (O.Oracle(with_adapter(base, pairs, alpha), "f32") for alpha in (1.0, 1.01))
            states = [oracle.state_init() for _ in range(3)]
            beside, off = more.state_init(), 0.0
            for s in range(4):
                m.state.load(m.state.init(), s)
                m.set_adapter(s, handle if s < 3 else None)
            for counts in ((9, 4, 1, 2), (1, 1, 1, 1), (20, 3, 30, 1)):
                toks = [rng.integers(1, 500, size=n).tolist() for n in counts]
                rows = m.infer_raw([0, 1, 2, 3], list(counts), sum(toks, []), [capi.OPTION_LAST] * 4)
                for s in range(3):
                    want, states[s] = oracle.run(toks[s], states[s])
                    assert rel_err(rows[s], want) <= 1e-4, (target, counts, s, rel_err(rows[s], want))
                    if s == 0:
                        other, beside = more.run(toks[s], beside)
                        off = max(off, rel_err(other, want))
            assert off > 4e-4, (target, off)
            for s in range(3):
                assert rel_err(m.state.back(s), states[s]) <= 1e-4
                m.set_adapter(s, None)
            handle.free()
    finally:
        m.close()
    assert served == (7 if preset == "tiny7" else 9)


def test_slots_without_an_adapter_keep_their_results():
    st = synth.make_st("tiny6", 0)
    toks = [[3, 9, 200], [41, 7], [5]]

    def run(adapter):
        m = runtime.Model(st, max_batch=4, token_chunk_size=32)
        try:
            for s in range(3):
                m.state.load(m.state.init(), s)
            if adapter:
                m.set_adapter(1, m.load_adapter(*files("tiny6")[0]))
            return [r.copy() for _ in range(3) for r in m.infer_raw([0, 1, 2], [len(t) for t in toks], sum(toks, []), [capi.OPTION_LAST] * 3)]
        finally:
            m.close()

    a, b = run(False), run(True)
    for i in range(9):
        assert np.array_equal(a[i], b[i]) == (i % 3 != 1), i


def test_binding_changes_between_calls():
    """One slot under one adapter, the other, none and the first again, with the captured step of before; an adapter of a larger rank comes later."""
    m, oracles, handles = setup("tiny6")
    try:
        state = oracles[0].state_init()
        wide, alpha = synth.make_lora_st("tiny6", rank=100, seed=9), 0.2
        for step, w in enumerate([1, 1, 2, 0, 3, 1, 3, 0]):
            if w == 3 and len(handles) == 3:
                handles.append(m.load_adapter(wide, alpha))
                oracles.append(O.Oracle(with_adapter(O.parse_st(synth.make_st("tiny6", 0)), O.parse_st(wide), alpha), "f16"))
            m.set_adapter(2, handles[w])
            got = m.infer_raw([2], [1], [step + 7], [capi.OPTION_LAST])[0]
            want, state = oracles[w].run([step + 7], state)
            assert rel_err(got, want) <= REL_TOL, (step, rel_err(got, want))
        m.set_adapter(2, handles[1])
        with pytest.raises(capi.B200Error) as ei:
            handles[1].free()                              # a slot has it
        assert ei.value.code == capi.ERR_STATE
        m.state.reset(2)                                   # an empty sequence, the same adapter
        got = m.infer_raw([2], [2], [5, 6], [capi.OPTION_LAST])[0]
        want, _ = oracles[1].run([5, 6], oracles[1].state_init())
        assert rel_err(got, want) <= REL_TOL
        m.set_adapter(2, None)
        handles[1].free()
        got = m.infer_raw([2], [2], [5, 6], [capi.OPTION_LAST])[0]
        assert np.isfinite(got).all()
    finally:
        m.close()


def test_launches_of_steps_with_adapters_are_counted():
    """b200rwkv_launch_count of steps with adapters: one kernel for the slots' adapters, and behind each projection launch one in steps of up to 256 tokens.  Longer
    steps order their tokens once, take three kernels behind each (sums, outputs, adapters of few tokens; 1536 tokens and more two), and one for each activation
    (gate, channel-mix key and receptance); the head's rows are few."""
    st = synth.make_st("tiny6", 0)
    counts = {}
    for adapter in (False, True):
        m = runtime.Model(st, max_batch=8, token_chunk_size=256)
        try:
            for s in range(8):
                m.state.load(m.state.init(), s)
            if adapter:
                m.set_adapter(1, m.load_adapter(*files("tiny6")[0]))

            def launched(n, slots):
                before = m.launch_count()
                m.infer_raw(list(range(slots)), [n] * slots, [5] * (n * slots), [capi.OPTION_LAST] * slots)
                return m.launch_count() - before

            counts[adapter] = [launched(1, 3), launched(1, 3), launched(20, 3), launched(100, 3), launched(220, 7)]
        finally:
            m.close()
    extra = [b - a for a, b in zip(counts[False], counts[True])]
    layers, behind = m.info["num_layer"], extra[0] - 1           # projection launches with adapters, the head's among them
    assert behind >= 4 * layers + 1
    assert extra[1] == extra[0] and extra[2] == extra[0]
    assert extra[3] == 2 + 3 * (behind - 1) + 3 * layers + 1
    assert extra[4] == 2 + 2 * (behind - 1) + 3 * layers + 1


def test_adapter_refusals():
    st = synth.make_st("tiny6", 0)
    m = runtime.Model(st, max_batch=2, token_chunk_size=32)

    def code(fn, *a):
        with pytest.raises(capi.B200Error) as ei:
            fn(*a)
        return ei.value.code

    try:
        pair = lambda base, i, o, r, dt=np.float16: {f"{base}.lora.0": np.zeros((i, r), dt), f"{base}.lora.1": np.zeros((o, r), dt)}  # noqa: E731
        load = lambda d: m.load_adapter(synth.pack_st(d))  # noqa: E731
        assert code(load, pair("blocks.0.att.time_mix_w1", 256, 160, 4)) == capi.ERR_UNSUPPORTED
        assert code(load, pair("blocks.9.att.key", 256, 256, 4)) == capi.ERR_UNSUPPORTED
        assert code(load, pair("blocks.0.att.key", 256, 256, 257)) == capi.ERR_UNSUPPORTED
        assert code(load, pair("blocks.0.att.key", 256, 256, 4, np.float32)) == capi.ERR_UNSUPPORTED
        assert code(load, pair("blocks.0.att.key", 128, 256, 4)) == capi.ERR_INVALID
        assert code(load, {"blocks.0.att.key.lora.0": np.zeros((256, 4), np.float16)}) == capi.ERR_INVALID
        assert code(load, {"blocks.0.att.key.lora.1": np.zeros((256, 4), np.float16)}) == capi.ERR_INVALID
        assert code(load, {"blocks.0.att.key.weight": np.zeros((256, 256), np.float16)}) == capi.ERR_UNSUPPORTED
        assert code(m.load_adapter, np.zeros(4, np.uint8)) == capi.ERR_INVALID
        assert code(m.load_adapter, synth.pack_st(pair("head", 256, 512, 4)), float("nan")) == capi.ERR_INVALID
        ghost = runtime.Adapter(m, 77)
        assert code(m.set_adapter, 0, ghost) == capi.ERR_STATE
        assert code(ghost.free) == capi.ERR_STATE
        one = load(pair("head", 256, 512, 256))
        assert code(m.set_adapter, 2, one) == capi.ERR_STATE and code(m.set_adapter, -1, one) == capi.ERR_STATE
        more = [load(pair("blocks.1.ffn.value", 896, 256, 1)) for _ in range(63)]
        assert code(load, pair("head", 256, 512, 8)) == capi.ERR_STATE          # 64 are held
        more[5].free()
        load(pair("head", 256, 512, 8))
        assert code(more[5].free) if more[5].id else True
    finally:
        m.close()
    layers = [synth.kemirax_layer("gla")]
    cfg, kst, _ = synth.make_kemirax(layers, seed=2)
    k = runtime.Model(kst, max_batch=2, token_chunk_size=32, config=cfg, kv_tokens=64, kv_page=8)
    try:
        assert code(k.load_adapter, files("tiny6")[0][0]) == capi.ERR_UNSUPPORTED
        k.set_adapter(0, None)
    finally:
        k.close()


# ---- whole rows for samplers ----
def rows_want(logits, kind, controls=None, history=None, history_from=None, allow=None, bias=None):
    l = logits.astype(np.float64).copy()
    for i, r in enumerate(l):
        rep, presence, frequency, decay, temperature = controls[i] if controls is not None else (1, 0, 0, 1, 1)
        h = history[i] if history is not None else []
        first = history_from[i] if history_from is not None else 0
        for t in set(h):
            r[t] = r[t] / rep if r[t] > 0 else r[t] * rep
        for t in set(h[first:]):
            r[t] -= presence + frequency * sum(decay ** (len(h) - 1 - j) for j in range(first, len(h)) if h[j] == t)
        for t, v in ((bias[i] or {}) if bias is not None else {}).items():
            r[t] += v
        if allow is not None:
            r[~allow[i]] = -np.inf
        r /= temperature
    if kind == "logits":
        return l
    d = l - l.max(1, keepdims=True)
    z = np.exp(d).sum(1, keepdims=True)
    return np.exp(d) / z if kind == "probs" else d - np.log(z)


@pytest.mark.parametrize("family", ["rwkv", "config.json"])
def test_sample_rows(family):
    if family == "rwkv":
        m = runtime.Model(synth.make_st("small6", 0), max_batch=4, token_chunk_size=32)
    else:
        cfg, st, _ = synth.make_kemirax([synth.kemirax_layer("gla"), synth.kemirax_layer("latent_attention")], seed=2)
        m = runtime.Model(st, max_batch=4, token_chunk_size=32, config=cfg, kv_tokens=256, kv_page=8)
    try:
        V = m.info["num_vocab"]
        for s in range(3):
            m.state.reset(s)
        rows = np.concatenate([r[-1:] for r in m.infer_raw([0, 1, 2], [3, 1, 2], [3, 9, 20, 41, 7, 6], [capi.OPTION_LAST, capi.OPTION_LAST, capi.OPTION_FULL])])
        rng = np.random.default_rng(1)
        slots = [2, 0, 2, 1]                               # a slot under two sets of controls
        controls = np.stack([rng.uniform(0.8, 1.4, 4), rng.uniform(0, 0.6, 4), rng.uniform(0, 0.6, 4), rng.uniform(0.9, 1, 4), rng.uniform(0.5, 2, 4)], 1).astype(np.float32)
        history = [rng.integers(0, V, n).tolist() * 2 for n in (30, 0, 5, 200)]
        allow = rng.random((4, V)) < 0.4
        bias = [{1: 4.0, V - 1: -3.0}, None, {}, {int(t): float(np.float32(v)) for t, v in zip(rng.choice(V, 40, replace=False), rng.normal(0, 3, 40))}]
        for kind in ("logits", "probs", "log_probs"):
            got = m.sample_rows(slots, kind)
            want = rows_want(rows[slots], kind)
            assert np.abs(got - want).max() <= 1e-5 * max(1.0, np.abs(want).max())
            kw = dict(controls=controls, history=history, history_from=[7, 0, 0, 100], allow=allow, bias=bias)
            got, want = m.sample_rows(slots, kind, **kw), rows_want(rows[slots], kind, **{**kw, "controls": controls.astype(np.float64)})
            fine = np.isfinite(want)
            assert np.array_equal(fine, np.isfinite(got))
            assert np.abs(got[fine] - want[fine]).max() <= 1e-5 * max(1.0, np.abs(want[fine]).max())
        soft = np.stack(m.softmax(list(rows)))
        assert np.abs(m.sample_rows([0, 1, 2]) - soft).max() <= 1e-6
        out = np.empty((2, V), np.float32)
        assert m.sample_rows([1, 1], out=out) is out and np.array_equal(out[0], out[1])
        assert m.sample_rows([]).shape == (0, V)
    finally:
        m.close()


def test_sample_rows_with_the_penalties_of_the_sampler():
    """Histories give NucleusSampler's distribution for a prompt; after generated tokens its map does as biases (b200rwkv_sample_topk with the map is the measure), and
    histories give another."""
    m = runtime.Model(synth.make_st("small6", 0), max_batch=2, token_chunk_size=32)
    try:
        V = m.info["num_vocab"]
        prompt = [3, 9, 20, 9, 41, 3, 3]
        m.state.reset(0)
        m.infer_raw([0], [len(prompt)], prompt, [capi.OPTION_LAST], keep_on_device=True)
        sampler = runtime.NucleusSampler(presence_penalty=0.4, frequency_penalty=0.6, penalty_decay=0.9)
        sampler.init(prompt)
        controls = np.array([[1.0, 0.4, 0.6, 0.9, 1.0]], np.float32)
        own = {5: 1.5, 41: -0.5}
        said = list(prompt)

        def measure(penalties):
            ids, probs = m.sample_topk([0], [penalties], [own])
            return ids[0].astype(int), probs[0]

        def near(row, ids, probs):
            # probabilities of two softmax kernels over the same logits: f32 sums of V terms, penalties of a dozen roundings, logits of some ten in size
            return np.abs(row[ids] - probs).max() <= 2.0 ** -18 * probs.max()

        ids, probs = measure(sampler.penalties)
        assert near(m.sample_rows([0], controls=controls, history=[said], bias=[own])[0], ids, probs)
        apart = 0
        for step in range(4):
            token = sampler.sample_candidates(ids, probs, 0.3 + 0.1 * step)
            said.append(token)
            m.infer_raw([0], [1], [token], [capi.OPTION_LAST], keep_on_device=True)
            ids, probs = measure(sampler.penalties)
            merged = {t: own.get(t, 0.0) - float(sampler.penalties.get(t, 0.0)) for t in {*own, *sampler.penalties}}
            assert near(m.sample_rows([0], bias=[merged])[0], ids, probs)
            apart += not near(m.sample_rows([0], controls=controls, history=[said], bias=[own])[0], ids, probs)
        assert apart == 4 and V > 128
    finally:
        m.close()


def test_sample_rows_refusals():
    m = runtime.Model(synth.make_st("tiny6", 0), max_batch=2, token_chunk_size=32)

    def code(*a, **k):
        with pytest.raises(capi.B200Error) as ei:
            m.sample_rows(*a, **k)
        return ei.value.code

    try:
        assert code([0]) == capi.ERR_STATE                 # no row yet
        m.state.reset(0)
        m.infer_raw([0], [1], [4], [capi.OPTION_LAST], keep_on_device=True)
        assert m.sample_rows([0]).shape == (1, 512)
        assert code([2]) == capi.ERR_STATE and code([-1]) == capi.ERR_STATE and code([0, 1]) == capi.ERR_STATE
        assert code([0], "odds") == capi.ERR_INVALID
        for bad in ([0, 0, 0, 1, 1], [1, 0, 0, 1, 0], [1, 0, 0, 1, -2], [1, 0, 0, 1.5, 1], [1, 0, 0, -0.1, 1], [1, np.nan, 0, 1, 1], [1, 0, 0, 1, np.inf]):
            assert code([0], controls=[bad]) == capi.ERR_INVALID, bad
        assert code([0], controls=[[1, 0, 0, 1]]) == capi.ERR_INVALID
        assert code([0], history=[[1], [2]]) == capi.ERR_INVALID and code([0], bias=[]) == capi.ERR_INVALID
        assert code([0], out=np.empty((1, 5), np.float32)) == capi.ERR_INVALID
        q = capi.RowControls(struct_bytes=8)
        assert capi.lib().b200rwkv_sample_rows(m._h, 1, q, None) == capi.ERR_INVALID
    finally:
        m.close()


def test_adapters_then_rows_as_a_server_uses_them():
    """A few tokens of three requests, two with adapters, sampled greedily from adjusted rows: the oracle's tokens."""
    m, oracles, handles = setup("tiny6")
    try:
        who = [1, 0, 2]
        for s, w in enumerate(who):
            m.set_adapter(s, handles[w])
        toks = [[3, 9, 200, 41], [41, 7], [5]]
        said = [list(t) for t in toks]
        states = [oracles[w].state_init() for w in who]
        feed = toks
        controls = np.array([[1.1, 0.4, 0.3, 0.996, 0.9]] * 3, np.float32)
        for _ in range(6):
            m.infer_raw([0, 1, 2], [len(t) for t in feed], sum(feed, []), [capi.OPTION_LAST] * 3, keep_on_device=True)
            probs = m.sample_rows([0, 1, 2], controls=controls, history=said, bias=[{0: -5.0}] * 3)
            nxt = []
            for s, w in enumerate(who):
                want, states[s] = oracles[w].run(feed[s], states[s])
                p = rows_want(want, "probs", controls[s:s + 1].astype(np.float64), [said[s]], bias=[{0: -5.0}])[0]
                # probabilities follow logits: relative distance of a probability is the absolute one of its logit over the temperature
                assert np.abs(probs[s] - p).max() <= p.max() * 4 * REL_TOL * np.abs(want).max() / 0.9
                nxt.append(int(p.argmax()))
                said[s].append(nxt[-1])
            feed = [[t] for t in nxt]
    finally:
        m.close()
