"""Operators on device memory that serve many requests at once, as a serving program calls them between the steps of its models:

  adapters   low-rank adapters of the requests of a batch beside their shared projections (ai00_server_b200.device_ops.low_rank): every
             token names the adapter of its request, or none
  logits     penalties for repeated tokens, biases and grammar masks on rows of logits, and what a sampler reads of them: the adjusted
             logits, probabilities or log-probabilities (ai00_server_b200.device_ops.logits)

Widths are those of the RWKV shapes this repository serves (hidden sizes 2048, 2560, 4096; feed-forwards of 3.5 times that; 65536 tokens
of vocabulary), or generic.  Everything a case says follows from its dict; values follow from the seed.
"""
from __future__ import annotations

import math

import torch

own = False                     # whether run() calls the framework's operators or computes their plain form

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _adapters(name, tokens, runs, k, n, rank, pool, **more):
    """tokens: rows of the batch, cut into `runs` sequences of uneven lengths; every `none`-th run has no adapter; parts: projections of k inputs
    and n outputs that the call serves; shuffled: rows of different requests lie side by side, as in a decode batch."""
    c = {"name": name, "op": "adapters", "tokens": tokens, "runs": runs, "k": k, "n": n, "rank": rank, "pool": pool, "none": 0, "parts": 1,
         "type": "f16", "out": "f32", "base": True, "shuffled": False}
    c.update(more)
    return c


def _logits(name, rows, vocab, **more):
    """history: tokens of the longest request (others are shorter); masks: grammar masks in the batch; allowed: share of the vocabulary they leave;
    bias: entries of the longest bias list."""
    c = {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "type": "f32", "kind": "probs", "history": 0, "repetition": False,
         "masks": 0, "allowed": 0.5, "bias": 0, "controls": True}
    c.update(more)
    return c


def listed():
    return [
        # one user with an adapter of its own, one token at a time: an attention output projection, latency alone
        _adapters("adapter_token", 1, 1, 2048, 2048, 16, 4),
        # a full server of 16 slots, eight adapters and some requests without: receptance, key, value and gate of a layer in one call
        _adapters("adapters_16_slots", 16, 16, 2560, 2560, 16, 8, none=5, parts=4, shuffled=True),
        # 64 slots, each request with its own adapter, the feed-forward's key projection of a 7B layer
        _adapters("adapters_64_slots", 64, 64, 4096, 14336, 32, 64, type="bf16", out="bf16", shuffled=True),
        # a mixed step: a few prompts of uneven lengths beside single tokens, odd counts
        _adapters("adapters_mixed_step", 333, 21, 2560, 8960, 24, 12, none=4, type="bf16"),
        # prompts of a few requests, the value projection of a feed-forward, high rank
        _adapters("adapters_prompts", 1021, 5, 8960, 2560, 128, 6, out="f16"),
        # a full prompt step of four requests through a 7B key projection: the largest
        _adapters("adapters_long_step", 2048, 4, 4096, 14336, 64, 4),
        # one row for a sampler that wants logits
        _logits("logits_row", 1, 65536, kind="logits", history=300),
        # 16 slots, the whole distribution for typical or mirostat sampling
        _logits("probs_16_slots", 16, 65536, history=2000, bias=30, repetition=True),
        # structured answers: each of 64 requests under its own grammar, a small vocabulary
        _logits("grammar_64", 64, 32000, type="f16", kind="log_probs", masks=64, allowed=0.02, history=150),
        # everything at once on a wide, odd vocabulary
        _logits("wide_96", 96, 100003, type="bf16", history=8000, masks=7, allowed=0.6, bias=300, repetition=True),
        # scoring: log-probabilities of a prompt's rows (perplexity, choices)
        _logits("score_512", 512, 65536, kind="log_probs", controls=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"], w["flops"]


def draw(rng):
    most = {c["name"]: _cost(c) for c in listed()}
    adapters = rng.random() < 0.5
    while True:
        if adapters:
            tokens = _log_int(rng, 1, 2048)
            decode = rng.random() < 0.4
            c = _adapters("", tokens, tokens if decode else min(tokens, _log_int(rng, 1, 32)), 8 * _log_int(rng, 32, 1120), 8 * _log_int(rng, 32, 1792),
                          8 * rng.randint(1, 16), _log_int(rng, 1, 64), none=rng.choice([0, 0, 3, 7]), parts=rng.choice([1, 1, 2, 4]),
                          type=rng.choice(["f16", "bf16"]), base=rng.random() < 0.8, shuffled=decode or rng.random() < 0.2)
            c["out"] = rng.choice(["f32", c["type"]])
            top = most["adapters_long_step"]
        else:
            c = _logits("", _log_int(rng, 1, 512), _log_int(rng, 2000, 200000), type=rng.choice(["f32", "f32", "f16", "bf16"]),
                        kind=rng.choice(["logits", "probs", "log_probs"]), history=rng.choice([0, _log_int(rng, 1, 8000)]), repetition=rng.random() < 0.5,
                        masks=rng.choice([0, 1, 5, 33]), allowed=rng.choice([0.001, 0.1, 0.7]), bias=rng.choice([0, _log_int(rng, 1, 500)]))
            top = most["score_512"]
        del c["name"]
        b, f = _cost(c)
        if b <= top[0] and f <= top[1]:
            return c


def _run_lengths(c):
    """Tokens of the runs: later ones are longer."""
    runs = c["runs"]
    cuts = [round(c["tokens"] * (i / runs) ** (1.0 if runs == c["tokens"] else 1.3)) for i in range(runs + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _run_adapters(c):
    """Adapter of each run before the pool is permuted: -1 for none."""
    return [-1 if c["none"] and r % c["none"] == c["none"] - 1 else r % c["pool"] for r in range(c["runs"])]


def _list_lengths(rows, longest):
    """Ragged lists: the first row has the longest, the others between none and that."""
    return [longest if i == 0 else (longest * ((i * 37) % 101)) // 100 for i in range(rows)]


def work(case):
    c = case
    if c["op"] == "adapters":
        lengths, ids = _run_lengths(c), _run_adapters(c)
        used = len({a for a, m in zip(ids, lengths) if m and a >= 0})
        served = sum(m for a, m in zip(ids, lengths) if a >= 0)
        o = _SIZE[c["out"]]
        part = served * c["k"] * 2 + used * c["rank"] * (c["k"] + c["n"]) * 2 + c["tokens"] * c["n"] * o * (2 if c["base"] else 1)
        return {"bytes": c["parts"] * part + 4 * c["tokens"] + 4 * used, "flops": c["parts"] * 2 * served * c["rank"] * (c["k"] + c["n"])}
    rows, V = c["rows"], c["vocab"]
    lists = sum(_list_lengths(rows, c["history"])) * 4 + sum(_list_lengths(rows, c["bias"])) * 8 + min(c["masks"], rows) * ((V + 31) // 32) * 4
    return {"bytes": rows * V * (_SIZE[c["type"]] + 4) + lists + (rows * 20 if c["controls"] else 0), "flops": rows * V * 8}


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    cpu = torch.Generator().manual_seed(int(seed) * 1000003 + 29)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    if c["op"] == "adapters":
        t, o = _T[c["type"]], _T[c["out"]]
        T, K, N, R, n = c["tokens"], c["k"], c["n"], c["rank"], c["pool"]
        perm = torch.randperm(n, generator=cpu).tolist()
        ids = [perm[a] if a >= 0 else -1 for a in _run_adapters(c)]
        index = torch.tensor([a for a, m in zip(ids, _run_lengths(c)) for _ in range(m)], dtype=torch.int32)
        if c["shuffled"]:
            index = index[torch.randperm(T, generator=cpu)]
        return {"case": c, "index": index.cuda(), "scale": 0.25 + 1.75 * torch.rand(n, generator=g, device="cuda"),
                "x": [normal(T, K, dtype=t) for _ in range(c["parts"])],
                "a": [normal(n, R, K, std=K ** -0.5, dtype=t) for _ in range(c["parts"])],
                "b": [normal(n, N, R, std=0.05, dtype=t) for _ in range(c["parts"])],
                "base": [normal(T, N, dtype=o) for _ in range(c["parts"])] if c["base"] else None,
                "out": [torch.empty(T, N, dtype=o, device="cuda") for _ in range(c["parts"])]}

    rows, V = c["rows"], c["vocab"]
    s = {"case": c, "logits": normal(rows, V, std=3.0, dtype=_T[c["type"]]), "out": torch.empty(rows, V, device="cuda"), "controls": None,
         "history": None, "history_offset": None, "history_from": None, "allow": None, "allow_row": None, "bias_offset": None, "bias_token": None,
         "bias_value": None}
    u = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    if c["controls"]:
        one = torch.ones(rows, device="cuda")
        # repetition, presence, frequency, decay of a token's weight with its age, temperature
        s["controls"] = torch.stack([u(1.02, 1.3) if c["repetition"] else one, u(0.0, 0.6), u(0.0, 0.6), 1.0 - u(0.0, 0.01), u(0.6, 1.4)], 1).contiguous()
    if c["history"]:
        lens = _list_lengths(rows, c["history"])
        total = sum(lens)
        # a few tokens come back again and again, most are rare
        s["history"] = (V * torch.rand(total, generator=g, device="cuda") ** 6).to(torch.int32).clamp_(max=V - 1)
        s["history_offset"] = torch.tensor([sum(lens[:i]) for i in range(rows + 1)], dtype=torch.int32).cuda()
        s["history_from"] = torch.tensor([m // 3 for m in lens], dtype=torch.int32).cuda()          # a third of it is the prompt
    if c["masks"]:
        m = min(c["masks"], rows)
        words = (V + 31) // 32
        keep = torch.rand(m, words * 32, generator=g, device="cuda") < c["allowed"]
        keep[:, 5] = True                                                                           # a grammar leaves something
        bits = (keep.view(m, words, 32).long() << torch.arange(32, device="cuda")).sum(2)
        s["allow"] = ((bits + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32)                         # the same 32 bits, signed
        row = torch.arange(rows) % m
        if m < rows:
            row[3::4] = -1                                                                          # requests without a grammar
        s["allow_row"] = row.to(torch.int32).cuda()
    if c["bias"]:
        lens = [min(n, V // 2) for n in _list_lengths(rows, c["bias"])]
        step = [V // max(1, n) for n in lens]                                                       # distinct tokens of a list
        s["bias_token"] = torch.tensor([(j * st + 1) % V for n, st in zip(lens, step) for j in range(n)], dtype=torch.int32).cuda()
        s["bias_value"] = normal(sum(lens), std=4.0)
        s["bias_offset"] = torch.tensor([sum(lens[:i]) for i in range(rows + 1)], dtype=torch.int32).cuda()
    return s


def run(state):
    s = state
    c = s["case"]
    if own:
        from ai00_server_b200 import device_ops
        if c["op"] == "adapters":
            return device_ops.low_rank(s["x"], s["a"], s["b"], s["index"], s["scale"], base=s["base"], out=s["out"])
        return device_ops.logits(s["logits"], kind=c["kind"], controls=s["controls"], history=s["history"], history_offset=s["history_offset"],
                                 history_from=s["history_from"], allow=s["allow"], allow_row=s["allow_row"], bias_offset=s["bias_offset"],
                                 bias_token=s["bias_token"], bias_value=s["bias_value"], out=s["out"])
    return _plain_adapters(s) if c["op"] == "adapters" else _plain_logits(s)


def _plain_adapters(s):
    """One product with all adapters side by side, rows of other requests' adapters zeroed between the two factors."""
    c = s["case"]
    n, R, T = c["pool"], c["rank"], c["tokens"]
    weight = (s["index"][:, None] == torch.arange(n, device="cuda", dtype=torch.int32)).float() * s["scale"]
    base = s["base"] or [None] * c["parts"]

    def part(x, a, b, y):
        low = (x.float() @ a.float().reshape(n * R, -1).t()).view(T, n, R) * weight[:, :, None]
        d = low.view(T, n * R) @ b.float().permute(0, 2, 1).reshape(n * R, -1)
        return (d if y is None else y.float() + d).to(_T[c["out"]])

    return list(map(part, s["x"], s["a"], s["b"], base))


def _rows_of(offset, total):
    rows = offset.numel() - 1
    return torch.repeat_interleave(torch.arange(rows, device="cuda"), (offset[1:] - offset[:-1]).long(), output_size=total)


def _plain_logits(s):
    c = s["case"]
    rows, V = c["rows"], c["vocab"]
    l = s["logits"].float()
    if s["history"] is not None:
        rep, presence, frequency, decay = (s["controls"][:, i, None] for i in range(4))
        off, tok = s["history_offset"].long(), s["history"].long()
        row = _rows_of(off, tok.numel())
        at = torch.arange(tok.numel(), device="cuda") - off[row]
        counts = at >= s["history_from"][row]
        age = (off[row + 1] - off[row] - 1 - at).double()
        w = torch.where(counts, decay[row, 0].double() ** age, 0.0)
        seen = torch.zeros(rows, V, dtype=torch.bool, device="cuda").index_put((row, tok), torch.tensor(True, device="cuda"))
        weight = torch.zeros(rows, V, dtype=torch.float64, device="cuda").index_put((row, tok), w, accumulate=True)
        said = torch.zeros(rows, V, device="cuda").index_put((row, tok), counts.float(), accumulate=True) > 0
        l = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
        l = l - (said * presence + weight.float() * frequency)
    if s["bias_token"] is not None:
        row = _rows_of(s["bias_offset"].long(), s["bias_token"].numel())
        l = l.index_put((row, s["bias_token"].long()), s["bias_value"], accumulate=True)
    if s["allow"] is not None:
        bits = (s["allow"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        bits = bits.view(bits.shape[0], -1)[:, :V].bool()
        free = s["allow_row"] < 0
        l = torch.where(bits[s["allow_row"].clamp(min=0).long()] | free[:, None], l, -math.inf)
    if s["controls"] is not None:
        l = l / s["controls"][:, 4, None]
    if c["kind"] == "logits":
        return l
    d = l - l.max(1, keepdim=True).values
    e = d.exp()
    z = e.sum(1, keepdim=True)
    return e / z if c["kind"] == "probs" else d - z.log()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "adapters":
        outs = []
        for p in range(c["parts"]):
            y = s["base"][p].double() if c["base"] else torch.zeros(c["tokens"], c["n"], dtype=torch.float64, device="cuda")
            for i in range(c["pool"]):
                t = (s["index"] == i).nonzero()[:, 0]
                if t.numel():
                    y[t] += float(s["scale"][i]) * ((s["x"][p][t].double() @ s["a"][p][i].double().t()) @ s["b"][p][i].double().t())
            outs.append(y)
        return outs
    V = c["vocab"]
    l = s["logits"].double()
    for i in range(c["rows"]):
        rep, presence, frequency, decay, temperature = s["controls"][i].double().tolist() if s["controls"] is not None else (1.0, 0.0, 0.0, 1.0, 1.0)
        r = l[i]
        if s["history"] is not None:
            a, b = s["history_offset"][i:i + 2].tolist()
            h = s["history"][a:b].long()
            if h.numel():
                u = h.unique()
                r[u] = torch.where(r[u] > 0, r[u] / rep, r[u] * rep)
                first = int(s["history_from"][i])
                w = decay ** torch.arange(h.numel() - 1 - first, -1, -1, device="cuda", dtype=torch.float64)
                sums = torch.bincount(h[first:], weights=w, minlength=V)
                r -= frequency * sums + presence * (torch.bincount(h[first:], minlength=V) > 0)
        if s["bias_token"] is not None:
            a, b = s["bias_offset"][i:i + 2].tolist()
            r[s["bias_token"][a:b].long()] += s["bias_value"][a:b].double()
        if s["allow"] is not None and int(s["allow_row"][i]) >= 0:
            t = torch.arange(V, device="cuda")
            r[((s["allow"][int(s["allow_row"][i])].long()[t // 32] >> (t % 32)) & 1) == 0] = -math.inf
        r /= temperature
        if c["kind"] != "logits":
            r -= r.max()
            z = r.exp().sum()
            l[i] = r.exp() / z if c["kind"] == "probs" else r - z.log()
    return l
