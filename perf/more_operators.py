"""Operators on device memory from the residual rows of a step to the tokens of its requests, as a serving program calls them between and behind its layers
(ai00_server_b200.device_ops):

  rms_norm      the residual's addition and a root-mean-square norm, with its output in 8 bits and a scale for every 128 columns of a row
  to_e4m3       rows (a scale for every 128 columns) or weights (a scale for every block of 128 x 128) in 8-bit floating point
  linear_e4m3   products of such rows and such weights
  sample        a token for each row of logits: temperature, top-k, top-p and min-p, from given random numbers

Widths are those of the RWKV shapes this repository serves (hidden sizes 2048, 2560, 4096; feed-forwards of 3.5 times that; 65536 tokens
of vocabulary), or generic.  Everything a case says follows from its dict; values follow from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False                     # whether run() calls the framework's operators or computes their plain form

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_E4M3 = torch.float8_e4m3fn
_TOP = 448.0                    # the largest e4m3 number
_LEAST = 2.0 ** -100            # scales are those of at least this much


def _norm(name, rows, width, **more):
    """residual: type of the residual rows (the sum is handed on in it), or none."""
    c = {"name": name, "op": "norm", "rows": rows, "width": width, "type": "bf16", "residual": "bf16", "weight": "f32", "offset": 0.0}
    c.update(more)
    return c


def _e4m3(name, rows, width, **more):
    """block: rows that share a scale (1: activations, 128: weights)."""
    c = {"name": name, "op": "e4m3", "rows": rows, "width": width, "type": "f16", "block": 1}
    c.update(more)
    return c


def _linear(name, tokens, k, n, **more):
    """base: rows that the products are added to."""
    c = {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "out": "bf16", "base": False}
    c.update(more)
    return c


def _sample(name, rows, vocab, **more):
    """top_k, top_p, min_p: the limits of the first row, others have theirs near it (0, 1, 0: no limit); greedy: every that many-th row takes the best token;
    sharp: how far apart the logits are."""
    c = {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "type": "f32", "top_k": 0, "top_p": 1.0, "min_p": 0.0, "greedy": 0, "sharp": 3.0}
    c.update(more)
    return c


def listed():
    return [
        # one sequence, one token: the norm in front of a layer's projections, latency alone
        _norm("norm_token", 1, 2560, type="f16", residual="f32"),
        # a full prompt step of a 7B layer
        _norm("norm_long_step", 2048, 4096),
        # what comes out of a feed-forward's activation in a mixed step, odd counts
        _e4m3("activations_mixed_step", 333, 8960),
        # a feed-forward's key matrix while a model is loaded
        _e4m3("weights_of_a_layer", 14336, 4096, type="bf16", block=128),
        # one sequence, one token, a square projection: latency
        _linear("linear_token", 1, 2560, 2560, out="f16"),
        # a full server of 16 slots through a 7B feed-forward's key projection
        _linear("linear_16_slots", 16, 4096, 14336),
        # a mixed step: a few prompts beside single tokens, added to the residual
        _linear("linear_mixed_step", 333, 8960, 2560, out="f32", base=True),
        # a full prompt step through a 7B feed-forward's key projection: the largest
        _linear("linear_long_step", 2048, 4096, 14336),
        # one row of a chat with the limits that most programs have by default
        _sample("sample_row", 1, 65536, top_k=50, top_p=0.95),
        # 16 slots, nucleus and min-p alone; every fifth request is greedy
        _sample("sample_16_slots", 16, 65536, top_p=0.9, min_p=0.02, greedy=5),
        # a wide, odd vocabulary in 16 bits, where many tokens are equal
        _sample("sample_96_wide", 96, 100003, type="bf16", top_k=1000, top_p=0.98, sharp=2.0),
        # many draws for the same kind of prompt (self-consistency, rollouts): no limits but the nucleus
        _sample("sample_512", 512, 65536, top_p=0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = {c["op"]: work(c) for c in listed()}          # the last of each operator is its largest
    op = rng.choice(["norm", "e4m3", "linear", "linear", "sample", "sample"])
    while True:
        t = rng.choice(["f32", "f16", "bf16"])
        if op == "norm":
            c = _norm("", _log_int(rng, 1, 2048), _log_int(rng, 100, 16384), type=t, residual=rng.choice(["", t, "f32"]), weight=rng.choice(["f32", t]),
                      offset=rng.choice([0.0, 1.0]))
        elif op == "e4m3":
            c = _e4m3("", _log_int(rng, 1, 16384), _log_int(rng, 100, 16384), type=t, block=rng.choice([1, 128]))
        elif op == "linear":
            c = _linear("", _log_int(rng, 1, 2048), 16 * _log_int(rng, 8, 600), _log_int(rng, 100, 65536), out=t, base=rng.random() < 0.4)
        else:
            c = _sample("", _log_int(rng, 1, 512), _log_int(rng, 2000, 200000), type=t, top_k=rng.choice([0, 0, _log_int(rng, 1, 2000)]),
                        top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 4)]),
                        greedy=rng.choice([0, 0, 3]), sharp=rng.choice([1.0, 2.0, 4.0, 8.0]))
        del c["name"]
        w = work(c)
        if w["bytes"] <= top[op]["bytes"] and w["flops"] <= top[op]["flops"]:
            return c


def work(case):
    c = case
    if c["op"] == "norm":
        n, groups = c["rows"] * c["width"], c["rows"] * -(-c["width"] // 128)
        return {"bytes": n * (_SIZE[c["type"]] + 2 * _SIZE.get(c["residual"], 0) + 1) + 4 * groups + c["width"] * _SIZE[c["weight"]], "flops": 6 * n}
    if c["op"] == "e4m3":
        n, groups = c["rows"] * c["width"], -(-c["rows"] // c["block"]) * -(-c["width"] // 128)
        return {"bytes": n * (_SIZE[c["type"]] + 1) + 4 * groups, "flops": 2 * n}
    if c["op"] == "linear":
        T, K, N, kb = c["tokens"], c["k"], c["n"], -(-c["k"] // 128)
        return {"bytes": T * K + N * K + 4 * kb * (T + -(-N // 128)) + T * N * _SIZE[c["out"]] * (2 if c["base"] else 1), "flops": 2 * T * N * K}
    return {"bytes": c["rows"] * (c["vocab"] * _SIZE[c["type"]] + 28), "flops": 8 * c["rows"] * c["vocab"]}


def _groups(x, rows):
    """[R, W] -> [R / rows, rows, W / 128, 128], zeros behind the edges."""
    R, W = x.shape
    x = torch.nn.functional.pad(x, (0, -W % 128, 0, -R % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128)


def _to_e4m3(x, rows):
    """(e4m3 numbers, scales) of f32 or f64 values."""
    g = _groups(x, rows)
    s = g.abs().amax((1, 3)).clamp(min=_LEAST) / _TOP
    q = (g / s[:, None, :, None]).reshape(-1, g.shape[2] * 128)[:x.shape[0], :x.shape[1]]
    return q.to(_E4M3), s


def _spread(q, s, rows, dtype):
    """The values that e4m3 numbers and their scales stand for."""
    g = _groups(q.to(dtype), rows) * s.to(dtype)[:, None, :, None]
    return g.reshape(-1, g.shape[2] * 128)[:q.shape[0], :q.shape[1]]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 41)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def uniform(n, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(n, generator=g, device="cuda")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if c["op"] == "norm":
        R, W, t = c["rows"], c["width"], _T[c["type"]]
        s = {"case": c, "x": normal(R, W, dtype=t), "weight": (1.0 - c["offset"] + normal(W, std=0.2)).to(_T[c["weight"]]), "residual": None, "sum": None,
             "out": empty(R, W, dtype=_E4M3), "scale": empty(R, -(-W // 128))}
        if c["residual"]:
            # a residual has a few columns that are far larger than the others
            r = normal(R, W, std=2.0) * (1.0 + 20.0 * (uniform(W) < 0.004).float())
            s["residual"], s["sum"] = r.to(_T[c["residual"]]), empty(R, W, dtype=_T[c["residual"]])
        return s
    if c["op"] == "e4m3":
        R, W = c["rows"], c["width"]
        # activations behind a unit are mostly small; weights are not
        x = normal(R, W).square_() if c["block"] == 1 else normal(R, W, std=W ** -0.5)
        return {"case": c, "x": x.to(_T[c["type"]]), "out": empty(R, W, dtype=_E4M3), "scale": empty(-(-R // c["block"]), -(-W // 128))}
    if c["op"] == "linear":
        T, K, N, o = c["tokens"], c["k"], c["n"], _T[c["out"]]
        x, xs = _to_e4m3(normal(T, K), 1)
        w, ws = _to_e4m3(normal(N, K, std=K ** -0.5), 128)
        return {"case": c, "x": x, "x_scale": xs, "w": w, "w_scale": ws, "base": normal(T, N, dtype=o) if c["base"] else None, "out": empty(T, N, dtype=o)}
    R, V = c["rows"], c["vocab"]
    s = {"case": c, "logits": normal(R, V, std=c["sharp"], dtype=_T[c["type"]]), "uniform": uniform(R), "temperature": uniform(R, 0.6, 1.4), "top_k": None,
         "top_p": None, "min_p": None, "tokens": empty(R, dtype=torch.int32), "probs": empty(R)}
    if c["greedy"]:
        s["temperature"][c["greedy"] - 1::c["greedy"]] = 0.0
    if c["top_k"]:
        s["top_k"] = (c["top_k"] * uniform(R, 1.0, 1.5)).to(torch.int32)
        s["top_k"][1::4] = 0                                    # requests without the limit
    if c["top_p"] < 1.0:
        s["top_p"] = (c["top_p"] + uniform(R, -0.05, 0.05)).clamp_(max=1.0)
    if c["min_p"]:
        s["min_p"] = c["min_p"] * uniform(R, 0.5, 1.5)
    return s


def run(state):
    s = state
    c = s["case"]
    if own:
        from ai00_server_b200 import device_ops
        if c["op"] == "norm":
            return device_ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=1e-5, offset=c["offset"], out=s["out"], scale=s["scale"], residual_out=s["sum"])
        if c["op"] == "e4m3":
            return device_ops.to_e4m3(s["x"], rows=c["block"], out=s["out"], scale=s["scale"])
        if c["op"] == "linear":
            return device_ops.linear_e4m3(s["x"], s["x_scale"], s["w"], s["w_scale"], base=s["base"], out=s["out"])
        return device_ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                 tokens=s["tokens"], probs=s["probs"])
    if c["op"] == "norm":
        return _plain_norm(s)
    if c["op"] == "e4m3":
        return _to_e4m3(s["x"].float(), c["block"])
    if c["op"] == "linear":
        y = _spread(s["x"], s["x_scale"], 1, torch.float32) @ _spread(s["w"], s["w_scale"], 128, torch.float32).t()
        return (y if s["base"] is None else s["base"].float() + y).to(_T[c["out"]])
    return _plain_sample(s)


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-5) * (s["case"]["offset"] + s["weight"].float())
    q, scale = _to_e4m3(y, 1)
    return q, scale, (None if s["residual"] is None else h.to(s["residual"].dtype))


def _plain_sample(s):
    """In 64 bits: a token is right or wrong, and the sums it is found by end next to one another."""
    l = s["logits"].double()
    R, V = l.shape
    T = s["temperature"].double()[:, None]
    d = l - l.max(1, keepdim=True).values
    w = torch.where(T > 0, torch.exp(d / T.clamp(min=1e-300)), (d == 0).double())
    _, order = l.sort(dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(V, device=l.device)
    k = torch.full((R, 1), V, device=l.device) if s["top_k"] is None else torch.where(s["top_k"] > 0, s["top_k"].long(), V)[:, None]
    ws = torch.where(rank < k, ws, 0.0)
    before = ws.cumsum(1) - ws
    keep = ws > 0
    if s["top_p"] is not None:
        keep &= (before < s["top_p"].double()[:, None] * ws.sum(1, keepdim=True)) | (s["top_p"][:, None] >= 1)
    if s["min_p"] is not None:
        keep &= ws >= s["min_p"].double()[:, None].clamp(max=1.0)
    keep[:, 0] = True
    keep &= (T > 0) | (rank == 0)
    kept = torch.zeros_like(w).scatter(1, order, torch.where(keep, ws, 0.0))
    sums = kept.cumsum(1)
    total = sums[:, -1:]
    token = ((sums <= s["uniform"].double()[:, None] * total).sum(1)).clamp(max=V - 1)
    return token.to(torch.int32), (kept.gather(1, token[:, None]) / total)[:, 0].float()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] in ("norm", "e4m3"):
        h = s["x"].double()
        y, block, total = h, 1, None
        if c["op"] == "norm":
            if s["residual"] is not None:
                total = h = h + s["residual"].double()
            y = h / (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / h.shape[1] + 1e-5).sqrt() * (s["weight"].double() + c["offset"])
        else:
            block = c["block"]
        R, W = y.shape
        scale = torch.empty(-(-R // block), -(-W // 128), dtype=torch.float64, device="cuda")
        q = torch.empty_like(y)
        top = y.abs() if block == 1 else torch.stack([y[i:i + block].abs().amax(0) for i in range(0, R, block)])
        for j in range(scale.shape[1]):
            cols = slice(128 * j, min(128 * j + 128, W))
            scale[:, j] = top[:, cols].amax(1).clamp(min=_LEAST) / _TOP
            q[:, cols] = y[:, cols] / scale[:, j].repeat_interleave(block)[:R, None]
        return (q, scale, total) if c["op"] == "norm" else (q, scale)
    if c["op"] == "linear":
        y = torch.zeros(c["tokens"], c["n"], dtype=torch.float64, device="cuda")
        of_row = torch.arange(c["n"], device="cuda") // 128
        for j in range(s["x_scale"].shape[1]):
            cols = slice(128 * j, 128 * j + 128)
            part = s["x"][:, cols].double() @ s["w"][:, cols].double().t()
            y += part * s["x_scale"][:, j, None].double() * s["w_scale"][of_row, j].double()
        return y if s["base"] is None else y + s["base"].double()
    logits, u, T = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy(), s["temperature"].double().cpu().numpy()
    at = lambda name, i, none: none if s[name] is None else s[name][i].item()  # noqa: E731
    tokens, probs = np.empty(c["rows"], np.int32), np.empty(c["rows"])
    for i, l in enumerate(logits):
        best = int(l.argmax())
        if T[i] == 0:
            tokens[i], probs[i] = best, 1.0
            continue
        w = np.exp((l - l[best]) / T[i])
        ids = np.lexsort((np.arange(l.size), -l))
        k = at("top_k", i, 0)
        ids = ids[:k] if k > 0 else ids
        p = at("top_p", i, 1.0)
        if p < 1:
            upto = np.cumsum(w[ids])
            ids = ids[:max(1, int(np.searchsorted(upto, p * upto[-1], side="left")) + 1)]
        least = min(at("min_p", i, 0.0), 1.0)
        ids = np.sort(ids[(w[ids] >= least) | (ids == best)])
        upto = np.cumsum(w[ids])
        j = min(int(np.searchsorted(upto, u[i] * upto[-1], side="right")), ids.size - 1)
        tokens[i], probs[i] = ids[j], w[ids[j]] / upto[-1]
    return torch.from_numpy(tokens), torch.from_numpy(probs)
