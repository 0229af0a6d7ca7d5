"""Operators on tensors in GPU memory (b200rwkv_op_*, include/b200rwkv.h): what the engine runs on its own buffers for the
requests of a batch, for programs that hold theirs as torch tensors.

  low_rank   low-rank adapters of many requests beside shared projections
  logits     rows of logits adjusted by penalties, biases and grammar masks, as logits, probabilities or log-probabilities

A call enqueues kernels on the current stream of its tensors' device and returns; it can be captured into a graph.  Arguments that
do not fit raise capi.B200Error before anything is enqueued.  Nothing here has a gradient: the operators serve.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import capi

_TYPE = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16}
_KIND = {"logits": capi.LOGITS, "probs": capi.PROBS, "log_probs": capi.LOG_PROBS}
_PARTS = [None] + [capi.AdapterPart * n for n in range(1, capi.MAX_PARTS + 1)]


def _bad(what: str):
    raise capi.B200Error(capi.ERR_INVALID, what)


def _check_list(t, name, dtype, device, size=None):
    """A contiguous vector or table of `dtype` on `device`; its address (None for None)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.device != device or not t.is_contiguous():
        _bad(f"{name} must be a contiguous {dtype} tensor on {device}")
    if size is not None and t.numel() != size:
        _bad(f"{name} has {t.numel()} elements, {size} are wanted")
    return t.data_ptr()


def _rows(t, name, rows, cols, dtype, device):
    """[rows, cols] with neighbouring columns; (address, elements between rows)."""
    if t.dtype is not dtype or t.device != device or t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
        _bad(f"{name} must be a [{rows}, {cols}] {dtype} tensor on {device}")
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        _bad(f"{name}: columns of a row must be neighbours")
    return t.data_ptr(), (s0 if rows > 1 else max(s0, cols))


def low_rank(x, a, b, index, scale, base=None, out=None, out_dtype=None):
    """out[t] = base[t] + scale[i] * (x[t] @ a[i].T) @ b[i].T with i = index[t]; tokens whose index names no adapter (negative, or beyond the
    last) keep their base, or zeros.

    x [tokens, in], a [adapters, rank, in], b [adapters, out, rank] are f16 or bf16 (one type; in and rank multiples of 8, rank <= 256); index
    [tokens] int32, scale [adapters] f32; base and out [tokens, out] are of that type or f32.  Lists of up to eight x, a, b, base and out
    stand for as many projections of the same tokens, served by one call.  `out` may be `base`: then only the tokens with an adapter are written.
    Returns out (a list for lists)."""
    many = isinstance(x, (list, tuple))
    if not many:
        x, a, b = [x], [a], [b]
        base = None if base is None else [base]
        out = None if out is None else [out]
    n = len(x)
    if not 1 <= n <= capi.MAX_PARTS or len(a) != n or len(b) != n or (base is not None and len(base) != n) or (out is not None and len(out) != n):
        _bad("x, a, b, base and out must be as many, at most 8")
    x0 = x[0]
    dtype, device = x0.dtype, x0.device
    if device.type != "cuda":
        _bad("low_rank: tensors must be in GPU memory")
    if x0.dim() != 2 or a[0].dim() != 3:
        _bad("low_rank: x is [tokens, in], a is [adapters, rank, in]")
    tokens, adapters = x0.shape[0], a[0].shape[0]
    if out is None:
        if out_dtype is None:
            out_dtype = dtype if base is None else base[0].dtype
        out = [torch.empty(tokens, w.shape[1] if w.dim() == 3 else 0, dtype=out_dtype, device=device) for w in b]
    o_dtype = out[0].dtype
    q = capi.Adapters()
    q.struct_bytes = C.sizeof(capi.Adapters)
    q.type, q.out_type = _TYPE.get(dtype, -1), _TYPE.get(o_dtype, -1)
    q.tokens, q.adapters, q.num_parts = tokens, adapters, n
    q.index = _check_list(index, "index", torch.int32, device, tokens)
    q.scale = _check_list(scale, "scale", torch.float32, device, adapters)
    parts = _PARTS[n]()
    for i in range(n):
        p, ai, bi = parts[i], a[i], b[i]
        if ai.dim() != 3 or bi.dim() != 3:
            _bad("low_rank: a is [adapters, rank, in], b is [adapters, out, rank]")
        _, rank, k = ai.shape
        width = bi.shape[1]
        if ai.shape[0] != adapters or bi.shape[0] != adapters or bi.shape[2] != rank:
            _bad("low_rank: shapes of a and b do not match")
        p.x, p.x_stride = _rows(x[i], "x", tokens, k, dtype, device)
        if tokens == 1:
            p.x_stride = k
        p.a = _check_list(ai, "a", dtype, device)
        p.b = _check_list(bi, "b", dtype, device)
        if base is not None:
            p.base, p.base_stride = _rows(base[i], "base", tokens, width, o_dtype, device)
        p.out, p.out_stride = _rows(out[i], "out", tokens, width, o_dtype, device)
        p.in_features, p.out_features, p.rank = k, width, rank
    q.parts = parts
    lib = capi.lib()
    need = lib.b200rwkv_op_adapters_workspace(tokens, adapters, n, max(w.shape[1] for w in a))
    if need > 0:
        work = torch.empty(need, dtype=torch.uint8, device=device)
        q.workspace, q.workspace_bytes = work.data_ptr(), need
    elif need < 0:
        capi.check(need)
    capi.check(lib.b200rwkv_op_adapters(device.index, torch.cuda.current_stream(device).cuda_stream, C.byref(q)))
    return out if many else out[0]


def logits(rows, kind="probs", controls=None, history=None, history_offset=None, history_from=None, allow=None, allow_row=None, bias_offset=None,
           bias_token=None, bias_value=None, out=None):
    """Rows of logits [n, vocab] (f32, f16 or bf16) adjusted for their requests, as `kind`: "logits", "probs" or "log_probs" (f32).

    controls [n, 5] f32: repetition, presence, frequency, decay, temperature of each row.  history: int32 tokens of all rows, oldest first, row i's
    from history_offset[i] to history_offset[i + 1]; a token in it has its logit divided (or, where it is not positive, multiplied) by repetition,
    and, where it is there at or behind place history_from[i] (None: everywhere), lowered by presence and by frequency times the sum of decay ** age
    over those places.  bias_offset, bias_token, bias_value: ragged lists of additions, of which a token's last counts.  allow [masks, (vocab + 31) // 32]
    int32 words: bit t % 32 of word t // 32 of mask allow_row[i] (None: i; no such mask: everything) says whether row i may hold token t.
    `out` may be `rows` itself where they are f32."""
    if rows.dim() != 2 or rows.device.type != "cuda":
        _bad("logits: rows must be a [rows, vocab] tensor in GPU memory")
    device = rows.device
    n, vocab = rows.shape
    if out is None:
        out = torch.empty(n, vocab, dtype=torch.float32, device=device)
    q = capi.Logits()
    q.struct_bytes = C.sizeof(capi.Logits)
    q.type, q.kind = _TYPE.get(rows.dtype, -1), _KIND.get(kind, -1)
    q.rows, q.vocab = n, vocab
    q.logits, q.logits_stride = _rows(rows, "rows", n, vocab, rows.dtype, device)
    q.out, q.out_stride = _rows(out, "out", n, vocab, torch.float32, device)
    if controls is not None:
        q.controls = _check_list(controls, "controls", torch.float32, device, n * 5)
    if history_offset is not None or history is not None:
        if history is None or history_offset is None:
            _bad("logits: history and history_offset come together")
        q.history_offset = _check_list(history_offset, "history_offset", torch.int32, device, n + 1)
        # (a tensor without elements has no address: no history at all)
        q.history = _check_list(history, "history", torch.int32, device) or q.history_offset
        q.history_from = _check_list(history_from, "history_from", torch.int32, device, n)
    if allow is not None:
        words = (vocab + 31) // 32
        if allow.dim() != 2 or allow.shape[1] != words:
            _bad(f"allow must be [masks, {words}]")
        q.allow, q.allow_rows = _check_list(allow, "allow", torch.int32, device), allow.shape[0]
        q.allow_row = _check_list(allow_row, "allow_row", torch.int32, device, n)
    if bias_offset is not None or bias_token is not None:
        if bias_offset is None or bias_token is None or bias_value is None or bias_token.numel() != bias_value.numel():
            _bad("logits: bias_offset, bias_token and bias_value come together, a value for each token")
        q.bias_offset = _check_list(bias_offset, "bias_offset", torch.int32, device, n + 1)
        q.bias_token = _check_list(bias_token, "bias_token", torch.int32, device) or q.bias_offset
        q.bias_value = _check_list(bias_value, "bias_value", torch.float32, device) or q.bias_offset
    capi.check(capi.lib().b200rwkv_op_logits(device.index, torch.cuda.current_stream(device).cuda_stream, C.byref(q)))
    return out
