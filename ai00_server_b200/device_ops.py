"""Operators on tensors in GPU memory (b200rwkv_op_*, include/b200rwkv.h): what the engine runs on its own buffers for the
requests of a batch, for programs that hold theirs as torch tensors.

  low_rank   low-rank adapters of many requests beside shared projections
  logits     rows of logits adjusted by penalties, biases and grammar masks, as logits, probabilities or log-probabilities

A call enqueues kernels on the current stream of its tensors' device and returns; it can be captured into a graph.  Arguments that
do not fit raise capi.B200Error before anything is enqueued, and so do tensors that ask for a gradient: the operators serve, they have none.
"""
from __future__ import annotations

import struct

import torch

from . import capi

_TYPE = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16}
_KIND = {"logits": capi.LOGITS, "probs": capi.PROBS, "log_probs": capi.LOG_PROBS}
# b200rwkv_adapter_part, b200rwkv_adapters and b200rwkv_logits as bytes: a call for a few microseconds of work has no time for a store by field
_PART, _ADAPTERS, _LOGITS = struct.Struct("@PqPPPqPqiiii"), struct.Struct("@IiiiiiPPPN"), struct.Struct("@IiiiiiPqPqPPPPPPPPP")
_I32, _F32 = torch.int32, torch.float32
_stream = torch._C._cuda_getCurrentRawStream        # the current stream of a device as a number


def _bad(what: str):
    raise capi.B200Error(capi.ERR_INVALID, what)


def _list(t, name, dtype, where, size):
    """Address of a contiguous vector or table of `dtype` on device `where` with `size` elements (None: any number)."""
    if t.dtype is not dtype or t.get_device() != where or not t.is_contiguous():
        _bad(f"{name} must be a contiguous {dtype} tensor on cuda:{where}")
    if t.requires_grad and torch.is_grad_enabled():
        _bad(f"{name} requires a gradient: these operators have none (call them under torch.no_grad())")
    if size is not None and t.numel() != size:
        _bad(f"{name} has {t.numel()} elements, {size} are wanted")
    return t.data_ptr()


def _row_stride(t, name, shape, dtype, where):
    """Elements between the rows of a [rows, cols] tensor with neighbouring columns."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != where:
        _bad(f"{name} must be a {list(shape)} {dtype} tensor on cuda:{where}")
    if t.requires_grad and torch.is_grad_enabled():
        _bad(f"{name} requires a gradient: these operators have none (call them under torch.no_grad())")
    s0, s1 = t.stride()
    if s1 != 1 and shape[1] > 1:
        _bad(f"{name}: columns of a row must be neighbours")
    return s0 if shape[0] > 1 else shape[1]


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
    dtype, where = x0.dtype, x0.get_device()
    if where < 0:
        _bad("low_rank: tensors must be in GPU memory")
    if x0.dim() != 2 or a[0].dim() != 3 or b[0].dim() != 3:
        _bad("low_rank: x is [tokens, in], a is [adapters, rank, in], b is [adapters, out, rank]")
    tokens, adapters = x0.shape[0], a[0].shape[0]
    if out is None:
        if out_dtype is None:
            out_dtype = dtype if base is None else base[0].dtype
        out = [torch.empty(tokens, w.shape[1], dtype=out_dtype, device=x0.device) for w in b]
    o_dtype = out[0].dtype
    parts, top = b"", 1
    for i in range(n):
        ai, bi, xi, oi = a[i], b[i], x[i], out[i]
        if ai.dim() != 3 or bi.dim() != 3:
            _bad("low_rank: a is [adapters, rank, in], b is [adapters, out, rank]")
        m, rank, k = ai.shape
        mb, width, rb = bi.shape
        if m != adapters or mb != adapters or rb != rank:
            _bad("low_rank: shapes of a and b do not match")
        if rank > top:
            top = rank
        shape = (tokens, width)
        at, stride = 0, 0
        if base is not None:
            at, stride = base[i].data_ptr(), _row_stride(base[i], "base", shape, o_dtype, where)
        parts += _PART.pack(xi.data_ptr(), _row_stride(xi, "x", (tokens, k), dtype, where), _list(ai, "a", dtype, where, None), _list(bi, "b", dtype, where, None),
                            at, stride, oi.data_ptr(), _row_stride(oi, "out", shape, o_dtype, where), k, width, rank, 0)
    lib = capi.lib()
    work, need = None, 0
    if tokens > capi.ADAPTERS_WITHOUT_WORKSPACE:
        need = lib.b200rwkv_op_adapters_workspace(tokens, adapters, n, min(top, capi.MAX_RANK))
        capi.check(min(need, 0))
        work = torch.empty(need, dtype=torch.uint8, device=x0.device)
    q = _ADAPTERS.pack(_ADAPTERS.size, _TYPE.get(dtype, -1), _TYPE.get(o_dtype, -1), tokens, adapters, n, _list(index, "index", _I32, where, tokens),
                       _list(scale, "scale", _F32, where, adapters), 0 if work is None else work.data_ptr(), need)
    code = lib.b200rwkv_op_adapters(where, _stream(where), q, parts)
    if code < 0:
        capi.check(code)
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
    dtype, where = rows.dtype, rows.get_device()
    if rows.dim() != 2 or where < 0:
        _bad("logits: rows must be a [rows, vocab] tensor in GPU memory")
    shape = rows.shape
    n, vocab = shape
    if out is None:
        out = torch.empty(n, vocab, dtype=_F32, device=rows.device)
    c = ho = h = hf = al = ar = bo = bt = bv = masks = 0
    if controls is not None:
        c = _list(controls, "controls", _F32, where, n * 5)
    if history_offset is not None or history is not None:
        if history is None or history_offset is None:
            _bad("logits: history and history_offset come together")
        ho = _list(history_offset, "history_offset", _I32, where, n + 1)
        h = _list(history, "history", _I32, where, None) or ho            # (a tensor without elements has no address)
        if history_from is not None:
            hf = _list(history_from, "history_from", _I32, where, n)
    if allow is not None:
        words = (vocab + 31) // 32
        if allow.dim() != 2 or allow.shape[1] != words:
            _bad(f"allow must be [masks, {words}]")
        masks = allow.shape[0]
        al = _list(allow, "allow", _I32, where, None)
        if allow_row is not None:
            ar = _list(allow_row, "allow_row", _I32, where, n)
    if bias_offset is not None or bias_token is not None:
        if bias_offset is None or bias_token is None or bias_value is None or bias_token.numel() != bias_value.numel():
            _bad("logits: bias_offset, bias_token and bias_value come together, a value for each token")
        bo = _list(bias_offset, "bias_offset", _I32, where, n + 1)
        bt = _list(bias_token, "bias_token", _I32, where, None) or bo
        bv = _list(bias_value, "bias_value", _F32, where, None) or bo
    q = _LOGITS.pack(_LOGITS.size, _TYPE.get(dtype, -1), _KIND.get(kind, -1), n, vocab, masks, rows.data_ptr(), _row_stride(rows, "rows", shape, dtype, where),
                     out.data_ptr(), _row_stride(out, "out", shape, _F32, where), c, ho, h, hf, al, ar, bo, bt, bv)
    code = capi.lib().b200rwkv_op_logits(where, _stream(where), q)
    if code < 0:
        capi.check(code)
    return out
