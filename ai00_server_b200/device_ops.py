"""Operators on tensors in GPU memory (b200rwkv_op_*, include/b200rwkv.h), for programs that hold theirs as torch tensors: what the engine runs on its own
buffers for the requests of a batch,

  low_rank   low-rank adapters of many requests beside shared projections
  logits     rows of logits adjusted by penalties, biases and grammar masks, as logits, probabilities or log-probabilities
  sample     a token for each row of logits, from given random numbers

and what stands in front of them in a step:

  rms_norm      the residual's addition and a root-mean-square norm, with its output in 8 bits (e4m3) and a scale for every 128 columns
  to_e4m3       rows or weights in 8 bits, with a scale for every 128 columns or every block of 128 x 128
  linear_e4m3   products of such rows and such weights

A call enqueues kernels on the current stream of its tensors' device and returns; it can be captured into a graph.  Arguments that
do not fit raise capi.B200Error before anything is enqueued, and so do tensors that ask for a gradient: the operators serve, they have none.

  lost_waits    waits in such kernels that ran out, on a device that does not get on: what hung on them is NaN
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import capi

_TYPE = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16, torch.float8_e4m3fn: capi.TYPE_E4M3}
_KIND = {"logits": capi.LOGITS, "probs": capi.PROBS, "log_probs": capi.LOG_PROBS}
# the structs of include/b200rwkv.h as bytes: a call for a few microseconds of work has no time for a store by field
_PART, _ADAPTERS, _LOGITS = struct.Struct("@PqPPPqPqiiii"), struct.Struct("@IiiiiiPPPN"), struct.Struct("@IiiiiiPqPqPPPPPPPPP")
_E4M3_ROWS, _NORM, _LINEAR, _SAMPLE = struct.Struct("@IiiiiiPqPqP"), struct.Struct("@IiiiiiiffiPqPqPqPPqP"), struct.Struct("@IiiiiiPqPPPPqPq"), struct.Struct("@IiiiPqPPPPPPP")
_I32, _F32, _E4M3 = torch.int32, torch.float32, torch.float8_e4m3fn
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


def _scales(t, name, n, m, where):
    """Address of contiguous f32 scales [n, m]: as many in another shape would be other blocks'."""
    if t.dtype is not _F32 or t.shape != (n, m) or t.get_device() != where or not t.is_contiguous():
        _bad(f"{name} must be a contiguous [{n}, {m}] {_F32} tensor on cuda:{where}")
    if t.requires_grad and torch.is_grad_enabled():
        _bad(f"{name} requires a gradient: these operators have none (call them under torch.no_grad())")
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


def to_e4m3(x, rows=1, out=None, scale=None):
    """x [n, width] (f32, f16 or bf16) in 8 bits: (out [n, width] float8_e4m3fn, scale f32) with x = out * scale, a scale for 128 neighbouring columns of a row
    (rows=1: scale [n, ceil(width / 128)], activations) or for a block of 128 rows of them (rows=128: scale [ceil(n / 128), ceil(width / 128)], weights).

    scale is the largest magnitude of its values (2^-100 at least) over 448, the largest e4m3 number."""
    dtype, where = x.dtype, x.get_device()
    if x.dim() != 2 or where < 0:
        _bad("to_e4m3: x must be a [rows, width] tensor in GPU memory")
    if rows != 1 and rows != 128:
        _bad("to_e4m3: a scale is for 1 or 128 rows")
    shape = x.shape
    n, width = shape
    down, across = -(-n // rows), -(-width // 128)
    if out is None:
        out = torch.empty(n, width, dtype=_E4M3, device=x.device)
    if scale is None:
        scale = torch.empty(down, across, dtype=_F32, device=x.device)
    q = _E4M3_ROWS.pack(_E4M3_ROWS.size, _TYPE.get(dtype, -1), n, width, rows, 0, x.data_ptr(), _row_stride(x, "x", shape, dtype, where), out.data_ptr(),
                        _row_stride(out, "out", shape, _E4M3, where), _scales(scale, "scale", down, across, where))
    code = capi.lib().b200rwkv_op_e4m3(where, _stream(where), q)
    if code < 0:
        capi.check(code)
    return out, scale


def rms_norm(x, weight=None, residual=None, eps=1e-5, offset=0.0, out=None, scale=None, residual_out=None, out_dtype=None):
    """h = x + residual;  residual_out = h;  y = h / sqrt(mean(h ** 2) + eps) * (offset + weight);  out, scale = y in 8 bits (to_e4m3), or out = y.

    x [n, width] is f32, f16 or bf16 (width up to 32768), residual and residual_out are of that type or f32, weight [width] any of the three (None: ones).  out is
    float8_e4m3fn with scale [n, ceil(width / 128)] f32, or, with out or out_dtype of the type of x, the rows themselves.  Sums are f32, and the norm reads h before it is
    rounded.  residual_out may be residual or x itself.  Returns (out, scale, residual_out), None for what is not there."""
    dtype, where = x.dtype, x.get_device()
    if x.dim() != 2 or where < 0:
        _bad("rms_norm: x must be a [rows, width] tensor in GPU memory")
    shape = x.shape
    n, width = shape
    if out is None:
        out = torch.empty(n, width, dtype=out_dtype or _E4M3, device=x.device)
    o_dtype = out.dtype
    w = s = r = ro = r_stride = ro_stride = 0
    w_type = r_type = _TYPE.get(dtype, -1)
    if weight is not None:
        w, w_type = _list(weight, "weight", weight.dtype, where, width), _TYPE.get(weight.dtype, -1)
    if o_dtype is _E4M3:
        if scale is None:
            scale = torch.empty(n, -(-width // 128), dtype=_F32, device=x.device)
        s = _scales(scale, "scale", n, -(-width // 128), where)
    elif scale is not None:
        _bad("rms_norm: scales come with an 8-bit out")
    if residual is not None:
        r_dtype = residual.dtype
        if residual_out is None:
            residual_out = torch.empty(n, width, dtype=r_dtype, device=x.device)
        r_type = _TYPE.get(r_dtype, -1)
        r, r_stride = residual.data_ptr(), _row_stride(residual, "residual", shape, r_dtype, where)
        ro, ro_stride = residual_out.data_ptr(), _row_stride(residual_out, "residual_out", shape, r_dtype, where)
    elif residual_out is not None:
        _bad("rms_norm: residual_out comes with a residual")
    q = _NORM.pack(_NORM.size, _TYPE.get(dtype, -1), r_type, w_type, _TYPE.get(o_dtype, -1), n, width, eps, offset, 0, x.data_ptr(), _row_stride(x, "x", shape, dtype, where),
                   r, r_stride, ro, ro_stride, w, out.data_ptr(), _row_stride(out, "out", shape, o_dtype, where), s)
    code = capi.lib().b200rwkv_op_norm(where, _stream(where), q)
    if code < 0:
        capi.check(code)
    return out, scale, residual_out


def linear_e4m3(x, x_scale, w, w_scale, base=None, out=None, out_dtype=None):
    """out[t, n] = base[t, n] + sum over blocks b of 128 inputs of x_scale[t, b] * w_scale[n // 128, b] * (x[t, b] @ w[n, b]).

    x [tokens, in] and w [out, in] are float8_e4m3fn as rms_norm and to_e4m3 make them (in a multiple of 16), x_scale [tokens, ceil(in / 128)] and w_scale
    [ceil(out / 128), ceil(in / 128)] f32; base and out [tokens, out] f32, f16 or bf16 (without either: out_dtype, or bf16).  `out` may be `base`.  Sums are f32."""
    where = x.get_device()
    if where < 0:
        _bad("linear_e4m3: tensors must be in GPU memory")
    if x.dim() != 2 or w.dim() != 2:
        _bad("linear_e4m3: x is [tokens, in], w is [out, in]")
    tokens, k = x.shape
    n, kw = w.shape
    if kw != k:
        _bad("linear_e4m3: shapes of x and w do not match")
    if out is None:
        out = torch.empty(tokens, n, dtype=out_dtype or (torch.bfloat16 if base is None else base.dtype), device=x.device)
    o_dtype, blocks = out.dtype, -(-k // 128)
    b = b_stride = 0
    if base is not None:
        b, b_stride = base.data_ptr(), _row_stride(base, "base", (tokens, n), o_dtype, where)
    q = _LINEAR.pack(_LINEAR.size, _TYPE.get(o_dtype, -1), tokens, k, n, 0, x.data_ptr(), _row_stride(x, "x", (tokens, k), _E4M3, where),
                     _scales(x_scale, "x_scale", tokens, blocks, where), _list(w, "w", _E4M3, where, None), _scales(w_scale, "w_scale", -(-n // 128), blocks, where),
                     b, b_stride, out.data_ptr(), _row_stride(out, "out", (tokens, n), o_dtype, where))
    code = capi.lib().b200rwkv_op_linear_e4m3(where, _stream(where), q)
    if code < 0:
        capi.check(code)
    return out


def sample(rows, uniform, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, probs=None):
    """A token for each row of logits [n, vocab] (f32, f16 or bf16) from uniform [n] f32 in [0, 1), as (tokens [n] int32, probs [n] f32).

    With w = exp((logit - largest) / temperature): kept are the row's first top_k tokens (larger logits first, of equal ones the lower id); of these the first so many that
    their weights reach top_p of all of these; of these the ones with w >= min_p.  The token is the lowest id at which the sum of kept weights, ids ascending, exceeds uniform times all
    of it, prob its share.  temperature, top_p, min_p [n] f32 and top_k [n] int32, None for 1 and no limits; temperature 0 takes the best token.  Logits of -inf are never drawn;
    a row of nothing else has token -1 and prob 0, one with a NaN token -1 and prob NaN.  The result does not depend on the order of any sum."""
    dtype, where = rows.dtype, rows.get_device()
    if rows.dim() != 2 or where < 0:
        _bad("sample: rows must be a [rows, vocab] tensor in GPU memory")
    shape = rows.shape
    n, vocab = shape
    if tokens is None:
        tokens = torch.empty(n, dtype=_I32, device=rows.device)
    if probs is None:
        probs = torch.empty(n, dtype=_F32, device=rows.device)
    t = 0 if temperature is None else _list(temperature, "temperature", _F32, where, n)
    k = 0 if top_k is None else _list(top_k, "top_k", _I32, where, n)
    p = 0 if top_p is None else _list(top_p, "top_p", _F32, where, n)
    m = 0 if min_p is None else _list(min_p, "min_p", _F32, where, n)
    q = _SAMPLE.pack(_SAMPLE.size, _TYPE.get(dtype, -1), n, vocab, rows.data_ptr(), _row_stride(rows, "rows", shape, dtype, where), _list(uniform, "uniform", _F32, where, n),
                     t, k, p, m, _list(tokens, "tokens", _I32, where, n), _list(probs, "probs", _F32, where, n))
    code = capi.lib().b200rwkv_op_sample(where, _stream(where), q)
    if code < 0:
        capi.check(code)
    return tokens, probs


def lost_waits(device=None):
    """Waits that ran out on a device (an index; None: the current one) in kernels of low_rank and linear_e4m3 that have ended: 0, or outputs that are NaN may be so for that reason."""
    total = ctypes.c_int64()
    capi.check(capi.lib().b200rwkv_op_lost_waits(torch.cuda.current_device() if device is None else device, ctypes.byref(total)))
    return total.value
