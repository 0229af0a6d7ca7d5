"""Refusals of the operators on device memory: every wrong argument that the host can see is an error before anything is enqueued (no GPU needed)."""
import ctypes as C

import pytest

from ai00_server_b200 import capi


def _adapters(**change):
    part = capi.AdapterPart(x=4096, x_stride=64, a=4096, b=4096, base=4096, base_stride=32, out=8192, out_stride=32, in_features=64, out_features=32, rank=16)
    q = capi.Adapters(struct_bytes=C.sizeof(capi.Adapters), type=capi.TYPE_F16, out_type=capi.TYPE_F32, tokens=4, adapters=2, num_parts=1, index=4096, scale=4096)
    for k, v in change.items():
        if k != "parts":
            setattr(part if hasattr(part, k) else q, k, v)
    return C.byref(q), (C.byref(part) if change.get("parts", 1) else None)


@pytest.mark.parametrize("change,code", [
    ({"struct_bytes": 8}, capi.ERR_INVALID), ({"type": capi.TYPE_F32}, capi.ERR_UNSUPPORTED), ({"type": 9}, capi.ERR_UNSUPPORTED),
    ({"out_type": capi.TYPE_BF16}, capi.ERR_UNSUPPORTED), ({"tokens": -1}, capi.ERR_INVALID), ({"tokens": (1 << 20) + 1}, capi.ERR_INVALID),
    ({"adapters": 0}, capi.ERR_INVALID), ({"adapters": 1025}, capi.ERR_INVALID), ({"num_parts": 0}, capi.ERR_INVALID), ({"num_parts": 9}, capi.ERR_INVALID),
    ({"parts": None}, capi.ERR_INVALID), ({"index": None}, capi.ERR_INVALID), ({"scale": None}, capi.ERR_INVALID),
    ({"in_features": 60}, capi.ERR_UNSUPPORTED), ({"in_features": 0}, capi.ERR_UNSUPPORTED), ({"out_features": 0}, capi.ERR_INVALID),
    ({"rank": 12}, capi.ERR_UNSUPPORTED), ({"rank": 264}, capi.ERR_UNSUPPORTED), ({"rank": 0}, capi.ERR_UNSUPPORTED), ({"x": None}, capi.ERR_INVALID),
    ({"a": None}, capi.ERR_INVALID), ({"b": None}, capi.ERR_INVALID), ({"out": None}, capi.ERR_INVALID), ({"x": 4098}, capi.ERR_INVALID),
    ({"a": 4104}, capi.ERR_INVALID), ({"b": 4104}, capi.ERR_INVALID), ({"x_stride": 68}, capi.ERR_INVALID), ({"x_stride": 56}, capi.ERR_INVALID),
    ({"out_stride": 31}, capi.ERR_INVALID), ({"base_stride": 31}, capi.ERR_INVALID), ({"out": 8194}, capi.ERR_INVALID),
    ({"out": 4096}, capi.ERR_INVALID), ({"base": 8192, "base_stride": 64}, capi.ERR_INVALID),       # its own x; the same rows with another stride
    ({"tokens": 300}, capi.ERR_INVALID),                                             # no workspace
    ({"tokens": 300, "workspace": 4096, "workspace_bytes": 64}, capi.ERR_INVALID),
    ({"tokens": 300, "workspace": 4100, "workspace_bytes": 1 << 20}, capi.ERR_INVALID)])
def test_op_adapters_refuses(change, code):
    with pytest.raises(capi.B200Error) as ei:
        capi.check(capi.lib().b200rwkv_op_adapters(0, None, *_adapters(**change)))
    assert ei.value.code == code
    assert "op_adapters" in str(ei.value)


@pytest.mark.parametrize("change", [{"out": 8192}, {"base": 8192}, {"x": 8192}, {"x": 12288 + 4096, "out": 4096}])
def test_op_adapters_refuses_parts_that_write_what_another_reads(change):
    def part(**c):
        return capi.AdapterPart(**{**dict(x=4096, x_stride=64, a=4096, b=4096, base=12288, base_stride=32, out=12288, out_stride=32, in_features=64, out_features=32, rank=16), **c})
    parts = (capi.AdapterPart * 2)(part(base=8192, out=8192), part(**change))
    q = capi.Adapters(struct_bytes=C.sizeof(capi.Adapters), type=capi.TYPE_F16, out_type=capi.TYPE_F32, tokens=4, adapters=2, num_parts=2, index=4096, scale=4096)
    with pytest.raises(capi.B200Error, match="of another") as ei:
        capi.check(capi.lib().b200rwkv_op_adapters(0, None, C.byref(q), parts))
    assert ei.value.code == capi.ERR_INVALID


@pytest.mark.parametrize("change,what", [
    ({"out": 4096 + 64, "base": None}, "own x"),                                          # rows of out inside rows of x
    ({"out": 4096 - 64, "base": None}, "own x"),
    ({"base": 8192 + 4, "out": 8192}, "own base"),                                         # one column further
    ({"base": 8192 + 3 * 128, "out": 8192}, "own base"),                                   # three rows further
    ({"base": 8192, "out": 8192 + 128 - 4, "base_stride": 64, "out_stride": 64}, "own base")])
def test_op_adapters_refuses_rows_that_overlap(change, what):
    """Not the same rows, but some of the same bytes (x: four rows of 128 bytes at 4096; out and base: 128 bytes a row, here at distances of 128 or 256)."""
    args = {**dict(base=12288, out=8192), **change}
    with pytest.raises(capi.B200Error, match=what) as ei:
        capi.check(capi.lib().b200rwkv_op_adapters(0, None, *_adapters(**args)))
    assert ei.value.code == capi.ERR_INVALID


@pytest.mark.parametrize("change", [{"out": 8192 + 128, "base": None}, {"base": 8192 + 384}, {"x": 8192 + 496}, {"out": 4096 + 64, "base": None}])
def test_op_adapters_refuses_parts_that_overlap(change):
    def part(**c):
        return capi.AdapterPart(**{**dict(x=4096, x_stride=64, a=4096, b=4096, base=16384, base_stride=32, out=16384, out_stride=32, in_features=64, out_features=32, rank=16), **c})
    parts = (capi.AdapterPart * 2)(part(base=8192, out=8192), part(**change))
    q = capi.Adapters(struct_bytes=C.sizeof(capi.Adapters), type=capi.TYPE_F16, out_type=capi.TYPE_F32, tokens=4, adapters=2, num_parts=2, index=4096, scale=4096)
    with pytest.raises(capi.B200Error, match="of another") as ei:
        capi.check(capi.lib().b200rwkv_op_adapters(0, None, C.byref(q), parts))
    assert ei.value.code == capi.ERR_INVALID


@pytest.mark.parametrize("change", [
    {"out": 4096 + 4}, {"out": 4096 + 400}, {"logits": 4096 + 796}, {"out": 4096 + 396, "logits_stride": 200, "out_stride": 200},
    {"type": capi.TYPE_F16, "out": 4096 + 396}, {"type": capi.TYPE_BF16, "logits": 4096 + 796, "out": 4096}])
def test_op_logits_refuses_rows_that_overlap(change):
    """Two rows of 100 tokens: 800 bytes of f32 or 400 of f16 from 4096 on."""
    with pytest.raises(capi.B200Error, match="overlap") as ei:
        capi.check(capi.lib().b200rwkv_op_logits(0, None, C.byref(_logits(**{**dict(logits=4096, out=4096), **change}))))
    assert ei.value.code == capi.ERR_INVALID


def test_op_adapters_null_struct_and_no_tokens():
    assert capi.lib().b200rwkv_op_adapters(0, None, None, None) == capi.ERR_INVALID
    assert capi.lib().b200rwkv_op_adapters(0, None, *_adapters(tokens=0, index=None, scale=None, x=None, out=None)) == 0


def test_op_adapters_workspace():
    f = capi.lib().b200rwkv_op_adapters_workspace
    assert f(256, 4, 1, 16) == 0
    assert f(257, 4, 1, 16) > 257 * 4
    assert f(1000, 4, 1, 16) < f(1000, 4, 2, 16) and f(1000, 4, 1, 64) < f(1000, 4, 1, 65)
    for bad in [(-1, 4, 1, 16), ((1 << 20) + 1, 4, 1, 16), (8, 0, 1, 16), (8, 1025, 1, 16), (8, 4, 0, 16), (8, 4, 9, 16), (8, 4, 1, 0), (8, 4, 1, 257)]:
        assert f(*bad) == capi.ERR_INVALID


def test_op_adapters_workspace_keeps_projections_on_boundaries():
    """What a further projection adds to the workspace is a multiple of sixteen bytes, whatever the tokens and the rank: every projection's S starts where
    sixteen-byte accesses may."""
    f = capi.lib().b200rwkv_op_adapters_workspace
    for tokens in [*range(257, 1025), 1021, 4099, 65537, 1 << 20]:
        for rank in range(1, capi.MAX_RANK + 1):
            assert (f(tokens, 4, 2, rank) - f(tokens, 4, 1, rank)) % 16 == 0, (tokens, rank)
        assert (f(tokens, 4, 8, 256) - f(tokens, 4, 1, 256)) % 16 == 0, tokens


def _logits(**change):
    q = capi.Logits(struct_bytes=C.sizeof(capi.Logits), type=capi.TYPE_F32, kind=capi.PROBS, rows=2, vocab=100, logits=4096, logits_stride=100, out=8192, out_stride=100)
    for k, v in change.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("change,code", [
    ({"struct_bytes": 4}, capi.ERR_INVALID), ({"type": 3}, capi.ERR_UNSUPPORTED), ({"type": -1}, capi.ERR_UNSUPPORTED), ({"kind": 3}, capi.ERR_INVALID),
    ({"kind": -1}, capi.ERR_INVALID), ({"rows": -1}, capi.ERR_INVALID), ({"vocab": 0}, capi.ERR_INVALID), ({"logits": None}, capi.ERR_INVALID),
    ({"out": None}, capi.ERR_INVALID), ({"logits_stride": 99}, capi.ERR_INVALID), ({"out_stride": 99}, capi.ERR_INVALID), ({"logits": 4098}, capi.ERR_INVALID),
    ({"out": 8194}, capi.ERR_INVALID), ({"history_offset": 4096}, capi.ERR_INVALID), ({"bias_offset": 4096}, capi.ERR_INVALID),
    ({"bias_offset": 4096, "bias_token": 4096}, capi.ERR_INVALID), ({"allow": 4096, "allow_rows": 1}, capi.ERR_INVALID),
    ({"allow": 4096, "allow_rows": -1, "allow_row": 4096}, capi.ERR_INVALID), ({"vocab": 524289, "logits_stride": 1 << 20, "out_stride": 1 << 20}, capi.ERR_UNSUPPORTED),
    ({"rows": (1 << 24) + 1}, capi.ERR_INVALID), ({"out": 4096, "type": capi.TYPE_F16}, capi.ERR_INVALID), ({"out": 4096, "out_stride": 128}, capi.ERR_INVALID)])
def test_op_logits_refuses(change, code):
    with pytest.raises(capi.B200Error) as ei:
        capi.check(capi.lib().b200rwkv_op_logits(0, None, C.byref(_logits(**change))))
    assert ei.value.code == code
    assert "op_logits" in str(ei.value)


def test_op_logits_null_struct_and_no_rows():
    assert capi.lib().b200rwkv_op_logits(0, None, None) == capi.ERR_INVALID
    assert capi.lib().b200rwkv_op_logits(0, None, C.byref(_logits(rows=0, logits=None, out=None))) == 0


def test_tensors_that_do_not_fit():
    torch = pytest.importorskip("torch")
    from ai00_server_b200 import device_ops
    x, a, b = torch.zeros(4, 64), torch.zeros(2, 8, 64), torch.zeros(2, 16, 8)
    with pytest.raises(capi.B200Error):              # not in GPU memory
        device_ops.low_rank(x, a, b, torch.zeros(4, dtype=torch.int32), torch.ones(2))
    with pytest.raises(capi.B200Error):
        device_ops.low_rank([x], [a, a], [b], torch.zeros(4, dtype=torch.int32), torch.ones(2))
    with pytest.raises(capi.B200Error):
        device_ops.logits(torch.zeros(2, 10))
    with pytest.raises(capi.B200Error):
        device_ops.logits(torch.zeros(20))


def test_structs_match_the_header(tmp_path):
    """Sizes and offsets of the operators' structs, as a C compiler has them."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = {"b200rwkv_adapter_part": capi.AdapterPart, "b200rwkv_adapters": capi.Adapters, "b200rwkv_logits": capi.Logits, "b200rwkv_row_controls": capi.RowControls}
    lines = []
    for name, cls in pairs.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        lines += [f'printf("%zu ", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "b200rwkv.h"\nint main(void) { ' + "\n".join(lines) + " return 0; }\n")
    exe = tmp_path / "s"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    want = []
    for cls in pairs.values():
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
    header = open(os.path.join(root, "include", "b200rwkv.h")).read()
    for name, value in [("MAX_PARTS", capi.MAX_PARTS), ("MAX_RANK", capi.MAX_RANK), ("MAX_ADAPTERS", capi.MAX_ADAPTERS), ("TYPE_F32", capi.TYPE_F32), ("TYPE_F16", capi.TYPE_F16),
                        ("TYPE_BF16", capi.TYPE_BF16), ("LOGITS", capi.LOGITS), ("PROBS", capi.PROBS), ("LOG_PROBS", capi.LOG_PROBS)]:
        assert f"#define B200RWKV_{name} {value}\n" in header, name
    from ai00_server_b200 import device_ops
    assert (device_ops._PART.size, device_ops._ADAPTERS.size, device_ops._LOGITS.size) == tuple(C.sizeof(c) for c in (capi.AdapterPart, capi.Adapters, capi.Logits))
    assert f"#define B200RWKV_ADAPTERS_WITHOUT_WORKSPACE {capi.ADAPTERS_WITHOUT_WORKSPACE} " in header


def test_engine_calls_refuse_null():
    lib = capi.lib()
    aid = C.c_uint64(5)
    assert lib.b200rwkv_adapter_load(None, None, 0, 1.0, C.byref(aid)) == capi.ERR_INVALID
    assert lib.b200rwkv_adapter_free(None, 1) == capi.ERR_INVALID
    assert lib.b200rwkv_slot_adapter(None, 0, 1) == capi.ERR_INVALID
    assert lib.b200rwkv_sample_rows(None, 1, C.byref(capi.RowControls()), None) == capi.ERR_INVALID


def test_a_freed_or_foreign_adapter_is_not_bound():
    """A handle that was freed must not unbind the slot as if it were None, nor one of another model bind what has its number here."""
    from ai00_server_b200 import runtime
    one, other = runtime.Model.__new__(runtime.Model), runtime.Model.__new__(runtime.Model)
    one._h = other._h = None
    with pytest.raises(capi.B200Error, match="freed") as ei:
        one.set_adapter(0, runtime.Adapter(one, 0))
    assert ei.value.code == capi.ERR_STATE
    with pytest.raises(capi.B200Error, match="another model") as ei:
        one.set_adapter(0, runtime.Adapter(other, 3))
    assert ei.value.code == capi.ERR_STATE
    for adapter in (None, runtime.Adapter(one, 3)):          # what the engine itself decides
        with pytest.raises(capi.B200Error, match="null engine"):
            one.set_adapter(0, adapter)
