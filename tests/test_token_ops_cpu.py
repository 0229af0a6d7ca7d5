"""Refusals of the operators from residual rows to tokens: every wrong argument that the host can see is an error before anything is enqueued (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest

from ai00_server_b200 import capi

INVALID, UNSUPPORTED = capi.ERR_INVALID, capi.ERR_UNSUPPORTED
STRUCTS = {"b200rwkv_e4m3": capi.E4m3, "b200rwkv_norm": capi.Norm, "b200rwkv_linear_e4m3": capi.LinearE4m3, "b200rwkv_sample": capi.Sample, "b200rwkv_draw": capi.Draw}


def made(cls, fields, change):
    q = cls(struct_bytes=C.sizeof(cls), **fields)
    for k, v in change.items():
        setattr(q, k, v)
    return q


# addresses far apart: nothing is read
E4M3 = dict(type=capi.TYPE_F16, rows=4, width=100, block_rows=1, x=1 << 20, x_stride=100, out=2 << 20, out_stride=100, scale=3 << 20)
NORM = dict(type=capi.TYPE_F16, residual_type=capi.TYPE_F32, weight_type=capi.TYPE_F32, out_type=capi.TYPE_E4M3, rows=4, width=100, eps=1e-5, x=1 << 20, x_stride=100,
            residual=2 << 20, residual_stride=100, residual_out=3 << 20, residual_out_stride=100, weight=4 << 20, out=5 << 20, out_stride=100, scale=6 << 20)
LINEAR = dict(out_type=capi.TYPE_BF16, tokens=4, in_features=144, out_features=100, x=1 << 20, x_stride=144, x_scale=2 << 20, w=3 << 20, w_scale=4 << 20, base=5 << 20, base_stride=100,
              out=6 << 20, out_stride=100)
SAMPLE = dict(type=capi.TYPE_F32, rows=4, vocab=100, logits=1 << 20, logits_stride=100, uniform=2 << 20, temperature=3 << 20, top_k=4 << 20, top_p=5 << 20, min_p=6 << 20, tokens=7 << 20,
              probs=8 << 20)
CALLS = {"op_e4m3": (capi.E4m3, E4M3), "op_norm": (capi.Norm, NORM), "op_linear_e4m3": (capi.LinearE4m3, LINEAR), "op_sample": (capi.Sample, SAMPLE)}
KB = 1 << 10


@pytest.mark.parametrize("call,change,code", [
    ("op_e4m3", {"struct_bytes": 8}, INVALID), ("op_e4m3", {"type": 3}, UNSUPPORTED), ("op_e4m3", {"type": -1}, UNSUPPORTED), ("op_e4m3", {"block_rows": 64}, UNSUPPORTED),
    ("op_e4m3", {"block_rows": 0}, UNSUPPORTED), ("op_e4m3", {"rows": -1}, INVALID), ("op_e4m3", {"rows": (1 << 24) + 1}, INVALID), ("op_e4m3", {"width": 0}, INVALID),
    ("op_e4m3", {"width": (1 << 24) + 1}, INVALID), ("op_e4m3", {"x": None}, INVALID), ("op_e4m3", {"out": None}, INVALID), ("op_e4m3", {"scale": None}, INVALID),
    ("op_e4m3", {"x_stride": 99}, INVALID), ("op_e4m3", {"out_stride": 99}, INVALID), ("op_e4m3", {"x": (1 << 20) + 1}, INVALID), ("op_e4m3", {"scale": (3 << 20) + 2}, INVALID),
    ("op_e4m3", {"out": (1 << 20) + 798}, INVALID), ("op_e4m3", {"scale": (1 << 20) + 796}, INVALID), ("op_e4m3", {"scale": (2 << 20) + 396}, INVALID), ("op_e4m3", {"out": 1 << 20}, INVALID),
    ("op_e4m3", {"rows": 1 << 24, "width": 1 << 24, "x_stride": 1 << 24, "out_stride": 1 << 24, "x": 1 << 52, "out": 1 << 54, "scale": 1 << 56}, UNSUPPORTED),
    ("op_norm", {"struct_bytes": 8}, INVALID), ("op_norm", {"type": 3}, UNSUPPORTED), ("op_norm", {"residual_type": capi.TYPE_BF16}, UNSUPPORTED), ("op_norm", {"weight_type": 3}, UNSUPPORTED),
    ("op_norm", {"out_type": capi.TYPE_F32}, UNSUPPORTED), ("op_norm", {"rows": -1}, INVALID), ("op_norm", {"width": 0}, INVALID), ("op_norm", {"eps": -1.0}, INVALID),
    ("op_norm", {"eps": float("nan")}, INVALID),
    ("op_norm", {"width": 32769, "x_stride": 1 << 16, "out_stride": 1 << 16, "residual_stride": 1 << 16, "residual_out_stride": 1 << 16}, UNSUPPORTED),
    ("op_norm", {"x": None}, INVALID), ("op_norm", {"out": None}, INVALID), ("op_norm", {"scale": None}, INVALID), ("op_norm", {"residual": None}, INVALID),
    ("op_norm", {"residual_out": None}, INVALID), ("op_norm", {"x_stride": 99}, INVALID), ("op_norm", {"residual_stride": 99}, INVALID), ("op_norm", {"residual_out_stride": 99}, INVALID),
    ("op_norm", {"out_stride": 99}, INVALID), ("op_norm", {"x": (1 << 20) + 1}, INVALID), ("op_norm", {"residual": (2 << 20) + 2}, INVALID), ("op_norm", {"weight": (4 << 20) + 2}, INVALID),
    ("op_norm", {"out": 1 << 20}, INVALID), ("op_norm", {"out": (2 << 20) + 8}, INVALID), ("op_norm", {"out": 3 << 20}, INVALID), ("op_norm", {"out": (4 << 20) + 396}, INVALID),
    ("op_norm", {"scale": 1 << 20}, INVALID), ("op_norm", {"scale": 2 << 20}, INVALID), ("op_norm", {"scale": 3 << 20}, INVALID), ("op_norm", {"scale": 4 << 20}, INVALID),
    ("op_norm", {"scale": 5 << 20}, INVALID), ("op_norm", {"residual_out": (2 << 20) + 4}, INVALID), ("op_norm", {"residual_out": 1 << 20}, INVALID),
    ("op_norm", {"residual_out": 2 << 20, "residual_out_stride": 104}, INVALID), ("op_norm", {"residual_out": 4 << 20}, INVALID),
    ("op_norm", {"residual_type": capi.TYPE_F16, "residual_out": (1 << 20) + 2}, INVALID),
    ("op_linear_e4m3", {"struct_bytes": 8}, INVALID), ("op_linear_e4m3", {"out_type": 3}, UNSUPPORTED), ("op_linear_e4m3", {"tokens": -1}, INVALID),
    ("op_linear_e4m3", {"tokens": (1 << 20) + 1}, INVALID), ("op_linear_e4m3", {"in_features": 136}, UNSUPPORTED), ("op_linear_e4m3", {"in_features": 0}, UNSUPPORTED),
    ("op_linear_e4m3", {"out_features": 0}, INVALID), ("op_linear_e4m3", {"x": None}, INVALID), ("op_linear_e4m3", {"w": None}, INVALID), ("op_linear_e4m3", {"x_scale": None}, INVALID),
    ("op_linear_e4m3", {"w_scale": None}, INVALID), ("op_linear_e4m3", {"out": None}, INVALID), ("op_linear_e4m3", {"x_stride": 128}, INVALID), ("op_linear_e4m3", {"x_stride": 152}, INVALID),
    ("op_linear_e4m3", {"x": (1 << 20) + 8}, INVALID), ("op_linear_e4m3", {"w": (3 << 20) + 8}, INVALID), ("op_linear_e4m3", {"out": (6 << 20) + 1}, INVALID),
    ("op_linear_e4m3", {"base": (5 << 20) + 1}, INVALID), ("op_linear_e4m3", {"out_stride": 99}, INVALID), ("op_linear_e4m3", {"base_stride": 99}, INVALID),
    ("op_linear_e4m3", {"base": 6 << 20, "base_stride": 104}, INVALID), ("op_linear_e4m3", {"base": (6 << 20) + 2}, INVALID), ("op_linear_e4m3", {"out": 1 << 20}, INVALID),
    ("op_linear_e4m3", {"out": 2 << 20}, INVALID), ("op_linear_e4m3", {"out": (3 << 20) + 14000}, INVALID), ("op_linear_e4m3", {"out": 4 << 20}, INVALID),
    ("op_linear_e4m3", {"x_scale": (2 << 20) + 1}, INVALID),
    ("op_sample", {"struct_bytes": 8}, INVALID), ("op_sample", {"type": 3}, UNSUPPORTED), ("op_sample", {"rows": -1}, INVALID), ("op_sample", {"vocab": 0}, INVALID),
    ("op_sample", {"vocab": 524289, "logits_stride": 1 << 20}, UNSUPPORTED), ("op_sample", {"logits": None}, INVALID), ("op_sample", {"uniform": None}, INVALID),
    ("op_sample", {"tokens": None}, INVALID), ("op_sample", {"logits_stride": 99}, INVALID), ("op_sample", {"logits": (1 << 20) + 2}, INVALID), ("op_sample", {"top_p": (5 << 20) + 2}, INVALID),
    ("op_sample", {"tokens": 1 << 20}, INVALID), ("op_sample", {"tokens": 2 << 20}, INVALID), ("op_sample", {"tokens": (4 << 20) + 12}, INVALID), ("op_sample", {"probs": 7 << 20}, INVALID),
    ("op_sample", {"probs": (1 << 20) + 1596}, INVALID), ("op_sample", {"probs": 6 << 20}, INVALID)])
def test_refused(call, change, code):
    cls, fields = CALLS[call]
    with pytest.raises(capi.B200Error) as ei:
        capi.check(getattr(capi.lib(), "b200rwkv_" + call)(0, None, C.byref(made(cls, fields, change))))
    assert ei.value.code == code
    assert call + ":" in str(ei.value)


@pytest.mark.parametrize("call", CALLS)
def test_null_struct_and_nothing_to_do(call):
    cls, fields = CALLS[call]
    f = getattr(capi.lib(), "b200rwkv_" + call)
    assert f(0, None, None) == INVALID
    none = {"tokens" if call == "op_linear_e4m3" else "rows": 0, **{n: None for n in ("x", "out", "logits") if n in fields}}
    assert f(0, None, C.byref(made(cls, fields, none))) == 0


def test_tensors_that_are_not_on_a_gpu():
    torch = pytest.importorskip("torch")
    from ai00_server_b200 import device_ops
    x = torch.zeros(4, 64)
    q = x.to(torch.float8_e4m3fn)
    for f in (lambda: device_ops.to_e4m3(x), lambda: device_ops.rms_norm(x), lambda: device_ops.linear_e4m3(q, x, q, x), lambda: device_ops.sample(x, torch.zeros(4)),
              lambda: device_ops.to_e4m3(x[0]), lambda: device_ops.rms_norm(x[0]), lambda: device_ops.sample(x[0], torch.zeros(4)), lambda: device_ops.linear_e4m3(q[0], x, q, x)):
        with pytest.raises(capi.B200Error):
            f()


def test_structs_match_the_header(tmp_path):
    """Sizes and offsets as a C compiler has them, and as device_ops packs them."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines, want = [], []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        lines += [f'printf("%zu ", offsetof({name}, {f[0]}));' for f in cls._fields_]
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "b200rwkv.h"\nint main(void) { ' + "\n".join(lines) + " return 0; }\n")
    exe = tmp_path / "s"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want
    assert f"#define B200RWKV_TYPE_E4M3 {capi.TYPE_E4M3}\n" in open(os.path.join(root, "include", "b200rwkv.h")).read()
    from ai00_server_b200 import device_ops as d
    for packed, cls in ((d._E4M3_ROWS, capi.E4m3), (d._NORM, capi.Norm), (d._LINEAR, capi.LinearE4m3), (d._SAMPLE, capi.Sample)):
        assert packed.size == C.sizeof(cls)
        # every field at its place: numbers that tell the fields apart
        kinds = [f[1] for f in cls._fields_]
        values = [float(i + 1) if k is C.c_float else i + 1 for i, k in enumerate(kinds)]
        q = cls.from_buffer_copy(packed.pack(*values))
        assert [getattr(q, f[0]) for f in cls._fields_] == values


def test_engine_call_refuses_null():
    q, d = capi.RowControls(struct_bytes=C.sizeof(capi.RowControls)), capi.Draw(struct_bytes=C.sizeof(capi.Draw))
    assert capi.lib().b200rwkv_sample_tokens(None, 1, C.byref(q), C.byref(d), None, None) == INVALID
