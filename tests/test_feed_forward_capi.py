"""Host-only checks of the feed-forward C ABI (no GPU work): include/sdxl_hip/feed_forward.h is exported
whole, every refusal comes before the first device call, empty problems are no-ops."""
import ctypes
import os
import re
import subprocess

import pytest

import sdxl_hip as sh

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sdxl_hip", "feed_forward.h")
P = 4096  # a pointer that is never followed: aligned to everything


def test_header_declarations_are_exported():
    names = set(re.findall(r"^(?:sdxl_status|size_t) (sdxl_\w+)\(", open(HEADER).read(), re.M))
    assert names == set(sh.FEED_FORWARD_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", sh.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert names <= exported
    header = re.search(r"typedef struct sdxl_ff_desc \{(.*?)\} sdxl_ff_desc;", open(HEADER).read(), re.S).group(1)
    fields = re.findall(r"int(?:32|64)_t (\w+);", header)
    assert fields == [f[0] for f in sh.FfDesc._fields_]


def desc(m=8, n=8, k=64, dtype=sh.F16, w_dtype=None, activation=2, **kw):
    return sh.FfDesc(m=m, n=n, k=k, dtype=dtype, w_dtype=dtype if w_dtype is None else w_dtype, activation=activation,
                     **kw)


def call(kind, d, x=P, w=P, scale=0, bias=0, res=0, out=P, dout=P, dx=P, dw=P, db=P, ws=P, ws_bytes=1 << 40):
    lib, ref = sh.load(), ctypes.byref(d) if d is not None else None
    if kind == "linear":
        return lib.sdxl_linear_act(ref, x, w, scale or None, bias or None, res or None, out, None)
    if kind == "gated":
        return lib.sdxl_gated_linear(ref, x, w, scale or None, bias or None, out, None)
    fn = lib.sdxl_gated_linear_backward if kind == "gated_backward" else lib.sdxl_linear_act_backward
    return fn(ref, dout, x, w, bias or None, dx, dw, db, ws, ws_bytes, None)


KINDS = ("linear", "gated", "linear_backward", "gated_backward")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad,status", [
    (dict(reserved=1), sh.INVALID_ARGUMENT),
    (dict(dtype=sh.F32), sh.INVALID_SHAPE),
    (dict(dtype=sh.E4M3), sh.INVALID_SHAPE),
    (dict(w_dtype=sh.BF16), sh.INVALID_SHAPE),
    (dict(activation=6), sh.INVALID_ARGUMENT),
    (dict(activation=-1), sh.INVALID_ARGUMENT),
    (dict(gate_first=2), sh.INVALID_ARGUMENT),
    (dict(m=-1), sh.INVALID_SHAPE),
    (dict(n=1 << 31), sh.INVALID_SHAPE),
    (dict(k=1 << 31), sh.INVALID_SHAPE),
    (dict(x_row_stride=63), sh.INVALID_SHAPE),
    (dict(w_row_stride=-64), sh.INVALID_SHAPE),
    (dict(out_row_stride=7), sh.INVALID_SHAPE),
    (dict(dw_row_stride=1 << 31), sh.INVALID_SHAPE),
])
def test_refused_descriptors(kind, bad, status):
    assert call(kind, desc(**bad)) == status
    assert sh.load().sdxl_last_error()


@pytest.mark.parametrize("kind", KINDS)
def test_refused_pointers(kind):
    assert call(kind, None) == sh.INVALID_ARGUMENT
    assert call(kind, desc(), x=0) == sh.INVALID_ARGUMENT
    assert call(kind, desc(), w=0) == sh.INVALID_ARGUMENT
    assert call(kind, desc(), x=P + 1) == sh.UNSUPPORTED
    assert call(kind, desc(), bias=P + 1) == sh.UNSUPPORTED
    if kind.endswith("backward"):
        assert call(kind, desc(), dout=0) == sh.INVALID_ARGUMENT
        assert call(kind, desc(), dw=P + 1) == sh.UNSUPPORTED
        assert call(kind, desc(w_dtype=sh.E4M3)) == sh.UNSUPPORTED
        for ws in (dict(ws=0), dict(ws=P + 128), dict(ws_bytes=8)):
            assert call(kind, desc(), **ws) == sh.INVALID_ARGUMENT
            assert "workspace" in sh.load().sdxl_last_error().decode()
    else:
        assert call(kind, desc(), out=0) == sh.INVALID_ARGUMENT
        assert call(kind, desc(), out=P + 1) == sh.UNSUPPORTED
        assert call(kind, desc(w_dtype=sh.E4M3)) == sh.INVALID_ARGUMENT  # no scales
        assert "scaling metadata" in sh.load().sdxl_last_error().decode()
        assert call(kind, desc(), scale=P + 2) == sh.UNSUPPORTED


def test_gate_first_is_for_gated_calls():
    assert call("linear", desc(gate_first=1)) == sh.INVALID_ARGUMENT
    assert call("linear_backward", desc(gate_first=1)) == sh.INVALID_ARGUMENT


@pytest.mark.parametrize("kind", KINDS)
def test_empty_problems_launch_nothing(kind):
    empty = dict(x=0, w=0, out=0, dout=0, dx=0, dw=0, db=0, ws=0, ws_bytes=0)
    for d in (desc(m=0), desc(n=0), desc(m=0, n=0, k=0)):
        assert call(kind, d, **empty) == sh.OK


def test_workspace_bytes():
    ws = sh.ff_backward_workspace_bytes
    assert ws(8, 8, 64, True, "gelu") >= 8 * 16 * 2
    assert ws(8, 5, 64, True, "gelu") >= 8 * 16 * 2  # rows padded to 16 bytes
    assert ws(8, 8, 64, False, "silu") >= 8 * 8 * 2
    assert ws(8, 8, 64, True, "gelu", sh.F32) == 0  # refused
    lib = sh.load()
    assert lib.sdxl_gated_linear_backward_workspace_bytes(None) == 0


def test_sublayer_refusals():
    def status(d, x=P, gamma=P, w_in=P, s_in=0, w_out=P, s_out=0, y=P, ws=P, ws_bytes=1 << 40):
        return sh.load().sdxl_ff_sublayer(ctypes.byref(d), x, gamma, P, w_in, s_in or None, None, w_out, s_out or None,
                                          None, y, ws, ws_bytes, None)

    def d(rows=4, width=64, inner=256, w_in_dtype=sh.F16, w_out_dtype=sh.F16, activation=2, **kw):
        return sh.FfSublayerDesc(rows=rows, width=width, inner=inner, w_in_dtype=w_in_dtype, w_out_dtype=w_out_dtype,
                                 activation=activation, **kw)

    assert status(d(rows=0), x=0, ws=0) == sh.OK
    assert status(d(reserved=1)) == sh.INVALID_ARGUMENT
    assert status(d(rows=-1)) == sh.INVALID_SHAPE
    assert status(d(width=0)) == sh.INVALID_SHAPE
    assert status(d(width=63)) == sh.UNSUPPORTED
    assert status(d(width=2050)) == sh.UNSUPPORTED
    assert status(d(inner=-1)) == sh.INVALID_SHAPE
    assert status(d(w_in_dtype=sh.BF16)) == sh.INVALID_SHAPE
    assert status(d(activation=9)) == sh.INVALID_ARGUMENT
    assert status(d(gate_first=3)) == sh.INVALID_ARGUMENT
    assert status(d(), x=0) == sh.INVALID_ARGUMENT
    assert status(d(), w_out=0) == sh.INVALID_ARGUMENT
    assert status(d(), x=P + 2) == sh.UNSUPPORTED
    assert status(d(), w_in=P + 1) == sh.UNSUPPORTED
    assert status(d(w_in_dtype=sh.E4M3)) == sh.INVALID_ARGUMENT
    assert status(d(w_out_dtype=sh.E4M3)) == sh.INVALID_ARGUMENT
    assert status(d(), ws=0) == sh.INVALID_ARGUMENT
    assert status(d(), ws_bytes=4 * (64 + 256) * 2 - 1) == sh.INVALID_ARGUMENT
    assert sh.load().sdxl_ff_sublayer_workspace_bytes(ctypes.byref(d())) >= 4 * (64 + 256) * 2
    assert sh.load().sdxl_ff_sublayer_workspace_bytes(ctypes.byref(d(width=63))) == 0


def test_torch_wrapper_refusals():
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)
    x, w = z(4, 16), z(8, 16)
    for refused in (
        lambda: sh.gated_linear(x.float(), w.float()),
        lambda: sh.gated_linear(x, w.bfloat16()),
        lambda: sh.gated_linear(x, z(7, 16)),                                   # odd number of rows
        lambda: sh.gated_linear(x, z(8, 15)),
        lambda: sh.gated_linear(x, w, bias=z(4)),
        lambda: sh.gated_linear(x, w, bias=z(8, dtype=torch.float32)),
        lambda: sh.gated_linear(x, w, activation="elu"),
        lambda: sh.gated_linear(x, w, out=z(4, 8)),
        lambda: sh.gated_linear(x, w, out=z(4, 4, dtype=torch.bfloat16)),
        lambda: sh.gated_linear(x, w.byte()),                                   # E4M3 without scales
        lambda: sh.gated_linear(x, w.byte(), w_scale=z(8)),
        lambda: sh.gated_linear(x[:1].expand(4, 16), w),                        # broadcast rows
        lambda: sh.gated_linear(z(16, 4).t(), w),                               # transposed
        lambda: sh.gated_linear(z(2, 2, 16), w),
        lambda: sh.linear_act(x, w, residual=z(4, 4)),
        lambda: sh.linear_act(x, w, residual=z(4, 8, dtype=torch.bfloat16)),
        lambda: sh.linear_act_backward(z(4, 4), x, w),
        lambda: sh.linear_act_backward(z(4, 8, dtype=torch.bfloat16), x, w),
        lambda: sh.gated_linear_backward(z(4, 4), x, w.byte()),
        lambda: sh.ff_sublayer(z(4, 16), z(16), z(16), z(32, 16), None, None, z(16, 16), None, None),
        lambda: sh.ff_sublayer(z(1, 4, 16), z(16), z(16), z(32, 16), None, None, z(16, 8), None, None),
        lambda: sh.ff_sublayer(z(1, 4, 16), z(16), z(16), z(32, 16), None, z(16), z(16, 16), None, None),
    ):
        with pytest.raises(sh.SdxlError):
            refused()


@pytest.mark.parametrize("kind", KINDS)
def test_outputs_in_place_of_inputs_are_refused(kind):
    X, W, B, R, OUT = (P * i for i in range(1, 6))
    if kind.endswith("backward"):
        D, DX, DW, DB, WS = (P * i for i in range(6, 11))
        given = dict(x=X, w=W, bias=B, dout=D, dx=DX, dw=DW, db=DB, ws=WS)
        cases = [dict(given, **{out: given[i]}) for out in ("dx", "dw", "db") for i in ("x", "w", "dout", "bias")]
    else:
        given = dict(x=X, w=W, bias=B, out=OUT)
        cases = [dict(given, out=given[i]) for i in ("x", "w", "bias")]
    for case in cases:
        assert call(kind, desc(), **case) == sh.INVALID_ARGUMENT
        assert "overlaps" in sh.load().sdxl_last_error().decode()
    if kind == "linear":  # the residual in place only row for row
        d = desc(out_row_stride=16, residual_row_stride=24)
        assert call(kind, d, x=X, w=W, res=R, out=R) == sh.INVALID_ARGUMENT


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(6, 8, dtype=torch.float16)
    for fn in (sh.linear_act, sh.gated_linear):
        with pytest.raises(sh.SdxlError, match="on a GPU"):
            fn(x, w)
    with pytest.raises(sh.SdxlError, match="on a GPU"):
        sh.linear_act_backward(torch.zeros(4, 6, dtype=torch.float16), x, w)
