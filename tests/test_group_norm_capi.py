"""Host-only checks of the group norm C ABI (no GPU work): include/sdxl_hip/group_norm.h is exported whole, every
refusal comes before the first launch, empty problems are no-ops, workspaces have their sizes."""
import ctypes
import os
import re
import subprocess

import pytest

import sdxl_hip as sh

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sdxl_hip", "group_norm.h")
P = 4096  # a pointer that is never followed: aligned to everything
GIB = 1 << 30


def test_header_declarations_are_exported():
    names = set(re.findall(r"^(?:sdxl_status|size_t) (sdxl_\w+)\(", open(HEADER).read(), re.M))
    assert names == set(sh.GROUP_NORM_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", sh.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert names <= {line.split()[-1] for line in out.splitlines() if " T " in line}
    header = re.search(r"typedef struct sdxl_group_norm_desc \{(.*?)\} sdxl_group_norm_desc;", open(HEADER).read(), re.S).group(1)
    assert re.findall(r"(?:int(?:32|64)_t|float) (\w+);", header) == [f[0] for f in sh.GroupNormDesc._fields_]


def desc(batch=2, pixels=1 << 17, channels=64, groups=8, dtype=sh.F16, **kw):
    return sh.GroupNormDesc(batch=batch, pixels=pixels, channels=channels, groups=groups, dtype=dtype, **kw)


ARGS = {"forward": ("x", "gamma", "beta", "y", "stats", "ws"), "i8": ("x", "gamma", "beta", "q", "ld_q", "q_scale", "stats", "ws"),
        "backward": ("dy", "x", "gamma", "beta", "stats", "dx", "dgamma", "dbeta", "ws")}
NAMES = {"forward": "sdxl_group_norm", "i8": "sdxl_group_norm_i8", "backward": "sdxl_group_norm_backward"}


def call(kind, d, ws_bytes=GIB, **given):
    """Every pointer a GiB from the next, but for those given."""
    at = {name: GIB * (i + 1) for i, name in enumerate(ARGS[kind])} | {"ld_q": 0} | given
    ref = ctypes.byref(d) if d is not None else None
    args = [at[n] if n == "ld_q" else at[n] or None for n in ARGS[kind]]
    return getattr(sh.load(), NAMES[kind])(ref, *args, ws_bytes, None)


@pytest.mark.parametrize("kind", ARGS)
@pytest.mark.parametrize("bad,status", [
    (dict(reserved=1), sh.INVALID_ARGUMENT), (dict(dtype=sh.E4M3), sh.INVALID_SHAPE), (dict(dtype=9), sh.INVALID_SHAPE),
    (dict(activation=6), sh.INVALID_ARGUMENT), (dict(activation=-1), sh.INVALID_ARGUMENT),
    (dict(eps=-1e-5), sh.INVALID_ARGUMENT), (dict(eps=float("nan")), sh.INVALID_ARGUMENT),
    (dict(eps=float("inf")), sh.INVALID_ARGUMENT), (dict(batch=-1), sh.INVALID_SHAPE),
    (dict(pixels=1 << 31), sh.INVALID_SHAPE), (dict(channels=-64), sh.INVALID_SHAPE), (dict(groups=0), sh.INVALID_SHAPE),
    (dict(groups=-8), sh.INVALID_SHAPE), (dict(groups=7), sh.INVALID_SHAPE), (dict(x_row_stride=63), sh.INVALID_SHAPE),
    (dict(y_row_stride=-64), sh.INVALID_SHAPE), (dict(dy_row_stride=1 << 31), sh.INVALID_SHAPE),
    (dict(batch=(1 << 31) - 1, pixels=(1 << 31) - 1), sh.INVALID_SHAPE),
])
def test_refused_descriptors(kind, bad, status):
    assert call(kind, desc(**bad)) == status
    assert sh.load().sdxl_last_error()
    size = getattr(sh.load(), NAMES[kind] + "_workspace_bytes")
    assert size(ctypes.byref(desc(**bad))) == 0


@pytest.mark.parametrize("kind", ARGS)
def test_refused_pointers(kind):
    assert call(kind, None) == sh.INVALID_ARGUMENT
    for name in ("x", "gamma", "beta"):
        assert call(kind, desc(), **{name: 0}) == sh.INVALID_ARGUMENT, name
        assert call(kind, desc(), **{name: P + 1}) == sh.UNSUPPORTED, name
    assert call(kind, desc(), stats=P + 2) == sh.UNSUPPORTED
    for ws in (dict(ws=0), dict(ws=P + 128), dict(ws_bytes=8)):
        assert call(kind, desc(), **ws) == sh.INVALID_ARGUMENT
        assert "workspace" in sh.load().sdxl_last_error().decode()
    if kind != "i8":
        assert call(kind, desc(dtype=sh.F32), x=P + 2) == sh.UNSUPPORTED
    if kind == "backward":
        assert call(kind, desc(), stats=0) == call(kind, desc(), dy=0) == sh.INVALID_ARGUMENT
        assert call(kind, desc(), dx=P + 1) == call(kind, desc(), dgamma=P + 1) == sh.UNSUPPORTED
    elif kind == "forward":
        assert call(kind, desc(), y=0) == sh.INVALID_ARGUMENT and call(kind, desc(), y=P + 1) == sh.UNSUPPORTED
    else:
        assert call(kind, desc(), q=0) == call(kind, desc(), q_scale=0) == sh.INVALID_ARGUMENT
        assert call(kind, desc(), q_scale=P + 2) == sh.UNSUPPORTED
        assert call(kind, desc(dtype=sh.F32)) == call(kind, desc(), ld_q=63) == call(kind, desc(), ld_q=1 << 31) == sh.INVALID_SHAPE


@pytest.mark.parametrize("kind", ARGS)
def test_overlaps_are_refused(kind):
    at = {name: GIB * (i + 1) for i, name in enumerate(ARGS[kind])}
    outputs = {"forward": ("y", "stats", "ws"), "i8": ("q", "q_scale", "stats", "ws"),
               "backward": ("dx", "dgamma", "dbeta", "ws")}[kind]
    inputs = [n for n in ARGS[kind] if n not in outputs and n != "ld_q"]
    for out in outputs:
        for other in [n for n in inputs + list(outputs) if n != out]:
            if (kind, out, other) == ("forward", "y", "x"):
                continue  # in place
            assert call(kind, desc(), **{out: at[other]}) == sh.INVALID_ARGUMENT, (out, other)
            assert "overlap" in sh.load().sdxl_last_error().decode()
    if kind == "forward":  # not with another stride, and not shifted
        assert call(kind, desc(y_row_stride=128), y=at["x"]) == sh.INVALID_ARGUMENT
        assert call(kind, desc(), y=at["x"] + 64) == sh.INVALID_ARGUMENT


@pytest.mark.parametrize("kind", ARGS)
def test_empty_problems_launch_nothing(kind):
    nothing = {name: 0 for name in ARGS[kind]}
    for d in (desc(batch=0), desc(pixels=0), desc(channels=0)):
        assert call(kind, d, ws_bytes=0, **nothing) == sh.OK
    if kind == "backward":
        assert call(kind, desc(), dx=0, dgamma=0, dbeta=0) == sh.OK  # nothing is wanted


def test_workspaces():
    for dtype in (sh.F16, sh.F32):
        assert sh.group_norm_workspace_bytes(2, 16, 64, 8, dtype) == 0  # one launch
        small = sh.group_norm_workspace_bytes(2, 1 << 17, 64, 8, dtype)
        assert small % 256 == 0 and 0 < small <= 1 << 18
        assert sh.group_norm_workspace_bytes(2, 1 << 17, 64, 8, dtype, call="backward") > small
    assert sh.group_norm_workspace_bytes(2, 16, 64, 8, call="i8") > 0
    # parts of the sums, not of the tensor: [1, 2^20, 128] fp32 is 512 MiB
    assert sh.group_norm_workspace_bytes(1, 1 << 20, 128, 32, sh.F32, call="backward") < 8 << 20


def test_python_refusals():
    x, g = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.float16)
    stats = torch.zeros(2, 8, 2)
    with pytest.raises(sh.SdxlError, match="GPU"):
        sh.group_norm(x, g, g, 8)
    for bad in (lambda: sh.group_norm(x[0], g, g, 8), lambda: sh.group_norm(x, g[:32], g, 8), lambda: sh.group_norm(x, g, g.float(), 8),
                lambda: sh.group_norm(x, g, g, 7), lambda: sh.group_norm(x.double(), g, g, 8),
                lambda: sh.group_norm(x, g, g, 8, activation="tanh"), lambda: sh.group_norm(x.transpose(1, 2), g[:4], g[:4], 2),
                lambda: sh.group_norm(x[:, :1].expand(2, 4, 64), g, g, 8), lambda: sh.group_norm(x, g, g, 8, out=x[:, :2]),
                lambda: sh.group_norm(torch.zeros(2, 8, 64, dtype=torch.float16)[:, ::2][:, :3], g, g, 8),
                lambda: sh.group_norm_backward(x[:, :2], x, g, g, 8, stats), lambda: sh.group_norm_backward(x, x, g, g, 8, stats[:1]),
                lambda: sh.group_norm_backward(x, x, g, g, 8, stats.double()),
                lambda: sh.group_norm_i8(x.float(), g.float(), g.float(), 8)):
        with pytest.raises(sh.SdxlError):
            bad()


def test_python_gradients_without_statistics():
    x, g = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.float16)
    with pytest.raises(sh.SdxlError, match="stats"):
        sh.group_norm_backward(x, x, g, g, 8, None)


def test_no_workspace_for_codes_of_fp32():
    assert call("i8", desc(dtype=sh.F32)) == sh.INVALID_SHAPE
    assert sh.group_norm_workspace_bytes(2, 1 << 17, 64, 8, sh.F32, call="i8") == 0
