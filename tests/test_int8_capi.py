"""Host-only checks of the 8-bit integer linears' C ABI (no GPU work): include/sdxl_hip/int8.h is exported whole, every
refusal comes before the first launch, empty problems are no-ops, workspaces have their sizes."""
import ctypes
import os
import re
import subprocess

import pytest

import sdxl_hip as sh

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sdxl_hip", "int8.h")
P = 4096  # a pointer that is never followed: aligned to everything
MIB = 1 << 20


def test_header_declarations_are_exported():
    names = set(re.findall(r"^(?:sdxl_status|size_t) (sdxl_\w+)\(", open(HEADER).read(), re.M))
    assert names == set(sh.INT8_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", sh.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert names <= {line.split()[-1] for line in out.splitlines() if " T " in line}
    header = re.search(r"typedef struct sdxl_i8_desc \{(.*?)\} sdxl_i8_desc;", open(HEADER).read(), re.S).group(1)
    assert re.findall(r"int(?:32|64)_t (\w+);", header) == [f[0] for f in sh.I8Desc._fields_]


def desc(m=8, n=8, k=64, dtype=sh.F16, x_dtype=sh.I8, **kw):
    return sh.I8Desc(m=m, n=n, k=k, dtype=dtype, x_dtype=x_dtype, **kw)


ARGS = ("x", "xs", "w", "ws", "bias", "res", "out", "work")


def call(gated, d, work_bytes=MIB, **given):
    """Every pointer a MiB from the next, but for those given."""
    at = {name: MIB * (i + 1) for i, name in enumerate(ARGS)} | given
    if d is not None and d.x_dtype != sh.I8 and "xs" not in given:
        at["xs"] = 0
    ref = ctypes.byref(d) if d is not None else None
    names = [n for n in ARGS if not (gated and n == "res")]
    fn = sh.load().sdxl_gated_linear_i8 if gated else sh.load().sdxl_linear_i8
    return fn(ref, *(at[n] or None for n in names), work_bytes, None)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bad,status", [
    (dict(reserved=1), sh.INVALID_ARGUMENT), (dict(dtype=sh.F32), sh.INVALID_SHAPE), (dict(dtype=sh.I8), sh.INVALID_SHAPE),
    (dict(x_dtype=sh.BF16), sh.INVALID_SHAPE), (dict(x_dtype=sh.E4M3), sh.INVALID_SHAPE), (dict(activation=6), sh.INVALID_ARGUMENT),
    (dict(activation=-1), sh.INVALID_ARGUMENT), (dict(gate_first=2), sh.INVALID_ARGUMENT), (dict(m=-1), sh.INVALID_SHAPE),
    (dict(n=1 << 31), sh.INVALID_SHAPE), (dict(k=1 << 31), sh.INVALID_SHAPE), (dict(k=131072), sh.UNSUPPORTED),
    (dict(x_row_stride=63), sh.INVALID_SHAPE), (dict(w_row_stride=-64), sh.INVALID_SHAPE), (dict(out_row_stride=7), sh.INVALID_SHAPE),
    (dict(residual_row_stride=1 << 31), sh.INVALID_SHAPE),
])
def test_refused_descriptors(gated, bad, status):
    assert call(gated, desc(**bad)) == status
    assert sh.load().sdxl_last_error()
    size = sh.load().sdxl_gated_linear_i8_workspace_bytes if gated else sh.load().sdxl_linear_i8_workspace_bytes
    assert size(ctypes.byref(desc(**bad))) == 0


@pytest.mark.parametrize("gated", [False, True])
def test_refused_pointers(gated):
    assert call(gated, None) == sh.INVALID_ARGUMENT
    for name in ("x", "xs", "w", "ws", "out"):
        assert call(gated, desc(), **{name: 0}) == sh.INVALID_ARGUMENT, name
    for name in ("xs", "ws", "bias", "out"):
        assert call(gated, desc(), **{name: P + 1}) == sh.UNSUPPORTED, name
    if not gated:
        assert call(gated, desc(gate_first=1)) == sh.INVALID_ARGUMENT
        assert call(gated, desc(), res=P + 1) == sh.UNSUPPORTED
    tokens = desc(x_dtype=sh.F16)
    assert call(gated, tokens, x=P + 1) == sh.UNSUPPORTED
    assert call(gated, tokens, xs=P) == sh.INVALID_ARGUMENT and "x_scale" in sh.load().sdxl_last_error().decode()
    for work in (dict(work=0), dict(work=P + 128), dict(work_bytes=8)):
        assert call(gated, tokens, **work) == sh.INVALID_ARGUMENT
        assert "workspace" in sh.load().sdxl_last_error().decode()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens", [False, True])
def test_overlaps_are_refused(gated, tokens):
    d = desc(x_dtype=sh.F16 if tokens else sh.I8)
    at = {name: MIB * (i + 1) for i, name in enumerate(ARGS)}
    inputs = ["x", "w", "ws", "bias"] + ([] if tokens else ["xs"])
    for out in ("out", "work") if tokens else ("out",):
        for other in inputs + (["work"] if tokens and out == "out" else []) + (["res"] if out == "work" and not gated else []):
            assert call(gated, d, **{out: at[other]}) == sh.INVALID_ARGUMENT, (out, other)
            assert "overlap" in sh.load().sdxl_last_error().decode()
    if not gated:  # in place: not shifted, not with another stride
        assert call(gated, d, out=at["res"] + 16) == sh.INVALID_ARGUMENT
        assert call(gated, desc(x_dtype=d.x_dtype, out_row_stride=16), out=at["res"]) == sh.INVALID_ARGUMENT


@pytest.mark.parametrize("gated", [False, True])
def test_empty_problems_launch_nothing(gated):
    nothing = {name: 0 for name in ARGS}
    for x_dtype in (sh.I8, sh.F16):
        for d in (desc(m=0, x_dtype=x_dtype), desc(n=0, x_dtype=x_dtype), desc(m=0, n=0, k=0, x_dtype=x_dtype)):
            assert call(gated, d, work_bytes=0, **nothing) == sh.OK


def test_workspaces():
    assert sh.linear_i8_workspace_bytes(10, 64, 100) == 1280 + 256  # codes in rows of 112 bytes, scales
    assert sh.linear_i8_workspace_bytes(10, 64, 100, gated=True, dtype=sh.BF16) == 1280 + 256
    assert sh.load().sdxl_linear_i8_workspace_bytes(ctypes.byref(desc())) == 0  # codes are there already
    assert sh.linear_i8_workspace_bytes(4, 64, 100) == 0  # quantised by the product
    assert sh.linear_i8_workspace_bytes(4, 64, 8) > 0 and sh.linear_i8_workspace_bytes(4, 64, 9000) > 0  # not by the general kernel, not so deep


def quantize(norm, rows=4, cols=64, dtype=sh.F16, ldx=0, ldq=0, eps=1e-5, **given):
    at = {name: MIB * (i + 1) for i, name in enumerate(("x", "gamma", "beta", "q", "scale"))} | given
    x, gamma, beta, q, scale = (at[n] or None for n in ("x", "gamma", "beta", "q", "scale"))
    lib = sh.load()
    if norm:
        return lib.sdxl_layer_norm_i8(rows, cols, dtype, x, ldx, gamma, beta, eps, q, ldq, scale, None)
    return lib.sdxl_quantize_i8_rows(rows, cols, dtype, x, ldx, q, ldq, scale, None)


@pytest.mark.parametrize("norm", [False, True])
def test_quantiser_refusals(norm):
    for bad in (dict(dtype=sh.F32), dict(dtype=sh.I8), dict(rows=-1), dict(cols=1 << 31), dict(ldx=63), dict(ldq=-1), dict(ldq=1 << 31)):
        assert quantize(norm, **bad) == sh.INVALID_SHAPE, bad
    for name in ("x", "q", "scale") + (("gamma", "beta") if norm else ()):
        assert quantize(norm, **{name: 0}) == sh.INVALID_ARGUMENT, name
        if name != "q":
            assert quantize(norm, **{name: P + 1}) == sh.UNSUPPORTED, name
    for bad in (dict(q=MIB), dict(scale=MIB), dict(q=5 * MIB)) + ((dict(q=2 * MIB), dict(scale=3 * MIB), dict(eps=-1.0), dict(eps=float("nan"))) if norm else ()):
        assert quantize(norm, **bad) == sh.INVALID_ARGUMENT, bad
    assert quantize(norm, rows=0, x=0, q=0, scale=0, gamma=0, beta=0) == sh.OK


def test_python_refusals():
    x, q, s = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    w, ws = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    with pytest.raises(sh.SdxlError, match="GPU"):
        sh.linear_i8(x, w, ws)
    b = torch.zeros(8, dtype=torch.bfloat16)
    for bad in (lambda: sh.linear_i8(q, w, ws, dtype=torch.float16), lambda: sh.linear_i8(q, w, ws, x_scale=s), lambda: sh.linear_i8(x, w, ws, x_scale=s),
                lambda: sh.linear_i8(x, w, ws, dtype=torch.bfloat16), lambda: sh.linear_i8(x, w, ws, bias=b),
                lambda: sh.linear_i8(q, w, ws, x_scale=s, bias=b, dtype=torch.float16), lambda: sh.linear_i8(x, x, ws),
                lambda: sh.linear_i8(x, w, ws[:4]), lambda: sh.linear_i8(x, w[:, :32], ws), lambda: sh.linear_i8(x, w, ws.double()),
                lambda: sh.linear_i8(q, w, ws, x_scale=s[:2], dtype=torch.float16), lambda: sh.gated_linear_i8(x, w[:7], ws[:7]),
                lambda: sh.linear_i8(x, w, ws, activation="tanh"), lambda: sh.quantize_i8_rows(x.float()),
                lambda: sh.layer_norm_i8(x, x[0, :32], x[0]), lambda: sh.quantize_i8_rows(x.t())):
        with pytest.raises(sh.SdxlError):
            bad()


# sizes (M, N, K) that reach each kernel, of the linear and of the gated form
KERNELS = {
    "rows/4": ((1, 9, 16), (2, 9, 48)), "rows/8": ((4, 9, 528), (3, 70, 832)), "rows/16": ((7, 8, 1136), (6, 8, 1072)),
    "rows/4 staged": ((3, 10, 19), (1, 8, 19)), "rows/8 staged": ((1, 11, 755), (2, 10, 515)), "rows/16 staged": ((6, 15, 1475), (3, 9, 1107)),
    "deep 32x32/8": ((19, 11, 288), (19, 9, 272)), "deep 32x32/8 staged": ((17, 9, 531), (19, 13, 387)),
    "deep 32x32/4": ((4604, 39, 656), (36, 2261, 544)), "deep 32x32/4 staged": ((523, 519, 275), (4141, 26, 275)),
    "deep 64x64/4": ((36, 10747, 4320), (36, 5158, 4192)), "deep 64x64/4 staged": ((392, 1589, 3907), (71, 3777, 2931)),
    "staged 64x64": ((20, 8, 19), (22, 12, 19)), "staged 128x128": ((1473, 2799, 19), (536, 3385, 19)),
    "tile 64x64": ((17, 8, 16), (18, 11, 16)), "tile 64x128": ((5538, 338, 16), (262, 3816, 16)),
    "tile 128x128": ((2589, 823, 2256), (414, 2358, 2096)), "tile 128x192": ((5630, 709, 16), (523, 3759, 16)),
    "tile 128x256": ((4379, 1353, 16), (1042, 2719, 16)), "tile 256x192": ((3334, 2446, 16), (4189, 995, 16)),
    "tile 256x256": ((5007, 2429, 16), (2094, 2881, 16)), "tile 256x320": ((4578, 3827, 16), (2105, 3881, 16)),
    "general": ((9, 33, 15), (70, 9, 7)),
}


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_sizes_of_kernels(kernel, gated):
    m, n, k = KERNELS[kernel][gated]
    for activation in sh.ACTIVATIONS.values():
        kw = dict(m=m, n=n, k=k, dtype=sh.BF16, activation=activation)
        assert sh.i8_kernels(desc(**kw), gated) == kernel
        own = m <= 4 and "rows" in kernel  # up to four tokens are quantised by the product's workgroups
        assert sh.i8_kernels(desc(**kw, x_dtype=sh.BF16), gated) == (kernel + " tokens" if own else "quantise; " + kernel)


def test_kernels_of_no_call():
    text, lib = ctypes.create_string_buffer(b"x" * 63, 64), sh.load()
    for d, gated in ((desc(m=0), 0), (desc(n=0), 1), (desc(reserved=1), 0), (desc(), 2)):
        assert lib.sdxl_i8_kernels(ctypes.byref(d), gated, text, 64) == 0 and text.value == b""
    assert lib.sdxl_i8_kernels(None, 0, text, 64) == 0
    whole = sh.i8_kernels(desc(m=40, x_dtype=sh.F16), True)
    for size in (1, 5, 64):
        assert lib.sdxl_i8_kernels(ctypes.byref(desc(m=40, x_dtype=sh.F16)), 1, text, size) == len(whole)
        assert text.value.decode() == whole[:size - 1]


# sizes that reach the kernels with stages of 128 bytes through more stages than their rings hold (at most four), the last one in part
DEEP_KERNELS = {
    "tile 64x64": ((5516, 67, 592), (33, 4162, 720)), "tile 64x128": ((6715, 265, 656), (133, 5494, 592)),
    "tile 128x128": ((2589, 823, 2256), (414, 2358, 2096)), "tile 128x192": ((6737, 523, 656), (6540, 265, 720)),
    "tile 128x256": ((6812, 769, 720), (522, 4953, 720)), "tile 256x192": ((5399, 1325, 688), (6543, 522, 720)),
    "tile 256x256": ((6520, 1745, 592), (1051, 4955, 656)), "tile 256x320": ((6620, 2308, 592), (1281, 5633, 624)),
    "staged 64x64": ((6412, 66, 715), (33, 4706, 587)), "staged 128x128": ((6551, 529, 651), (279, 5458, 715)),
}


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kernel", DEEP_KERNELS)
def test_sizes_of_kernels_in_depth(kernel, gated):
    m, n, k = DEEP_KERNELS[kernel][gated]
    assert k > 4 * 128 and k % 128 != 0 and m % 32 != 0
    assert sh.i8_kernels(desc(m=m, n=n, k=k), gated) == kernel and sh.i8_kernels(desc(m=m, n=n, k=k, dtype=sh.BF16), gated) == kernel


def test_every_tile_has_a_size_in_depth():
    assert set(DEEP_KERNELS) == {k for k in KERNELS if k.startswith(("tile", "staged"))}
