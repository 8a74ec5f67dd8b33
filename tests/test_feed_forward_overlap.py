"""Host-only: calls of the feed-forward C ABI that would write what they read, or that fail in a later step, are
refused before the first launch. Pointers are made up: a call that is not refused fails to launch without a GPU, and must
not be made with one."""
import ctypes

import pytest

import sdxl_hip as sh

torch = pytest.importorskip("torch")
if torch.cuda.is_available():
    pytest.skip("made-up pointers", allow_module_level=True)
MIB = 1 << 20  # pointers a MiB apart, never followed
SUBLAYER = ("x", "gamma", "beta", "w_in", "s_in", "b_in", "w_out", "s_out", "b_out", "y", "ws")


def sublayer(rows=4, width=64, inner=256, w_in_dtype=sh.F16, w_out_dtype=sh.F16, **given):
    d = sh.FfSublayerDesc(rows=rows, width=width, inner=inner, w_in_dtype=w_in_dtype, w_out_dtype=w_out_dtype, activation=2)
    at = {name: MIB * (i + 1) for i, name in enumerate(SUBLAYER)} | given
    size = sh.load().sdxl_ff_sublayer_workspace_bytes(ctypes.byref(d))
    status = sh.load().sdxl_ff_sublayer(ctypes.byref(d), *(at[n] or None for n in SUBLAYER), size, None)
    return status, sh.load().sdxl_last_error().decode()


@pytest.mark.parametrize("inner", [0, 256])
def test_sublayer_scales_are_checked_first(inner):
    """sdxl_linear_act needs the scales of E4M3 weights without columns too: not after the LayerNorm is launched."""
    status, error = sublayer(inner=inner, w_out_dtype=sh.E4M3, s_out=0)
    assert status == sh.INVALID_ARGUMENT and "scaling metadata" in error


@pytest.mark.parametrize("fp8", [False, True])
def test_sublayer_output_in_place_of_a_parameter_is_refused(fp8):
    dtype = sh.E4M3 if fp8 else sh.F16
    for name in ("gamma", "beta", "w_in", "b_in", "w_out", "b_out", "ws") + (("s_in", "s_out") if fp8 else ()):
        at = MIB * (SUBLAYER.index(name) + 1)
        status, error = sublayer(w_in_dtype=dtype, w_out_dtype=dtype, y=at)
        assert status == sh.INVALID_ARGUMENT and "overlaps" in error, name


BACKWARD = ("dout", "x", "w", "bias", "dx", "dw", "db", "ws")


def backward(gated, m=8, n=8, k=64, **given):
    d = sh.FfDesc(m=m, n=n, k=k, activation=2)
    at = {name: MIB * (i + 1) for i, name in enumerate(BACKWARD)} | given
    name = "sdxl_gated_linear_backward" if gated else "sdxl_linear_act_backward"
    size = getattr(sh.load(), name + "_workspace_bytes")(ctypes.byref(d))
    status = getattr(sh.load(), name)(ctypes.byref(d), *(at[n] or None for n in BACKWARD), size, None)
    return status, sh.load().sdxl_last_error().decode()


@pytest.mark.parametrize("gated", [False, True])
def test_gradients_in_one_place_are_refused(gated):
    dx, dw, db, ws = (MIB * (BACKWARD.index(name) + 1) for name in ("dx", "dw", "db", "ws"))
    for given in (dict(dw=dx), dict(db=dx), dict(db=dw), dict(dx=ws), dict(dw=ws), dict(db=ws)):
        status, error = backward(gated, **given)
        assert status == sh.INVALID_ARGUMENT and "overlaps" in error, given
    status, error = backward(gated, m=0, dw=db, x=0, dout=0)  # zeros are written too
    assert status == sh.INVALID_ARGUMENT and "overlaps" in error


def forward(gated, m=8, n=24, k=64, strides=(0, 0, 0, 0), **given):
    """strides: of x, w, out, residual"""
    names = ("x", "w", "scale", "bias") + (() if gated else ("residual",)) + ("out",)
    d = sh.FfDesc(m=m, n=n, k=k, activation=2, x_row_stride=strides[0], w_row_stride=strides[1], out_row_stride=strides[2],
                  residual_row_stride=strides[3])
    at = {name: MIB * (i + 1) for i, name in enumerate(names)} | given
    fn = sh.load().sdxl_gated_linear if gated else sh.load().sdxl_linear_act
    status = fn(ctypes.byref(d), *(at[n] or None for n in names), None)
    return status, sh.load().sdxl_last_error().decode()


def refused(result):
    return result[0] == sh.INVALID_ARGUMENT and "overlap" in result[1]


@pytest.mark.parametrize("gated", [False, True])
def test_partial_overlap_is_refused(gated):
    n, rows = 24, 48 if gated else 24
    sizes = dict(x=8 * 64 * 2, w=rows * 64 * 2, scale=rows * 4, bias=rows * 2)
    if not gated:
        sizes["residual"] = 8 * n * 2
    out_bytes = 8 * n * 2
    for i, (name, size) in enumerate(sizes.items()):
        at = MIB * (i + 1)
        for out in (at + size - 2, at - out_bytes + 2) + (() if name == "residual" else (at,)):
            assert refused(forward(gated, out=out)), (name, out)
        for out in (at + size, at - out_bytes):
            assert not refused(forward(gated, out=out)), (name, out)


def test_rows_between_rows():
    """Column slices of one tensor, whose rows lie between each other's, do not overlap."""
    ld = 200
    at = lambda column: MIB + 2 * column
    for x, out, bad in ((0, 64, False), (0, 63, True), (24, 0, False), (23, 0, True), (0, ld - 24, False), (0, ld - 23, True),
                        (30, ld + 30 - 24, False), (30, ld + 30 - 23, True), (0, 64 + 7 * ld, False), (0, 63 + 7 * ld, True),
                        (0, 63 + 8 * ld, False), (70, 7 * ld, False), (64 + 8 * ld, ld, False), (0, 8 * ld, False)):
        assert refused(forward(False, strides=(ld, 0, ld, 0), x=at(x), out=at(out))) == bad, (x, out)
    # one dense, or a single row
    for x, out, bad in ((0, 0, True), (0, 7 * ld + 63, True), (0, 7 * ld + 64, False), (8 * 24, 0, False), (8 * 24 - 1, 0, True),
                        (100, 100 - 8 * 24, False)):
        assert refused(forward(False, strides=(ld, 0, 0, 0), x=at(x), out=at(out))) == bad, (x, out)
    assert not refused(forward(False, m=1, n=136, strides=(ld, 0, 0, 0), x=at(0), out=at(64)))
    wide = (1 << 31) - 1  # extents past 63 bits of bytes
    assert refused(forward(False, m=wide, strides=(wide, 0, wide, 0), x=at(0), out=at(0)))
    assert not refused(forward(False, m=1, strides=(wide, 0, wide, 0), x=at(0), out=at(64)))


def test_residual_in_place_only_row_for_row():
    R = MIB * 5
    assert not refused(forward(False, residual=R, out=R))
    assert not refused(forward(False, strides=(0, 0, 40, 40), residual=R, out=R))
    assert refused(forward(False, strides=(0, 0, 40, 24), residual=R, out=R))
    assert refused(forward(False, strides=(0, 0, 40, 32), residual=R, out=R))
    assert refused(forward(False, strides=(0, 0, 40, 32), residual=R, out=R + 2 * (7 * 32 - 7 * 40)))  # the last rows
    assert refused(forward(False, residual=R, out=R + 2)) and refused(forward(False, residual=R, out=R - 48))


@pytest.mark.parametrize("gated", [False, True])
def test_backward_partial_overlap_is_refused(gated):
    at = {name: MIB * (i + 1) for i, name in enumerate(BACKWARD)}
    for out in ("dx", "dw", "db"):
        for other in ("dout", "x", "w", "bias", "ws") + tuple(g for g in ("dx", "dw", "db") if g != out):
            assert refused(backward(gated, **{out: at[other] + 2})), (out, other)
    for name in ("dout", "x", "w", "bias"):
        assert refused(backward(gated, **{name: at["ws"] + 16})), name
    assert not refused(backward(gated))


def test_sublayer_partial_overlap_is_refused():
    at = {name: MIB * (i + 1) for i, name in enumerate(SUBLAYER)}
    for name in ("x", "gamma", "beta", "w_in", "b_in", "w_out", "b_out"):
        assert refused(sublayer(y=at[name] + 4)), name
        assert refused(sublayer(**{name: at["ws"] + 4})), name
    assert refused(sublayer(y=at["ws"] + 4))
    assert not refused(sublayer()) and not refused(sublayer(y=at["x"]))
