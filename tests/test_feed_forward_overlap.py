"""Host-only: calls of the feed-forward C ABI that would write what they read, or that fail in a later step, are
refused before the first launch (a launch fails here without a GPU, with another status)."""
import ctypes

import pytest

import sdxl_hip as sh

pytest.importorskip("torch")
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
