"""Host-only: which kernel the feed-forward operators run by size (sdxl_ff_kernels). The sizes that the GPU tests take
for each kernel and tile (feed_forward_sizes.py) do run on it, every kernel and tile has such a size, and every kernel
that a performance case runs on is among them."""
import ctypes
import re

import pytest

import feed_forward_sizes as sizes
import sdxl_hip as sh

pytest.importorskip("torch")
TILES = ("64x64", "64x128", "128x128", "128x192", "128x256", "256x256", "256x320")
PROJECTIONS = {"linear": sizes.LINEAR, "gated": sizes.GATED, "linear_e4m3": sizes.LINEAR_E4M3, "gated_e4m3": sizes.GATED_E4M3}
DZ = {"linear": sizes.LINEAR_DZ, "gated": sizes.GATED_DZ}


def kernels(m, n, k, gated=False, activation="gelu", w_dtype=sh.BF16, dtype=sh.BF16, gradients=(), **strides):
    return sh.ff_kernels(sh.FfDesc(m=m, n=n, k=k, dtype=dtype, w_dtype=w_dtype, activation=sh.ACTIVATIONS[activation], **strides),
                         gated, gradients)


def both_widths(m, n, k):
    """n and, for the tiles' 16-byte epilogues, the multiple of 8 below it"""
    return {(m, n, k), (m, max(n // 8 * 8, min(n, 8)), k)}


@pytest.mark.parametrize("form", PROJECTIONS)
def test_sizes_of_projections(form):
    for kernel, size in PROJECTIONS[form].items():
        for m, n, k in both_widths(*size):
            for activation in ("relu", "gelu"):
                got = kernels(m, n, k, "gated" in form, activation, sh.E4M3 if "e4m3" in form else sh.BF16)
                assert got == kernel, (m, n, k)


@pytest.mark.parametrize("form", DZ)
def test_sizes_of_dz(form):
    for kernel, size in DZ[form].items():
        for m, n, k in both_widths(*size):
            got = kernels(m, n, k, form == "gated", "relu", gradients=("dx", "dw", "dbias"))
            assert got.split("; ")[0] == "dz " + kernel, (m, n, k)


def test_sizes_of_gradients():
    for kernel, (wanted, (m, n, k)) in sizes.GRADIENTS.items():
        assert kernels(m, n, k, activation="none", gradients=wanted) == kernel, (m, n, k)
        if "dw" in wanted:
            assert kernels(m, n, k, activation="none", gradients=wanted + ("dbias",)) == kernel, (m, n, k)


def test_every_kernel_has_a_size():
    through = {f"{k}{s}" for k in ("deep 32x32/8", "deep 32x32/4", "deep 64x64/4") for s in ("", " staged")}
    through |= {"staged 64x64", "staged 128x128", "general"}
    rows = {f"rows/{w}{s}" for w in (4, 8, 16) for s in ("", " staged")}
    tiles = {"tile " + t for t in TILES}
    for form, table in PROJECTIONS.items():
        # (128 x 128 tiles share a stage's depth, which E4M3 codes do not allow)
        assert set(table) == through | rows | tiles - ({"tile 128x128"} if "e4m3" in form else set())
    for table in DZ.values():
        assert set(table) == through | tiles
    text = "; ".join(sizes.GRADIENTS)
    alone = {part for key in sizes.GRADIENTS for part in key.split("; ") if " + " not in part}
    pair = ("128x128", "128x256", "256x256")
    for g in ("dw", "dx"):
        assert {f"{g} tile {t}" for t in TILES} | {f"{g} staged 64x64", f"{g} staged 128x128", f"{g} general"} <= alone
        for a in pair:
            assert re.search(rf"{g} tile {a} in \d shares", text), (g, a)
            for b in pair:  # either one's tasks first
                assert any(re.fullmatch(rf"dw tile {a} \+ dx tile {b}|dx tile {b} \+ dw tile {a}", key) for key in sizes.GRADIENTS)
        assert re.search(rf"{g} staged 64x64 in \d shares", text)


def test_performance_cases_run_on_tested_kernels():
    from perf import operators
    plain = lambda text: re.sub(r" in \d shares", "", text)
    tested = {plain(key) for key in sizes.GRADIENTS}
    for case in operators.listed():
        gated, wanted = case["kind"] == "gated", ("dx", "dw") + (("dbias",) if case["bias"] else ())
        size = (case["rows"], case["inner"], case["width"])
        if not case["backward"]:
            form = case["kind"] + ("_e4m3" if case["weights"] == "e4m3" else "")
            assert kernels(*size, gated, case["activation"], sh.E4M3 if "e4m3" in form else sh.BF16) in PROJECTIONS[form]
            continue
        *dz, grads = kernels(*size, gated, case["activation"], gradients=wanted).split("; ")
        assert plain(grads) in tested, (case["name"], grads)
        for text in dz:
            assert text.removeprefix("dz ") in DZ[case["kind"]], case["name"]


def test_strides_and_alignment_decide():
    assert kernels(2048, 1280, 1280) == kernels(2048, 1280, 1280, x_row_stride=1288)
    assert "staged" in kernels(2048, 1280, 1280, x_row_stride=1281)
    assert kernels(2048, 1280, 1280, x_row_stride=(1 << 20) + 8) == "general"
    assert "staged" in kernels(2048, 1280, 1288, w_dtype=sh.E4M3)  # rows of codes in chunks of 16
    assert kernels(8192, 5120, 64, activation="none", gradients=("dbias",)) == "dbias in 32 shares"
    assert kernels(8, 512, 64, activation="none", gradients=("dbias",)) == "dbias"
    assert kernels(8, 512, 0, gradients=("dx", "dw")) == "" and kernels(0, 512, 64) == ""


def test_refused_queries():
    lib, d = sh.load(), sh.FfDesc(m=64, n=64, k=64, activation=2)
    text = ctypes.create_string_buffer(b"x" * 63, 64)
    for bad in (sh.FfDesc(m=-1, n=64, k=64), sh.FfDesc(m=64, n=64, k=64, activation=9), sh.FfDesc(m=64, n=64, k=64, reserved=1)):
        assert lib.sdxl_ff_kernels(ctypes.byref(bad), 0, 0, text, 64) == 0 and text.value == b""
    for gated, gradients in ((2, 0), (-1, 0), (0, 8), (0, -1)):
        assert lib.sdxl_ff_kernels(ctypes.byref(d), gated, gradients, text, 64) == 0 and lib.sdxl_last_error()
    assert lib.sdxl_ff_kernels(None, 0, 0, text, 64) == 0
    e4m3 = sh.FfDesc(m=64, n=64, k=64, w_dtype=sh.E4M3)
    assert lib.sdxl_ff_kernels(ctypes.byref(e4m3), 0, 1, text, 64) == 0  # no gradients through codes
    whole = sh.ff_kernels(d, True, ("dx", "dw", "dbias"))
    for size in (0, 1, 5, len(whole), len(whole) + 1):  # cut off, terminated
        text = ctypes.create_string_buffer(b"x" * 299, 300)
        assert lib.sdxl_ff_kernels(ctypes.byref(d), 1, 7, text, size) == len(whole)
        assert size == 0 or text.value.decode() == whole[:size - 1]
        assert text.raw[max(size, 0):299] == b"x" * (299 - size)
    assert lib.sdxl_ff_kernels(ctypes.byref(d), 1, 7, None, 0) == len(whole)
