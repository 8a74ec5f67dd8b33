"""The feed-forward operators against plain 64-bit forms on the same inputs.

Tolerances are bounds, element by element, from 64-bit quantities: every output is rounded once (half a
step h of the type); sums of K fp32 products differ from exact ones by at most (K + 3) 2^-24 times the sum
of the products' magnitudes (and the bias); the activations are evaluated to 2e-5 of their value, slopes to
2e-5 (gelu's tail polynomial has a relative error of 1.1e-5, exp2 and the reciprocal one unit in the last
place each), their slopes are at most 1.13 and their second derivatives at most 1.2 (quick gelu's 2 * 1.702 / 4
at 0 is 0.851, silu's 0.5, gelu's 0.798); the backward's dz is rounded to the type before its products.
"""
import ctypes
import math
import os
import subprocess

import pytest

import sdxl_hip as sh

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -126}  # half a subnormal step (bf16: below fp32's smallest normal)
E32, ACT = 2.0 ** -24, 2e-5


def values(seed, *shape, std=1.0, dtype=F16):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)


def e4m3(seed, rows, cols):
    w = values(seed, rows, cols, std=max(cols, 1) ** -0.5, dtype=torch.float32)
    scale = (w.abs().amax(dim=-1).clamp_min(1e-12) / 448.0) if cols else torch.ones(rows, device=DEV)
    codes = (w / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), scale, codes.double() * scale.double()[:, None]


def act64(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z * (1.702 if name == "quick_gelu" else 1.0))


def slope64(name, z):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(act64(name, z).sum(), z)[0]


def within(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), (got.double() - want).abs()[bad].max().item(), bound[bad].min().item())


def projections(x, w64, bias):
    """z and the bound of its fp32 error."""
    z, mass = x.double() @ w64.t(), x.double().abs() @ w64.abs().t()
    if bias is not None:
        z, mass = z + bias.double(), mass + bias.double().abs()
    return z, (x.shape[1] + 3) * E32 * mass


def split(z, gate_first):
    a, b = z.chunk(2, dim=-1)
    return (b, a) if gate_first else (a, b)


def check_forward(x, w64, bias, activation, got, gated, gate_first=False, residual=None):
    z, ez = projections(x, w64, bias)
    if gated:
        (v, g), (ev, eg) = split(z, gate_first), split(ez, gate_first)
        a = act64(activation, g)
        want, err = v * a, ev * a.abs() + (v.abs() + ev) * (1.13 * eg + ACT * a.abs() + E32) + 2 * E32 * (v * a).abs()
    else:
        want = act64(activation, z)
        err = 1.13 * ez + ACT * want.abs()
        if residual is not None:
            want = want + residual.double()
            err = err + E32 * want.abs()
    within(got, want, err + HALF[x.dtype] * (want.abs() + err) + TINY[x.dtype], ("forward", activation, x.shape, w64.shape))


def dz_of(dout, x, w64, bias, activation, gated, gate_first=False):
    """dz and the bound of the error of the rounded one that the products take."""
    d = dout.double()
    h = HALF[x.dtype]
    if not gated and activation == "none":
        return d, torch.zeros_like(d)
    z, ez = projections(x, w64, bias)

    def slope_error(z, ez):  # second derivative, evaluation, and relu's step
        err = 1.2 * ez + ACT
        return err + (z.abs() <= ez).double() if activation == "relu" else err

    if gated:
        (v, g), (ev, eg) = split(z, gate_first), split(ez, gate_first)
        a, s = act64(activation, g), slope64(activation, g)
        dv, dg = d * a, d * v * s
        edv = d.abs() * (1.13 * eg + ACT * a.abs() + E32)
        edg = d.abs() * (ev * s.abs() + (v.abs() + ev) * slope_error(g, eg))
        dz, e = torch.cat((dg, dv) if gate_first else (dv, dg), -1), torch.cat((edg, edv) if gate_first else (edv, edg), -1)
    else:
        s = slope64(activation, z)
        dz, e = d * s, d.abs() * slope_error(z, ez)
    e = e + 3 * E32 * dz.abs()
    return dz, e + h * (dz.abs() + e) + TINY[x.dtype]


def check_backward(dout, x, w, bias, activation, grads, gated, gate_first=False):
    dx, dw, db = grads
    dz, edz = dz_of(dout, x, w.double(), bias, activation, gated, gate_first)
    h, tiny = HALF[x.dtype], TINY[x.dtype]
    x64, w64 = x.double(), w.double()
    for what, got, want, mass, err, terms in (  # (got None: not asked for)
        ("dx", dx, dz @ w64, dz.abs() @ w64.abs(), edz @ w64.abs(), w.shape[0]),
        ("dw", dw, dz.t() @ x64, dz.abs().t() @ x64.abs(), edz.t() @ x64.abs(), x.shape[0]),
        ("db", db, dz.sum(0), dz.abs().sum(0), edz.sum(0), x.shape[0]),
    ):
        if got is not None:
            err = err + (terms + 3) * E32 * (mass + err)
            within(got, want, err + h * (want.abs() + err) + tiny, (what, activation, x.shape, w.shape))


# one element; less than a tile; tile edges; more than a tile; widths that 16-byte rows divide and that they
# do not; a depth of several steps with a tail
SIZES = [(1, 1, 1), (1, 8, 16), (3, 5, 7), (2, 1280, 320), (17, 33, 40), (64, 64, 64), (65, 129, 72), (130, 96, 200),
         (257, 320, 128), (300, 331, 64), (96, 40, 1003)]
ACTS = ("none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu")


def dims(i, m, n, k):
    """(dtype, activation, bias, gate_first) so that a run over sizes meets every value"""
    return (F16, BF16)[i % 2], ACTS[(i + m) % 6], i % 3 != 0, i % 2 == 0


@pytest.mark.parametrize("case", range(2 * len(SIZES)))
def test_forward(case):
    m, n, k = SIZES[case % len(SIZES)]
    dtype, activation, has_bias, gate_first = dims(case // len(SIZES) + case, m, n, k)
    x, bias_g = values(case, m, k, dtype=dtype), values(case + 1, 2 * n, std=0.3, dtype=dtype) if has_bias else None
    w = values(case + 2, 2 * n, k, std=k ** -0.5, dtype=dtype)
    got = sh.gated_linear(x, w, bias=bias_g, activation=activation, gate_first=gate_first)
    check_forward(x, w.double(), bias_g, activation, got, True, gate_first)
    residual = values(case + 3, m, n, dtype=dtype) if gate_first else None
    bias = bias_g[:n].clone() if has_bias else None
    got = sh.linear_act(x, w[:n], bias=bias, residual=residual, activation=activation)
    check_forward(x, w[:n].double(), bias, activation, got, False, residual=residual)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_forward_every_activation(activation, dtype):
    x, w = values(1, 70, 96, std=2.0, dtype=dtype), values(2, 144, 96, std=0.3, dtype=dtype)
    check_forward(x, w.double(), None, activation, sh.gated_linear(x, w, activation=activation), True)
    check_forward(x, w.double(), None, activation, sh.linear_act(x, w, activation=activation), False)


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 320, 640), (5, 7, 9), (2, 66, 80), (70, 144, 96), (300, 328, 192), (33, 40, 77)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_forward_e4m3_weights(m, n, k, dtype):
    x = values(3, m, k, dtype=dtype)
    codes, scale, w64 = e4m3(4, 2 * n, k)
    bias = values(5, 2 * n, std=0.3, dtype=dtype)
    check_forward(x, w64, bias, "gelu", sh.gated_linear(x, codes, bias=bias, w_scale=scale), True)
    residual = values(6, m, 2 * n, dtype=dtype)
    got = sh.linear_act(x, codes, bias=bias, w_scale=scale, residual=residual, activation="silu")
    check_forward(x, w64, bias, "silu", got, False, residual=residual)


def test_scales_of_16_bit_weights():
    x, w = values(1, 40, 64), values(2, 48, 64, std=0.125)
    scale = values(3, 48, dtype=torch.float32).abs()
    got = sh.linear_act(x, w, w_scale=scale, activation="silu")
    check_forward(x, w.double() * scale.double()[:, None], None, "silu", got, False)


@pytest.mark.parametrize("case", range(2 * len(SIZES)))
def test_backward(case):
    m, n, k = SIZES[case % len(SIZES)]
    dtype, activation, has_bias, gate_first = dims(case // len(SIZES) + case, m, n, k)
    x, w = values(case, m, k, dtype=dtype), values(case + 1, 2 * n, k, std=k ** -0.5, dtype=dtype)
    bias = values(case + 2, 2 * n, std=0.3, dtype=dtype) if has_bias else None
    dout = values(case + 3, m, n, std=0.3, dtype=dtype)
    grads = sh.gated_linear_backward(dout, x, w, bias=bias, activation=activation, gate_first=gate_first)
    assert (grads[2] is None) == (bias is None)
    check_backward(dout, x, w, bias, activation, grads, True, gate_first)
    bias = bias[:n].clone() if has_bias else None
    grads = sh.linear_act_backward(dout, x, w[:n], bias=bias, activation=activation)
    check_backward(dout, x, w[:n], bias, activation, grads, False)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_backward_every_activation(activation, dtype):
    x, w = values(1, 70, 96, std=2.0, dtype=dtype), values(2, 144, 96, std=0.3, dtype=dtype)
    dout, bias = values(3, 70, 72, std=0.3, dtype=dtype), values(4, 144, dtype=dtype)
    check_backward(dout, x, w, bias, activation,
                   sh.gated_linear_backward(dout, x, w, bias=bias, activation=activation), True)
    dout = values(5, 70, 144, std=0.3, dtype=dtype)
    check_backward(dout, x, w, bias, activation, sh.linear_act_backward(dout, x, w, bias=bias, activation=activation),
                   False)


# few rows: one token to 16 rows (depths below a block, of one step and of several steps of 2048), then tens of
# rows with much depth, with at most one 32 x 32 tile of sums per CU and with more; ragged edges
FEW_ROWS = [(1, 1283, 2120), (2, 1280, 320), (16, 40, 4112), (5, 2056, 80), (9, 20, 16), (17, 72, 1304), (64, 643, 1296),
            (150, 650, 528), (33, 3001, 336), (63, 16, 9000), (460, 1283, 5120), (250, 1030, 8208)]


@pytest.mark.parametrize("m,n,k", FEW_ROWS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_few_rows(m, n, k, dtype):
    x, w = values(1, m, k, dtype=dtype), values(2, 2 * n, k, std=k ** -0.5, dtype=dtype)
    bias, residual = values(3, 2 * n, std=0.3, dtype=dtype), values(4, m, n, dtype=dtype)
    check_forward(x, w.double(), bias, "gelu", sh.gated_linear(x, w, bias=bias, gate_first=True), True, True)
    got = sh.linear_act(x, w[:n], bias=bias[:n].clone(), residual=residual, activation="silu")
    check_forward(x, w[:n].double(), bias[:n], "silu", got, False, residual=residual)
    dout = values(6, m, n, std=0.3, dtype=dtype)
    check_backward(dout, x, w, bias, "gelu", sh.gated_linear_backward(dout, x, w, bias=bias), True)
    codes, scale, w64 = e4m3(5, 2 * n, k)
    if k % 16 == 0:
        check_forward(x, w64, bias, "silu", sh.gated_linear(x, codes, bias=bias, w_scale=scale, activation="silu"), True)
        got = sh.linear_act(x, codes[:n], w_scale=scale[:n], residual=residual)
        check_forward(x, w64[:n], None, "none", got, False, residual=residual)


# rows and columns of sums that each tile of the tiled kernel takes at a depth of 328 (six stages, the last one
# ragged), largest tile last, every edge ragged
# (as measured costs choose, some of these meet on one tile and 64 x 64 has none: every tile, by name, is in
# test_feed_forward_kernels_gpu.py)
TILES = [(200, 4104), (4100, 520), (4100, 744), (4100, 1032), (4100, 1496), (4100, 2056), (4100, 4104)]


@pytest.mark.parametrize("rows,cols", TILES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_tile_forward(rows, cols, dtype):
    x, w = values(1, rows, 328, dtype=dtype), values(2, cols, 328, std=0.055, dtype=dtype)
    bias, residual = values(3, cols, std=0.3, dtype=dtype), values(4, rows, cols, dtype=dtype)
    check_forward(x, w.double(), bias, "gelu", sh.gated_linear(x, w, bias=bias), True)
    got = sh.linear_act(x, w, bias=bias, residual=residual, activation="silu")
    check_forward(x, w.double(), bias, "silu", got, False, residual=residual)


@pytest.mark.parametrize("rows,cols", TILES)
def test_every_tile_forward_e4m3(rows, cols):
    x = values(1, rows, 336)
    codes, scale, w64 = e4m3(2, cols, 336)
    check_forward(x, w64, None, "gelu", sh.gated_linear(x, codes, w_scale=scale), True)
    check_forward(x, w64, None, "none", sh.linear_act(x, codes, w_scale=scale), False)


@pytest.mark.parametrize("rows,cols", TILES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_tile_backward(rows, cols, dtype):
    """dz on the tile, then dx with few features, then dw with few rows"""
    x, w = values(1, rows, 328, dtype=dtype), values(2, cols, 328, std=0.055, dtype=dtype)
    bias = values(3, cols, std=0.3, dtype=dtype)
    dout = values(4, rows, cols // 2, std=0.3, dtype=dtype)
    check_backward(dout, x, w, bias, "gelu", sh.gated_linear_backward(dout, x, w, bias=bias), True)
    dout = values(5, rows, cols, std=0.3, dtype=dtype)
    grads = sh.linear_act_backward(dout, x, w, bias=bias, activation="silu")
    check_backward(dout, x, w, bias, "silu", grads, False)
    x, w, dout = values(6, rows, cols, dtype=dtype), values(7, 328, cols, std=0.05, dtype=dtype), values(8, rows, 328, dtype=dtype)
    check_backward(dout, x, w, None, "none", sh.linear_act_backward(dout, x, w, need_dw=False), False)
    x, w, dout = values(6, 328, cols, dtype=dtype), values(7, rows, cols, std=0.05, dtype=dtype), values(8, 328, rows, dtype=dtype)
    grads = sh.linear_act_backward(dout, x, w, need_dx=False, need_dbias=True)
    check_backward(dout, x, w, None, "none", grads, False)


# dw and dx in one launch, either one's tasks first, on every pair of their tiles that the sizes of a call lead to
# (rows, columns, features)
# (five of the nine pairs; all of them, by name, are in test_feed_forward_kernels_gpu.py)
@pytest.mark.parametrize("m,n,k", [(2056, 1283, 328), (328, 2056, 1288), (2400, 200, 1800), (200, 2400, 1800), (4100, 648, 2056),
                                   (648, 4100, 2056), (1111, 640, 640), (4104, 2056, 264), (70, 6001, 136)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_backward_in_one_launch(m, n, k, dtype):
    x, w = values(1, m, k, dtype=dtype), values(2, n, k, std=k ** -0.5, dtype=dtype)
    dout, bias = values(3, m, n, std=0.3, dtype=dtype), values(4, n, std=0.3, dtype=dtype)
    check_backward(dout, x, w, bias, "gelu", sh.linear_act_backward(dout, x, w, bias=bias, activation="gelu"), False)


# few tiles and a long sum: the depth of dx, of dw or of both in shares that do not come out even, joined afterwards
@pytest.mark.parametrize("m,n,k,gated,activation", [(300, 2571, 136, True, "gelu"), (4100, 72, 264, False, "none"),
                                                    (8192, 136, 128, True, "silu"), (2200, 1288, 648, False, "gelu"),
                                                    (90, 6000, 1000, False, "relu"), (1100, 1099, 72, False, "silu"),
                                                    (2, 2571, 141, True, "gelu"), (4100, 72, 261, False, "none"), (4101, 71, 72, False, "silu"),
                                                    (300, 4000, 137, True, "silu")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_backward_of_split_sums(m, n, k, gated, activation, dtype):
    features = 2 * n if gated else n
    x, w = values(1, m, k, dtype=dtype), values(2, features, k, std=k ** -0.5, dtype=dtype)
    dout, bias = values(3, m, n, std=0.3, dtype=dtype), values(4, features, std=0.3, dtype=dtype)
    fn = sh.gated_linear_backward if gated else sh.linear_act_backward
    grads = fn(dout, x, w, bias=bias, activation=activation)
    check_backward(dout, x, w, bias, activation, grads, gated)
    for a, b in zip(grads, fn(dout, x, w, bias=bias, activation=activation)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_backward_parts(gated, activation):
    """Each gradient alone (its product may run on another tile than in the whole call, so its sums' order may
    differ); a bias gradient without a bias; nothing asked."""
    x, w = values(1, 100, 64), values(2, 80, 64, std=0.125)
    dout = values(3, 100, 40 if gated else 80)
    fn = sh.gated_linear_backward if gated else sh.linear_act_backward
    whole = fn(dout, x, w, activation=activation, need_dbias=True)
    check_backward(dout, x, w, None, activation, whole, gated)
    for part in range(3):
        need = dict(zip(("need_dx", "need_dw", "need_dbias"), (part == 0, part == 1, part == 2)))
        alone = fn(dout, x, w, activation=activation, **need)
        assert [g is not None for g in alone] == [part == i for i in range(3)]
        check_backward(dout, x, w, None, activation, alone, gated)
    assert fn(dout, x, w, activation=activation, need_dx=False, need_dw=False, need_dbias=False) == (None, None, None)


@pytest.mark.parametrize("m,n,k", [(154, 5120, 1288), (8200, 200, 136), (300, 2571, 137), (2200, 2056, 648), (40, 16, 2056)])
def test_one_gradient_of_split_sums(m, n, k):
    x, w, dout = values(1, m, k), values(2, n, k, std=k ** -0.5), values(3, m, n, std=0.3)
    for activation in ("none", "gelu"):
        got = sh.linear_act_backward(dout, x, w, activation=activation, need_dw=False)
        check_backward(dout, x, w, None, activation, got, False)
        got = sh.linear_act_backward(dout, x, w, activation=activation, need_dx=False, need_dbias=True)
        check_backward(dout, x, w, None, activation, got, False)


# the bias gradient without the weights': one share of the rows and many, whole and ragged groups of 8 columns, odd strides
@pytest.mark.parametrize("m,n,pad", [(1, 3, 0), (127, 520, 0), (128, 512, 8), (5000, 1283, 0), (4097, 640, 3), (300, 10007, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_bias_gradient_alone(m, n, pad, dtype):
    x, w = values(1, m, 24, dtype=dtype), values(2, n, 24, std=0.2, dtype=dtype)
    dout = values(3, m, n + pad, dtype=dtype)[:, :n]
    for activation in ("none", "silu"):
        got = sh.linear_act_backward(dout, x, w, activation=activation, need_dx=False, need_dw=False, need_dbias=True)
        check_backward(dout, x, w, None, activation, got, False)


@pytest.mark.parametrize("gated", [False, True])
def test_empty_sums(gated):
    """No input features: the bias alone. No rows: gradients of zeros. No output features: dx of zeros."""
    bias = values(1, 12)
    w = values(2, 12, 0)
    x = values(3, 5, 0)
    fn = sh.gated_linear if gated else sh.linear_act
    check_forward(x, w.double(), bias, "gelu", fn(x, w, bias=bias, activation="gelu"), gated)
    back = sh.gated_linear_backward if gated else sh.linear_act_backward
    n = 6 if gated else 12
    dx, dw, db = back(values(4, 5, n), x, w, bias=bias, activation="gelu")
    assert dx.shape == (5, 0) and dw.shape == (12, 0)
    check_backward(values(4, 5, n), x, w, bias, "gelu", (dx, dw, db), gated)
    dx, dw, db = back(values(4, 0, n), values(5, 0, 8), values(6, 12, 8), bias=bias, activation="gelu")
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    dx, dw, db = back(values(4, 5, 0), values(5, 5, 8), values(6, 0, 8), activation="gelu")
    assert dx.shape == (5, 8) and not dx.any() and dw.shape == (0, 8)
    assert fn(values(5, 0, 8), values(6, 12, 8)).shape == (0, n)


@pytest.mark.parametrize("m,n,k,pad", [(37, 24, 40, 8), (37, 24, 40, 5), (140, 136, 72, 64), (9, 11, 13, 3)])
def test_row_strides(m, n, k, pad):
    """Column slices of wider tensors, and outputs that leave the rest of their rows as it was."""
    def wide(seed, rows, cols, std=1.0):
        t = values(seed, rows, cols + pad, std=std)
        return t, t[:, :cols]

    (_, x), (_, w), (_, res), (_, dout) = wide(1, m, k), wide(2, 2 * n, k, k ** -0.5), wide(3, m, 2 * n), wide(4, m, n)
    buf, out = wide(5, m + 2, n)
    before = buf.clone()
    sh.gated_linear(x, w, activation="silu", out=out[1:m + 1])
    check_forward(x, w.double(), None, "silu", out[1:m + 1], True)
    buf[1:m + 1, :n] = before[1:m + 1, :n]
    assert torch.equal(buf, before)
    check_forward(x, w.double(), None, "gelu", sh.linear_act(x, w, residual=res, activation="gelu"), False, residual=res)
    check_backward(dout, x, w, None, "gelu", sh.gated_linear_backward(dout, x, w), True)
    check_backward(dout, x, w[:n], None, "none", sh.linear_act_backward(dout, x, w[:n]), False)


# rows that no 16-byte access divides, on 64 x 64 and on 128 x 128 tiles: the last chunk of a row of 8 elements or more is
# its last 16 bytes; E4M3 rows of 16 codes or more
@pytest.mark.parametrize("m,n,k", [(1, 1283, 321), (16, 1291, 2123), (7, 37, 4109), (5, 2056, 81), (19, 72, 1303), (63, 643, 1297),
                                   (150, 651, 525), (33, 1501, 337), (40, 16, 9001), (620, 1283, 3411), (620, 641, 3411), (40, 9, 8), (77, 100, 9), (130, 331, 71), (301, 257, 645), (2200, 1091, 133),
                                   (4100, 1543, 68)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_odd_rows(m, n, k, dtype):
    x, w = values(1, m, k, dtype=dtype), values(2, 2 * n, k, std=k ** -0.5, dtype=dtype)
    bias, residual, dout = values(3, 2 * n, std=0.3, dtype=dtype), values(4, m, n, dtype=dtype), values(5, m, n, std=0.3, dtype=dtype)
    check_forward(x, w.double(), bias, "gelu", sh.gated_linear(x, w, bias=bias), True)
    got = sh.linear_act(x, w[:n], bias=bias[:n].clone(), residual=residual, activation="silu")
    check_forward(x, w[:n].double(), bias[:n], "silu", got, False, residual=residual)
    check_backward(dout, x, w, bias, "silu", sh.gated_linear_backward(dout, x, w, bias=bias, activation="silu"), True)
    check_backward(dout, x, w[:n], None, "none", sh.linear_act_backward(dout, x, w[:n]), False)
    if k >= 16:
        codes, scale, w64 = e4m3(6, 2 * n, k)
        check_forward(x, w64, bias, "gelu_tanh", sh.gated_linear(x, codes, bias=bias, w_scale=scale, activation="gelu_tanh"), True)
        check_forward(x, w64[:n], None, "relu", sh.linear_act(x, codes[:n], w_scale=scale[:n], activation="relu"), False)


@pytest.mark.parametrize("m,n,k,pad,shift", [(70, 136, 72, 8, 0), (70, 136, 72, 5, 0), (70, 136, 75, 8, 0), (70, 137, 72, 8, 1),
                                             (9, 72, 64, 8, 0), (2100, 1032, 88, 8, 0), (2100, 1033, 91, 3, 2), (80, 640, 648, 8, 0)])
def test_what_lies_beside_the_rows_is_not_read_into_them(m, n, k, pad, shift):
    """x, w, dout and the residual are column slices of tensors that are NaN everywhere else."""
    def slice_of(seed, rows, cols, std=1.0):
        t = torch.full((rows + 2, cols + pad + shift), float("nan"), dtype=F16, device=DEV)
        part = t[1:rows + 1, shift:cols + shift]
        part.copy_(values(seed, rows, cols, std=std))
        return part

    x, w, dout, residual = slice_of(1, m, k), slice_of(2, 2 * n, k, k ** -0.5), slice_of(3, m, n, 0.3), slice_of(4, m, n)
    check_forward(x, w.double(), None, "gelu", sh.gated_linear(x, w), True)
    got = sh.linear_act(x, w[:n], residual=residual, activation="silu")
    check_forward(x, w[:n].double(), None, "silu", got, False, residual=residual)
    check_backward(dout, x, w, None, "gelu", sh.gated_linear_backward(dout, x, w, need_dbias=True), True)
    check_backward(dout, x, w[:n], None, "none", sh.linear_act_backward(dout, x, w[:n], need_dbias=True), False)


# rows half a million elements apart (offsets past 32 bits at the last ones) and beyond the fast kernels' strides
@pytest.mark.parametrize("m,ld", [(4600, 1 << 19), (4600, (1 << 19) + 1), (40, (1 << 20) + 8)])
def test_rows_far_apart(m, ld):
    n, k = 72, 136
    wide = torch.empty(m, ld, dtype=F16, device=DEV)
    x, out, dout = wide[:, 8:8 + k], wide[:, 1024:1024 + n], wide[:, 2048:2048 + n]
    x.copy_(values(1, m, k))
    dout.copy_(values(2, m, n, std=0.3))
    w, bias = values(3, 2 * n, k, std=k ** -0.5), values(4, 2 * n, std=0.3)
    sh.gated_linear(x, w, bias=bias, out=out)
    check_forward(x, w.double(), bias, "gelu", out, True)
    check_backward(dout, x, w, bias, "gelu", sh.gated_linear_backward(dout, x, w, bias=bias), True)


def test_strided_gradients_through_the_c_abi():
    m, n, k = 40, 24, 72
    x, w, dout = values(1, m, k), values(2, n, k, std=0.12), values(3, m, n)
    dx, dw = values(4, m, k + 9), values(5, n, k + 16)
    dx0, dw0 = dx.clone(), dw.clone()
    d = sh.FfDesc(m=m, n=n, k=k, dx_row_stride=k + 9, dw_row_stride=k + 16, activation=5)
    lib = sh.load()
    ws = torch.empty(lib.sdxl_linear_act_backward_workspace_bytes(ctypes.byref(d)), dtype=torch.uint8, device=DEV)
    rc = lib.sdxl_linear_act_backward(ctypes.byref(d), dout.data_ptr(), x.data_ptr(), w.data_ptr(), None, dx.data_ptr(),
                                      dw.data_ptr(), None, ws.data_ptr(), ws.numel(), sh._stream(x))
    assert rc == sh.OK
    check_backward(dout, x, w, None, "silu", (dx[:, :k], dw[:, :k], None), False)
    assert torch.equal(dx[:, k:], dx0[:, k:]) and torch.equal(dw[:, k:], dw0[:, k:])


def test_residual_in_place():
    for m, n, k in ((300, 320, 64), (33, 31, 17), (1, 640, 2560)):
        x, w, hidden = values(1, m, k), values(2, n, k, std=k ** -0.5), values(3, m, n)
        want = sh.linear_act(x, w, residual=hidden)
        check_forward(x, w.double(), None, "none", want, False, residual=hidden)
        assert sh.linear_act(x, w, residual=hidden, out=hidden) is hidden
        assert torch.equal(hidden, want)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("m", [4, 200])
def test_large_and_non_finite_projections(activation, m):
    """bf16 projections of 1e30, of an infinity and of NaN: the activation's limit, slopes of 0 or 1, NaN kept;
    rows and columns beside them untouched."""
    k, n = 64, 80
    x, w = values(1, m, k, dtype=BF16), values(2, n, k, std=0.125, dtype=BF16)
    x[:, 0] = 0
    w[:, 0] = 0
    clean = sh.linear_act(x, w, activation=activation)
    w[:4, 0] = torch.tensor([1.0, -1.0, 1.0, 1.0], dtype=BF16)
    w[4:, 0] = 0.0
    big = x.clone()
    big[0, 0] = 1e30
    out = sh.linear_act(big, w, activation=activation)
    same = activation == "none"
    low = torch.tensor(-1e30 if same else 0.0, dtype=BF16)
    assert out[0, 0] == torch.tensor(1e30, dtype=BF16) and out[0, 1] == low.to(DEV)
    assert torch.equal(out[1:, 4:], clean[1:, 4:]) and torch.equal(out[0, 4:], clean[0, 4:])
    dout = torch.ones(m, n, dtype=BF16, device=DEV)
    db = sh.linear_act_backward(dout[:1], big[:1], w, activation=activation, need_dbias=True)[2]
    assert db[0] == 1.0 and db[1] == (1.0 if same else 0.0)
    for value in (math.inf, math.nan):
        bad = x[:, :1].clone(), w[:, :1].clone()
        bad[0][0, 0], bad[1][4:, 0] = value, 1.0
        out = sh.linear_act(bad[0], bad[1], activation=activation)
        if math.isnan(value):
            assert out[0].isnan().all()
        else:
            assert out[0, 0] == math.inf and out[0, 1] == (-math.inf if same else 0.0)
        assert not out[1:].isnan().any()


def test_repeated_calls_agree():
    x, w, dout = values(1, 500, 192), values(2, 400, 192, std=0.07), values(3, 500, 200)
    first = (sh.gated_linear(x, w), *sh.gated_linear_backward(dout, x, w, need_dbias=True))
    for _ in range(3):
        again = (sh.gated_linear(x, w), *sh.gated_linear_backward(dout, x, w, need_dbias=True))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_streams_at_once():
    cases = []
    for i in range(2):
        cases.append((values(i, 700, 320), values(i + 2, 1280, 320, std=0.05), values(i + 4, 700, 640)))
    want = [(sh.gated_linear(x, w), *sh.gated_linear_backward(d, x, w)[:2]) for x, w, d in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [None, None]
    for _ in range(3):
        for i, (x, w, d) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = (sh.gated_linear(x, w), *sh.gated_linear_backward(d, x, w)[:2])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def chain(x, w_in, b_in, w_out, b_out, hidden, dy):
    """A feed-forward block and its gradients, as a training step runs it."""
    h = sh.gated_linear(x, w_in, bias=b_in)
    y = sh.linear_act(h, w_out, bias=b_out, residual=hidden)
    dh, dw_out, db_out = sh.linear_act_backward(dy, h, w_out, bias=b_out)
    dx, dw_in, db_in = sh.gated_linear_backward(dh, x, w_in, bias=b_in)
    return h, y, dh, dw_out, db_out, dx, dw_in, db_in


def chain_inputs(m, width, inner, seed=0, dtype=F16):
    return (values(seed, m, width, dtype=dtype), values(seed + 1, 2 * inner, width, std=width ** -0.5, dtype=dtype),
            values(seed + 2, 2 * inner, std=0.2, dtype=dtype), values(seed + 3, width, inner, std=inner ** -0.5, dtype=dtype),
            values(seed + 4, width, std=0.2, dtype=dtype), values(seed + 5, m, width, dtype=dtype),
            values(seed + 6, m, width, std=0.5, dtype=dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_together(dtype):
    """Every step of the run within the bound of its own inputs; the whole against the gradients of the whole."""
    x, w_in, b_in, w_out, b_out, hidden, dy = args = chain_inputs(333, 128, 512, dtype=dtype)
    h, y, dh, dw_out, db_out, dx, dw_in, db_in = chain(*args)
    check_forward(x, w_in.double(), b_in, "gelu", h, True)
    check_forward(h, w_out.double(), b_out, "none", y, False, residual=hidden)
    check_backward(dy, h, w_out, b_out, "none", (dh, dw_out, db_out), False)
    check_backward(dh, x, w_in, b_in, "gelu", (dx, dw_in, db_in), True)


def test_gradients_against_differences():
    """Directional derivatives of sum(dout * out) in 64 bits, by central differences of the formula: the call's
    gradients along the direction differ by at most their own bound along it."""
    m, n, k, step = 45, 24, 40, 1e-4
    x, w, bias, dout = values(1, m, k), values(2, 2 * n, k, std=0.16), values(3, 2 * n, std=0.3), values(4, m, n)
    for activation in ("gelu", "gelu_tanh", "quick_gelu", "silu"):
        grads = sh.gated_linear_backward(dout, x, w, bias=bias, activation=activation)
        dz, edz = dz_of(dout, x, w.double(), bias, activation, True)

        def loss(x64, w64, b64):
            v, g = (x64 @ w64.t() + b64).chunk(2, dim=-1)
            return (dout.double() * v * act64(activation, g)).sum()

        leaves = [x.double(), w.double(), bias.double()]
        bounds = [edz @ w.double().abs(), edz.t() @ x.double().abs(), edz.sum(0)]
        for i, (grad, bound) in enumerate(zip(grads, bounds)):
            along = values(10 + i, *grad.shape, dtype=torch.float32).double()
            moved = [[l + s * step * along if j == i else l for j, l in enumerate(leaves)] for s in (1, -1)]
            slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
            slack = ((bound + HALF[F16] * grad.double().abs()) * along.abs()).sum()
            # the difference's own error, step^2 / 6 of the third derivative: z moves by up to some 10 step here
            scale = (grad.double().abs() * along.abs()).sum()
            assert abs(slope - (grad.double() * along).sum()) <= slack * 1.01 + 1e-6 * scale, (activation, i)


def test_captured_and_replayed():
    """The whole run in a graph, with eager work between the replays; two graphs over one workspace."""
    args = chain_inputs(200, 128, 320)
    want = chain(*args)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        chain(*args)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = chain(*args)
    for replay in range(4):
        for g in got:
            g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), replay
        args[0].copy_(values(50 + replay, *args[0].shape))
        want = chain(*args)
        torch.cuda.synchronize()


def test_two_graphs_share_a_workspace():
    x, w, dout = values(1, 150, 128), values(2, 256, 128, std=0.09), values(3, 150, 128)
    n = sh.ff_backward_workspace_bytes(150, 128, 128, True, "gelu")
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    want = [sh.gated_linear_backward(d, x, w, need_dbias=True) for d in (dout, -dout)]
    graphs, got = [], []
    for d in (dout, -dout):
        d = d.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(sh.gated_linear_backward(d, x, w, need_dbias=True, workspace=ws))
        graphs.append((graph, d))
    for _ in range(3):
        for i in (0, 1, 1, 0):
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want[i], got[i]))
        ws.fill_(255)


# joined shares of a sum, rows through registers, few rows, a bias gradient alone: one graph each, over one workspace that
# is overwritten between the replays, with another shape's eager call in between
@pytest.mark.parametrize("m,n,k,parts", [(1111, 640, 320, "xwb"), (300, 2571, 136, "xwb"), (70, 643, 331, "xwb"), (2, 643, 645, "xw"),
                                         (4100, 640, 72, "b")])
def test_captured_gradients_of_every_kind(m, n, k, parts):
    x, w, dout = values(1, m, k), values(2, 2 * n, k, std=k ** -0.5), values(3, m, n, std=0.3)
    need = dict(need_dx="x" in parts, need_dw="w" in parts, need_dbias="b" in parts)
    ws = torch.empty(sh.ff_backward_workspace_bytes(m, n, k, True, "gelu"), dtype=torch.uint8, device=DEV)
    want = sh.gated_linear_backward(dout, x, w, workspace=ws, **need)
    other = [values(4, 500, 72), values(5, 144, 72, std=0.1), values(6, 500, 144)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sh.gated_linear_backward(dout, x, w, workspace=ws, **need)
    for _ in range(4):
        for g in got:
            if g is not None:
                g.fill_(float("nan"))
        ws.fill_(255)
        sh.linear_act_backward(other[2], other[0], other[1], activation="gelu")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got) if a is not None)


@pytest.mark.parametrize("m,n,k", [(3, 72, 64), (70, 136, 72), (300, 331, 71), (2100, 1288, 136)])
def test_vectors_off_alignment(m, n, k):
    """bias and scales that begin anywhere: elements' alignment is all they need."""
    x, w = values(1, m, k), values(2, 2 * n, k, std=k ** -0.5)
    bias = values(3, 2 * n + 1, std=0.3)[1:]
    scale = values(4, 2 * n + 1, dtype=torch.float32).abs()[1:]
    w64 = w.double() * scale.double()[:, None]
    check_forward(x, w64, bias, "gelu", sh.gated_linear(x, w, bias=bias, w_scale=scale), True)
    check_forward(x, w64, bias, "silu", sh.linear_act(x, w, bias=bias, w_scale=scale, activation="silu"), False)
    dout = values(5, m, n, std=0.3)
    check_backward(dout, x, w, bias, "gelu", sh.gated_linear_backward(dout, x, w, bias=bias), True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("B,S,W", [(2, 50, 128), (1, 1, 640), (1, 77, 66)])
def test_sublayer_is_its_steps(B, S, W, fp8):
    inner = 4 * W
    x, gamma, beta = values(1, B, S, W), 1 + values(2, W, std=0.1), values(3, W, std=0.1)
    if fp8:
        (w_in, s_in, _), (w_out, s_out, _) = e4m3(4, 2 * inner, W), e4m3(5, W, inner)
    else:
        w_in, w_out, s_in, s_out = values(4, 2 * inner, W, std=W ** -0.5), values(5, W, inner, std=inner ** -0.5), None, None
    b_in, b_out = values(6, 2 * inner, std=0.2), values(7, W, std=0.2)
    got = sh.ff_sublayer(x, gamma, beta, w_in, s_in, b_in, w_out, s_out, b_out)
    normed = sh.layer_norm(x, gamma, beta).view(B * S, W)
    h = sh.gated_linear(normed, w_in, bias=b_in, w_scale=s_in)
    want = sh.linear_act(h, w_out, bias=b_out, w_scale=s_out, residual=x.view(B * S, W))
    assert torch.equal(got.view(B * S, W), want)
    in_place = x.clone()
    assert sh.ff_sublayer(in_place, gamma, beta, w_in, s_in, b_in, w_out, s_out, b_out, out=in_place) is in_place
    assert torch.equal(in_place, got)


def test_transformer_block_halves_in_a_row():
    """Self-attention, cross-attention and feed-forward halves of one block, as the UNet runs them, in place."""
    B, S, H = 2, 64, 2
    W = 64 * H
    x = values(1, B, S, W)
    norm = lambda i: (1 + values(i, W, std=0.1), values(i + 1, W, std=0.1))
    w = lambda i, r, c: values(i, r, c, std=c ** -0.5)
    kv = sh.project_context_kv(values(2, B, 77, 256), w(3, 2 * W, 256))
    a = sh.attn_sublayer(x, *norm(10), w(12, 3 * W, W), None, w(13, W, W), values(14, W), H)
    b = sh.cross_attn_sublayer(a, *norm(20), w(22, W, W), None, kv, w(23, W, W), values(24, W), H)
    ff = (*norm(30), w(32, 8 * W, W), None, values(33, 8 * W, std=0.2), w(34, W, 4 * W), None, values(35, W))
    c = sh.ff_sublayer(b, *ff)
    normed = sh.layer_norm(b, *ff[:2]).view(B * S, W)
    h = sh.gated_linear(normed, ff[2], bias=ff[4])
    check_forward(normed, ff[2].double(), ff[4], "gelu", h, True)
    check_forward(h, ff[5].double(), ff[7], "none", c.view(B * S, W), False, residual=b.view(B * S, W))


def test_cpp_host_api():
    """The C++ Ops on the same kernels, against 64 bits on the host."""
    exe = os.path.join(ROOT, "sdxl-end2end_amd", "bin", "sdxl_hip_ops_test")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "feed-forward cases passed" in r.stdout, r.stdout + r.stderr
