"""8-bit integer linears and the quantisers before them, against plain forms.

Codes and scales of given rows are equal to the definition's in IEEE fp32. Products: sums of codes are exact integers,
so that z = sum * x_scale * w_scale + bias is off by at most 4 u (|z - bias| + |bias|), u = 2^-24 (the integer's
conversion, two products, one addition); activations are evaluated to 2e-5 of their value, their slopes are at most
1.13, and the output is rounded once (in fp16 to infinity where its range ends). Norms before the codes: values are off as in the group norm's tests, a code by
half a step more.
"""
import pytest

import sdxl_hip as sh
from test_group_norm_gpu import BF16, DEV, F16, HALF, TINY, U, act64, check_forward, normal_form, values, within
from test_int8_capi import DEEP_KERNELS, KERNELS

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
ACT = 2e-5
HALVES = (F16, BF16)


def codes(seed, *shape, low=-127):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(low, 128, shape, generator=gen, dtype=torch.int32).to(torch.int8).to(DEV)


def scales(seed, n):
    gen = torch.Generator().manual_seed(seed)
    return ((torch.rand(n, generator=gen) + 0.5) * 0.01).to(DEV)


def quantized(x):
    """Codes and scales of rows by the definition, in IEEE fp32 on the host."""
    v = x.float().cpu()
    amax = torch.where(v.isfinite(), v.abs(), torch.zeros(())).amax(dim=-1) if v.shape[-1] else torch.zeros(v.shape[:-1])
    scale = torch.where(amax > 0, torch.clamp_min(amax / 127.0, 1e-12), torch.ones_like(amax))
    scale = torch.where(v.isnan().any(dim=-1), torch.full_like(scale, float("nan")), scale)
    return torch.round(v / scale[..., None]).clamp(-127, 127), scale.reshape(-1)


def product64(x, x_scale, w, w_scale, bias):
    z = (x.double() @ w.double().t()) * x_scale.double()[:, None] * w_scale.double()
    ez = 4 * U * z.abs()
    if bias is not None:
        z, ez = z + bias.double(), ez + 4 * U * bias.double().abs()
    return z, ez


def check(got, x, x_scale, w, w_scale, bias, activation, gated, gate_first=False, residual=None):
    z, ez = product64(x, x_scale, w, w_scale, bias)
    if gated:
        (a, b), (ea, eb) = z.chunk(2, dim=-1), ez.chunk(2, dim=-1)
        (v, ev), (g, eg) = ((b, eb), (a, ea)) if gate_first else ((a, ea), (b, eb))
        act = act64(activation, g)
        want = v * act
        err = ev * act.abs() + (v.abs() + ev) * (1.13 * eg + ACT * act.abs() + U) + 2 * U * want.abs()
    else:
        want = act64(activation, z)
        err = 1.13 * ez + ACT * want.abs()
        if residual is not None:
            want = want + residual.double()
            err = err + U * want.abs()
    h, tiny = HALF[got.dtype], TINY[got.dtype]
    if got.dtype == F16:  # from 65520 on, half a step past the largest value, the rounding gives infinity
        far = (want.abs() + err >= 65520.0) & got.isinf() & (got.sign() == want.sign())
        assert (got.isinf() <= far).all()
        got, want = torch.where(far, 0.0, got.double()).to(got.dtype), torch.where(far, 0.0, want)
    within(got, want, err + h * (want.abs() + err) + tiny, (tuple(x.shape), tuple(w.shape), activation, gated, got.dtype))


# (M, N, K): one element; rows shorter than 16 bytes; tile and stage edges; few rows of several depths (whole blocks,
# ragged ones, more than are in flight at once); depths that 16-byte accesses divide and that they do not; one tile and many
SIZES = [(1, 1, 1), (1, 8, 15), (3, 5, 7), (2, 7, 16), (1, 640, 320), (4, 33, 1280), (16, 48, 2048), (7, 100, 4112), (16, 40, 9000),
         (1, 129, 5120), (5, 64, 1003), (17, 33, 48), (32, 64, 128), (64, 64, 64), (65, 129, 144), (130, 96, 400), (257, 320, 128),
         (300, 331, 64), (96, 40, 1003), (154, 1280, 640), (128, 256, 256), (250, 1281, 336), (512, 512, 1280), (40, 1280, 5120),
         (1000, 640, 645), (2048, 2560, 320), (600, 640, 640)]
ACTS = ("none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_products(i, gated):
    M, N, K = SIZES[i]
    for turn in range(2):
        dtype, activation, gate_first = HALVES[(i + turn) % 2], ACTS[(i + 3 * turn + gated) % 6], gated and (i + turn) % 3 == 0
        features = 2 * N if gated else N
        x, w = codes(i, M, K, low=-128), codes(i + 40, features, K)
        xs, ws = scales(i, M), scales(i + 1, features)
        bias = values(i + 2, features, dtype=dtype) if turn == 0 else None
        if gated:
            got = sh.gated_linear_i8(x, w, ws, x_scale=xs, bias=bias, activation=activation, gate_first=gate_first, dtype=dtype)
            check(got, x, xs, w, ws, bias, activation, True, gate_first)
        else:
            residual = values(i + 3, M, N, dtype=dtype) if (i + turn) % 2 else None
            got = sh.linear_i8(x, w, ws, x_scale=xs, bias=bias, residual=residual, activation=activation, dtype=dtype)
            check(got, x, xs, w, ws, bias, activation, False, residual=residual)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_tokens_are_quantised_as_by_the_quantiser(i, gated):
    M, N, K = SIZES[i]
    dtype = HALVES[i % 2]
    x, w, ws = values(i, M, K, std=2.0, dtype=dtype), codes(i + 40, 2 * N if gated else N, K), scales(i, 2 * N if gated else N)
    q, xs = sh.quantize_i8_rows(x)
    fn = sh.gated_linear_i8 if gated else sh.linear_i8
    got = fn(x, w, ws, activation="silu")
    check(got, q, xs, w, ws, None, "silu", gated)
    assert torch.equal(got, fn(q, w, ws, x_scale=xs, activation="silu", dtype=dtype))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_each_kernel(kernel, gated):
    M, N, K = KERNELS[kernel][gated]
    dtype, features = HALVES[len(kernel) % 2], 2 * N if gated else N
    tokens, w, ws, bias = values(1, M, K, std=2.0, dtype=dtype), codes(2, features, K), scales(3, features), values(4, features, dtype=dtype)
    q, xs = sh.quantize_i8_rows(tokens)
    fn = sh.gated_linear_i8 if gated else sh.linear_i8
    given = dict(bias=bias, activation="gelu") | ({} if gated else dict(residual=values(5, M, N, dtype=dtype)))
    got = fn(q, w, ws, x_scale=xs, dtype=dtype, **given)
    check(got, q, xs, w, ws, bias, "gelu", gated, residual=given.get("residual"))
    assert torch.equal(got, fn(tokens, w, ws, **given))


# widths: one; shorter than a vector; ends inside one; a wave's, several waves', more than registers hold
WIDTHS = (1, 7, 8, 9, 77, 320, 512, 640, 1003, 1280, 2048, 2560, 2563, 5120, 10240, 11000, 40961, 70000)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("K", WIDTHS)
def test_quantiser(K, dtype):
    rows = 37 if K < 10000 else 3
    x = values(K, rows, K, std=3.0, dtype=dtype)
    x[0] = 0.0
    x[1] *= 1e-7 if dtype == F16 else 1e-14  # (bf16: below the smallest scale)
    if rows > 4 and K > 2:
        x[2, K // 2] = float("inf")
        x[3, K - 1] = float("-inf")
        x[4, 0] = float("nan")
        x[5] = float("inf")
    q, s = sh.quantize_i8_rows(x)
    want_q, want_s = quantized(x)
    assert torch.equal(s.cpu().nan_to_num(-1.0), want_s.nan_to_num(-1.0))
    fine = ~want_s.isnan()
    assert torch.equal(q.cpu()[fine].float(), want_q[fine])


def test_quantiser_ties_and_strides():
    """Exact halves go to even; rows apart and off alignment, and what lies between them."""
    wide = torch.zeros(9, 101, dtype=F16, device=DEV)
    x = wide[:, 3:98]
    x[:] = (torch.arange(95, device=DEV) - 47.0) + 0.5  # amax 47.5
    x[:, 0] = 127.0
    q, s = sh.quantize_i8_rows(x)
    assert (s == 1.0).all()
    want = torch.round(x.float())
    want[:, 0] = 127
    assert torch.equal(q.float(), want)
    lib, out = sh.load(), torch.full((9, 120), 55, dtype=torch.int8, device=DEV)
    scale = torch.empty(9, device=DEV)
    assert lib.sdxl_quantize_i8_rows(9, 95, sh.F16, x.data_ptr(), 101, out.data_ptr() + 5, 120, scale.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream) == sh.OK
    assert torch.equal(out[:, 5:100], q) and (out[:, :5] == 55).all() and (out[:, 100:] == 55).all()
    assert sh.quantize_i8_rows(torch.empty(4, 0, dtype=F16, device=DEV))[1].tolist() == [1.0] * 4


def check_norm_codes(q, s, z, ez):
    """Codes of values z that are off by at most ez: half a step, and the scale's own error."""
    rows = z.reshape(q.shape[0] * (q.shape[1] if q.dim() == 3 else 1), -1)
    e = ez.reshape(rows.shape)
    amax, top = rows.abs().amax(dim=1), e.amax(dim=1)
    step = amax / 127
    within(s, step, top / 127 + 4 * U * step + 1e-12, "scale")
    got = q.reshape(rows.shape).double() * s.double()[:, None]
    # (the largest codes: a value may pass 127 steps by the errors)
    within(got, rows, e + 0.5 * s.double()[:, None] * (1 + 4 * U) + 260 * U * s.double()[:, None] + top[:, None], "codes")
    assert (q.reshape(rows.shape).abs().amax(dim=1) == 127).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("K", WIDTHS[2:])
def test_layer_norm_codes(K, dtype):
    rows = 29 if K < 10000 else 3
    x = values(K, rows, K, std=2.0, mean=0.5, dtype=dtype)
    gamma, beta = values(1, K, std=0.2, mean=1.0, dtype=dtype), values(2, K, std=0.2, dtype=dtype)
    q, s = sh.layer_norm_i8(x, gamma, beta, eps=1e-5)
    # a LayerNorm is a group norm of one group over one pixel; sums of a row are made in fewer than 1024 steps a thread
    _, _, z, ez, _, _ = normal_form(x[:, None], gamma, beta, 1, 1e-5)
    check_norm_codes(q, s, z, ez * (1 + K / 64))
    if K <= 2048 and K % 2 == 0 and dtype == F16:  # beside the framework's LayerNorm: half a step of fp16 apart
        y = sh.layer_norm(x, gamma, beta).double()
        within(q.double() * s.double()[:, None], y, 0.51 * s.double()[:, None] + 1.01 * HALF[F16] * y.abs() + 1e-4, "layer_norm")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("B,P,C,G", [(1, 3, 7, 7), (2, 33, 64, 8), (2, 50, 320, 32), (1, 300, 640, 32), (2, 1024, 1280, 32), (1, 77, 2560, 32),
                                     (3, 41, 1003, 17), (1, 20, 10240, 32), (1, 5, 20000, 4), (2, 2500, 128, 32)])
def test_group_norm_codes(B, P, C, G, dtype):
    x = values(C, B, P, C, std=2.0, mean=0.5, dtype=dtype)
    gamma, beta = values(1, C, std=0.2, mean=1.0, dtype=dtype), values(2, C, std=0.2, dtype=dtype)
    q, s, stats = sh.group_norm_i8(x, gamma, beta, G, eps=1e-6, with_stats=True)
    assert q.shape == x.shape and s.shape == (B * P,)
    _, _, z, ez, _, _ = normal_form(x, gamma, beta, G, 1e-6)
    check_norm_codes(q, s, z, ez)
    y, y_stats = sh.group_norm(x, gamma, beta, G, eps=1e-6, with_stats=True)
    check_forward(x, gamma, beta, G, "none", 1e-6, y, stats)
    check_forward(x, gamma, beta, G, "none", 1e-6, y, y_stats)
    q, s = sh.group_norm_i8(x, gamma, beta, G, activation="silu", eps=1e-6)
    a = act64("silu", z)
    check_norm_codes(q, s, a, 1.13 * ez + ACT * a.abs())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(3, 40, 320), (70, 100, 640), (300, 260, 1280)])
def test_strided_rows_and_any_alignment(M, N, K, gated):
    """Slices of wider tensors, from elements that 16 bytes do not divide; what lies beside out stays."""
    features = 2 * N if gated else N
    for pad, first in ((16, 16), (5, 3), (24, 8)):
        x, w = codes(1, M, K + pad + first)[:, first:first + K], codes(2, features, K + pad + first)[:, first:first + K]
        tokens = values(3, M, K + pad + first)[:, first:first + K]
        xs, ws, bias = scales(1, M + 1)[1:], scales(2, features + 1)[1:], values(4, features + 1)[1:]
        wide = torch.full((M, N + pad + first), 7.0, dtype=F16, device=DEV)
        out = wide[:, first:first + N]
        fn = sh.gated_linear_i8 if gated else sh.linear_i8
        got = fn(x, w, ws, x_scale=xs, bias=bias, activation="gelu", out=out)
        check(got, x, xs, w, ws, bias, "gelu", gated)
        keep = torch.ones(N + pad + first, dtype=torch.bool, device=DEV)
        keep[first:first + N] = False
        assert (wide[:, keep] == 7.0).all()
        q, qs = sh.quantize_i8_rows(tokens)
        check(fn(tokens, w, ws, bias=bias, activation="gelu"), q, qs, w, ws, bias, "gelu", gated)
    if not gated:  # the residual in place
        residual = values(5, M, N + 8)[:, :N]
        before = residual.clone()
        got = sh.linear_i8(x, w, ws, x_scale=xs, residual=residual, out=residual)
        check(got, x, xs, w, ws, None, "none", False, residual=before)


def test_huge_strides_take_the_general_kernel():
    M, N, K = 2, 24, 64
    x = torch.empty(M, (1 << 20) + 16, dtype=torch.int8, device=DEV)[:, :K]
    x.copy_(codes(1, M, K))
    w, xs, ws = codes(2, N, K), scales(1, M), scales(2, N)
    check(sh.linear_i8(x, w, ws, x_scale=xs, dtype=F16), x, xs, w, ws, None, "none", False)


@pytest.mark.parametrize("M,N", [(1, 24), (40, 24), (300, 70)])
@pytest.mark.parametrize("K", [131071, 131056])
def test_largest_sums(M, N, K):
    """128 * 128 * k at its largest: the sums are integers up to 2^31."""
    x, w = torch.full((M, K), -128, dtype=torch.int8, device=DEV), torch.full((N, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    one = torch.ones(max(M, N), device=DEV)
    xs, ws = one[:M] * 2.0 ** -16, one[:N]
    check(sh.linear_i8(x, w, ws, x_scale=xs, dtype=BF16), x, xs, w, ws, None, "none", False)


def test_what_is_not_finite():
    """A token with a NaN: its row of the output, and no other; an infinite one stands for 127 steps."""
    for M, N, K in ((4, 40, 320), (200, 300, 640)):
        x, w, ws = values(1, M, K), codes(2, N, K), scales(2, N)
        clean = sh.linear_i8(x, w, ws)
        x[2, 5] = float("nan")
        got = sh.linear_i8(x, w, ws)
        assert got[2].isnan().all() and torch.equal(got[:2], clean[:2]) and torch.equal(got[3:], clean[3:])
        x[2, 5] = float("inf")
        got = sh.linear_i8(x, w, ws)
        assert got.isfinite().all() and torch.equal(got[3:], clean[3:])


def test_empty():
    w, ws = codes(1, 8, 64), scales(1, 8)
    assert sh.linear_i8(torch.empty(0, 64, dtype=F16, device=DEV), w, ws).shape == (0, 8)
    assert sh.linear_i8(torch.empty(4, 64, dtype=F16, device=DEV), w[:0], ws[:0]).shape == (4, 0)
    bias = values(1, 8)
    for x, xs in ((torch.empty(4, 0, dtype=F16, device=DEV), None), (torch.empty(4, 0, dtype=torch.int8, device=DEV), scales(2, 4))):
        assert torch.equal(sh.linear_i8(x, w[:, :0], ws, x_scale=xs, bias=bias), bias.expand(4, 8))
        got = sh.gated_linear_i8(x, w[:, :0], ws, x_scale=xs, bias=bias, activation="none")
        assert torch.equal(got, (bias[:4] * bias[4:]).expand(4, 4))


@pytest.mark.parametrize("B,P", [(1, 9), (2, 700)])
def test_transformer_entry_captured(B, P):
    """Group norm, proj_in, LayerNorm, gated projection and output projection with the residual as one graph on a side
    stream, replayed with eager calls between, against the same calls one by one."""
    C, inner = 320, 640
    x = values(1, B, P, C, std=2.0)
    g1, b1, g2, b2 = values(2, C, mean=1.0), values(3, C), values(4, C, mean=1.0), values(5, C)
    weights = [sh.quantize_i8_rows(values(6 + i, *s, std=s[1] ** -0.5)) for i, s in enumerate(((C, C), (2 * inner, C), (C, inner)))]
    bias = [values(10 + i, n) for i, n in enumerate((C, 2 * inner, C))]

    def run():
        q, s = sh.group_norm_i8(x, g1, b1, 32, eps=1e-6)
        h = sh.linear_i8(q.view(B * P, C), *weights[0], x_scale=s, bias=bias[0])
        q, s = sh.layer_norm_i8(h, g2, b2)
        inner_h = sh.gated_linear_i8(q, *weights[1], x_scale=s, bias=bias[1])
        return h, inner_h, sh.linear_i8(inner_h, *weights[2], bias=bias[2], residual=h)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = run()
    for turn in range(4):
        x.copy_(values(20 + turn, B, P, C, std=2.0))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for got, expected in zip(outs, want):
            assert torch.equal(got, expected), turn
    # against 64 bits: the steps' errors add up, a code's half step (1/254 of its row's largest value) above all
    q, s = sh.layer_norm_i8(outs[0], g2, b2)
    check(outs[1], q.view(B * P, C), s, *weights[1], bias[1], "gelu", True)
    q, s = sh.quantize_i8_rows(outs[1])
    check(outs[2], q, s, *weights[2], bias[2], "none", False, residual=outs[0])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("P,C,G", [(1, 64, 8), (300, 64, 8), (50, 1280, 32), (20, 3200, 4), (9, 6, 3)])
def test_group_norm_codes_of_constant_groups(P, C, G, dtype):
    """x - mean is 0, so that z is beta itself, whatever the mean and rstd = 1 / sqrt(eps): codes and scales are beta's."""
    gamma, beta = values(2, C, mean=1.0, dtype=dtype), values(3, C, dtype=dtype)
    want_q, want_s = quantized(beta.expand(2, P, C))
    for value in (3.0, 1000.0, -60000.0 if dtype == F16 else -2.0 ** 26):
        x = torch.full((2, P, C), value, dtype=dtype, device=DEV)
        q, s = sh.group_norm_i8(x, gamma, beta, G, eps=1e-6)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().float(), want_q), value


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("K", [8, 77, 1280, 2563, 8200, 10239, 10240, 11001])
def test_layer_norm_codes_of_constant_rows(K, dtype):
    """x - mean is 0, so that the codes and scales are beta's."""
    gamma, beta = values(2, K, mean=1.0, dtype=dtype), values(3, K, dtype=dtype)
    want_q, want_s = quantized(beta.expand(5, K))
    for value in (3.0, 2047.0, -2047.0 * 32, 0.1):
        q, s = sh.layer_norm_i8(torch.full((5, K), value, dtype=dtype, device=DEV), gamma, beta)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().float(), want_q), value


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kernel", DEEP_KERNELS)
def test_each_tile_in_depth(kernel, gated):
    """More stages than the ring holds, the last one in part; distinct codes, scales and biases in every place."""
    M, N, K = DEEP_KERNELS[kernel][gated]
    for dtype in HALVES:
        features = 2 * N if gated else N
        x, xs, w, ws = codes(1, M, K, low=-128), scales(1, M), codes(2, features, K), scales(3, features)
        bias = values(4, features, dtype=dtype)
        fn = sh.gated_linear_i8 if gated else sh.linear_i8
        given = dict(bias=bias, activation="none") | ({} if gated else dict(residual=values(5, M, N, dtype=dtype)))
        check(fn(x, w, ws, x_scale=xs, dtype=dtype, **given), x, xs, w, ws, bias, "none", gated, residual=given.get("residual"))
