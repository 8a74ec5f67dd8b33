"""Every kernel and tile of the feed-forward operators (feed_forward_sizes.py; test_feed_forward_dispatch.py holds the
sizes to their kernels), in two ways.

Small integers: with x, w and dout of -1, 0 and 1 and relu or no activation, every product, sum, slope and dz is a whole
number (or a multiple of a half, with E4M3 scales of powers of two) below 2^24, and dz at most 256, exact in both types.
Any order of summation gives the exact result, whose one rounding is the output: compared for equality, so that no row,
column or share can be missing or count twice. (A z has K terms of -1, 0 and 1, of which 4/9 are not 0: a deviation of
sqrt(4 K / 9) <= 32 and with 10^7 values at most about 6 of them, 190; bias at most 3.)

Normal values with gelu: within the bounds of test_feed_forward_gpu.py."""
import pytest

import feed_forward_sizes as sizes
import sdxl_hip as sh

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from test_feed_forward_gpu import DEV, F16, BF16, check_backward, check_forward  # noqa: E402


def generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def integers(seed, *shape, limit=1, dtype=F16):
    return torch.randint(-limit, limit + 1, shape, generator=generator(seed), device=DEV).to(dtype)


def normal(seed, *shape, std=1.0, dtype=F16):
    return (torch.randn(*shape, generator=generator(seed), device=DEV) * std).to(dtype)


def codes_of(w):
    return w.to(torch.float8_e4m3fn).view(torch.uint8)


def widths(m, n, k):
    return sorted({n, n // 8 * 8 if n >= 8 else n})


def exact(got, want, what):
    want = want.to(got.dtype)
    bad = got != want
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())


def split(z, gate_first):
    a, b = z.chunk(2, dim=-1)
    return (b, a) if gate_first else (a, b)


def cases(**tables):
    return [pytest.param(form, kernel, size, id=f"{form}-{kernel.replace(' ', '-')}")
            for form, table in tables.items() for kernel, size in table.items()]


PROJECTIONS = cases(linear=sizes.LINEAR, gated=sizes.GATED, linear_e4m3=sizes.LINEAR_E4M3, gated_e4m3=sizes.GATED_E4M3)
DZ = cases(linear=sizes.LINEAR_DZ, gated=sizes.GATED_DZ)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form,kernel,size", PROJECTIONS)
def test_projections_of_integers(form, kernel, size, dtype):
    m, _, k = size
    gated, fp8 = "gated" in form, "e4m3" in form
    for n in widths(*size):
        features = 2 * n if gated else n
        x, w = integers(1, m, k, dtype=dtype), integers(2, features, k, dtype=dtype)
        bias, residual = integers(3, features, limit=3, dtype=dtype), integers(4, m, n, limit=3, dtype=dtype)
        w64, scale, given = w.double(), None, w
        if fp8:
            scale = 2.0 ** integers(5, features, dtype=torch.float32)
            given, w64 = codes_of(w), w64 * scale.double()[:, None]
        z = x.double() @ w64.t() + bias.double()
        if gated:
            for gate_first in (False, True):
                v, g = split(z, gate_first)
                got = sh.gated_linear(x, given, bias=bias, w_scale=scale, activation="relu", gate_first=gate_first)
                exact(got, v * g.clamp_min(0), ("relu", n, gate_first))
            got = sh.gated_linear(x, given, bias=bias, w_scale=scale, activation="none")
            exact(got, z[:, :n] * z[:, n:], ("none", n))
        else:
            got = sh.linear_act(x, given, bias=bias, w_scale=scale, residual=residual, activation="relu")
            exact(got, z.clamp_min(0) + residual.double(), ("relu", n))
            exact(sh.linear_act(x, given, w_scale=scale), z - bias.double(), ("none", n))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form,kernel,size", PROJECTIONS)
def test_projections_of_normal_values(form, kernel, size, dtype):
    m, n, k = size
    gated = "gated" in form
    features = 2 * n if gated else n
    x, w = normal(1, m, k, dtype=dtype), normal(2, features, k, std=k ** -0.5, dtype=dtype)
    bias, scale, w64 = normal(3, features, std=0.3, dtype=dtype), None, w.double()
    if "e4m3" in form:
        scale = w.float().abs().amax(dim=-1) / 448.0
        codes = (w.float() / scale[:, None]).to(torch.float8_e4m3fn)
        w, w64 = codes.view(torch.uint8), codes.double() * scale.double()[:, None]
    if gated:
        got = sh.gated_linear(x, w, bias=bias, w_scale=scale, activation="gelu", gate_first=True)
        check_forward(x, w64, bias, "gelu", got, True, True)
    else:
        residual = normal(4, m, n, dtype=dtype)
        got = sh.linear_act(x, w, bias=bias, w_scale=scale, residual=residual, activation="gelu")
        check_forward(x, w64, bias, "gelu", got, False, residual=residual)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form,kernel,size", DZ)
def test_dz_of_integers(form, kernel, size, dtype):
    """All gradients of a call whose dz is exact: rows or columns that dz leaves out, and what stands in the columns it is
    padded with, show up in them."""
    m, _, k = size
    gated = form == "gated"
    for n in widths(*size):
        features = 2 * n if gated else n
        x, w = integers(1, m, k, dtype=dtype), integers(2, features, k, dtype=dtype)
        bias, dout = integers(3, features, limit=3, dtype=dtype), integers(4, m, n, dtype=dtype)
        z, d = x.double() @ w.double().t() + bias.double(), dout.double()
        for gate_first in (False, True)[:2 if gated else 1]:
            if gated:
                v, g = split(z, gate_first)
                dv, dg = d * g.clamp_min(0), d * v * (g > 0)
                dz = torch.cat((dg, dv) if gate_first else (dv, dg), -1)
                workspace = torch.full((sh.ff_backward_workspace_bytes(m, n, k, True, "relu", sh.F16 if dtype == F16 else sh.BF16),),
                                       255, dtype=torch.uint8, device=DEV)  # NaN where nothing is written
                grads = sh.gated_linear_backward(dout, x, w, bias=bias, activation="relu", gate_first=gate_first, workspace=workspace)
            else:
                dz = d * (z > 0)
                workspace = torch.full((sh.ff_backward_workspace_bytes(m, n, k, False, "relu", sh.F16 if dtype == F16 else sh.BF16),),
                                       255, dtype=torch.uint8, device=DEV)
                grads = sh.linear_act_backward(dout, x, w, bias=bias, activation="relu", workspace=workspace)
            for what, got, want in zip(("dx", "dw", "db"), grads, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))):
                exact(got, want, (what, n, gate_first))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form,kernel,size", DZ)
def test_dz_of_normal_values(form, kernel, size, dtype):
    m, n, k = size
    features = 2 * n if form == "gated" else n
    x, w = normal(1, m, k, dtype=dtype), normal(2, features, k, std=k ** -0.5, dtype=dtype)
    bias, dout = normal(3, features, std=0.3, dtype=dtype), normal(4, m, n, std=0.3, dtype=dtype)
    if form == "gated":
        grads = sh.gated_linear_backward(dout, x, w, bias=bias, activation="gelu", gate_first=True)
        check_backward(dout, x, w, bias, "gelu", grads, True, True)
    else:
        check_backward(dout, x, w, bias, "gelu", sh.linear_act_backward(dout, x, w, bias=bias, activation="gelu"), False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel", sizes.GRADIENTS)
def test_gradients_of_integers(kernel, dtype):
    wanted, (m, n, k) = sizes.GRADIENTS[kernel]
    x, w, dout = integers(1, m, k, dtype=dtype), integers(2, n, k, dtype=dtype), integers(3, m, n, dtype=dtype)
    want = {"dx": lambda: dout.double() @ w.double(), "dw": lambda: dout.double().t() @ x.double(), "dbias": lambda: dout.double().sum(0)}
    for with_sums in (False, True)[:2 if "dw" in wanted else 1]:
        grads = sh.linear_act_backward(dout, x, w, need_dx="dx" in wanted, need_dw="dw" in wanted, need_dbias=with_sums)
        for what, got in zip(("dx", "dw", "dbias"), grads):
            assert (got is not None) == (what in wanted or (what == "dbias" and with_sums))
            if got is not None:
                exact(got, want[what](), what)


@pytest.mark.parametrize("dtype,step", [(F16, 2.0 ** -24), (F16, 2.0 ** -20), (BF16, 2.0 ** -133)])
@pytest.mark.parametrize("form,kernel,size", cases(linear=sizes.LINEAR))
def test_subnormal_values_count(form, kernel, size, dtype, step):
    """Small gradients and activations, whole multiples of the type's smallest step, are not flushed on the way."""
    m, n, k = size
    x, w, dout = integers(1, m, k, dtype=dtype), integers(2, n, k, dtype=dtype), integers(3, m, n, dtype=dtype)
    small = lambda t: (t.double() * step).to(dtype)
    exact(sh.linear_act(small(x), w), x.double() @ w.double().t() * step, "x")
    exact(sh.linear_act(x, small(w)), x.double() @ w.double().t() * step, "w")
    dx, dw, db = sh.linear_act_backward(small(dout), x, w, need_dbias=True)
    for what, got, want in (("dx", dx, dout.double() @ w.double()), ("dw", dw, dout.double().t() @ x.double()), ("db", db, dout.double().sum(0))):
        exact(got, want * step, what)
    exact(sh.linear_act_backward(small(dout), x, w, need_dx=False, need_dw=False, need_dbias=True)[2], dout.double().sum(0) * step, "db alone")
