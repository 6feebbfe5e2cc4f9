"""gshell_amd.nn.linear where an activation saturates: y and the gradients of each column relative to that column's own values.

x is one input of 1 and w[n] the pre-activation of column n, so that z is exact and every row of a column has the same z.  Tolerances: u = eps / 2 of the layer's type, w = 2^-24.
A sum of M terms of one sign in 32 bits is off by M w of itself; every result is rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
W = 2.0 ** -24


def tail(act, z, beta):
    """y and act' for z < 0 in 64 bits, without cancellation."""
    if act == "softplus":
        return torch.log1p(torch.exp(beta * z)) / beta, 1 / (1 + torch.exp(-beta * z))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def column_inputs(lo, hi, dtype, N=96, scale=1.0):
    return (torch.linspace(lo, hi, N, dtype=torch.float64) * scale).to(dtype)


@pytest.mark.parametrize("M", [24, 200])
@pytest.mark.parametrize("act,beta,lo,hi", [("softplus", 1.0, -22.0, -12.0), ("softplus", 1.0, -85.0, -20.0), ("softplus", 100.0, -0.85, -0.12), ("silu", 1.0, -85.0, -9.0), ("gelu", 1.0, -12.5, -4.0)])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_gradients_of_saturated_columns(kind, act, beta, lo, hi, M):
    """act' reaches the backward pass with half a step of the layer's type (fp32: as it is) and is off by itself by the exponent's roundings, 4 w |exponent|, and 32 w (exponential,
    reciprocal, polynomial: some ten roundings).  16-bit gelu's Phi, 4e-5 of itself, is at most a tenth of z pdf here.  dW takes gz rounded once more, db does not."""
    from gshell_amd import nn
    dtype, N = TYPES[kind], 96
    u = torch.finfo(dtype).eps / 2
    z = column_inputs(lo, hi, dtype)
    w = torch.zeros(N, 8, dtype=dtype)
    w[:, 0] = z
    x = torch.zeros(M, 8, dtype=dtype)
    x[:, 0] = 1
    g = (torch.rand(M, N, generator=torch.Generator().manual_seed(M)) + 0.5).to(dtype)
    leaf = [t.to(DEV).requires_grad_(True) for t in (x, w, torch.zeros(N, dtype=dtype))]
    y = nn.linear(*leaf, activation=act, beta=beta)
    _, dw, db = (t.cpu().double() for t in torch.autograd.grad(y, leaf, g.to(DEV)))
    _, d = tail(act, z.double(), beta)
    exponent = (z.double() ** 2 / 2) if act == "gelu" else (beta * z.double()).abs()
    ref = g.double().sum(0) * d
    kept = (u if kind == "bf16" else 0) + 4 * W * exponent + 32 * W + 1e-5 * (act == "gelu" and kind == "bf16")
    # fp32 products: a value's three bf16 parts count where they are 2^-126 or more, so a term lacks at most two parts of less than that
    lost = M * 2.0 ** -125 if kind == "fp32" else 0
    for got, extra, low in ((db, 0, 0), (dw[:, 0], u, lost)):
        bar = (kept + extra + u + M * W) * 1.01 * ref.abs() + low
        assert ((got - ref).abs() <= bar).all(), float(((got - ref).abs() / ref.abs()).max())


def test_an_infinite_gradient_passes_where_the_derivative_is_not_zero():
    from gshell_amd import nn
    for dtype in TYPES.values():
        w = torch.full((16, 8), -8.0, dtype=dtype, device=DEV)
        x = torch.ones(40, 8, dtype=dtype, device=DEV, requires_grad=True)
        b = torch.zeros(16, dtype=dtype, device=DEV, requires_grad=True)
        y = nn.linear(x, w, b, activation="softplus")          # act'(-64) = 1.6e-28
        g = torch.zeros_like(y)
        g[3, 5] = float("inf")
        dx, db = torch.autograd.grad(y, [x, b], g)
        assert (dx[3] == float("-inf")).all() and db[5] == float("inf") and not db[:5].any() and not db[6:].any()


@pytest.mark.parametrize("M", [5, 130])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_gelu_of_16_bit_layers_is_relative_in_its_tail(kind, M):
    """Phi(z) is 2^-14 of itself there and the exponential 4 w z^2 / 2; the result is rounded once, fp16's below 2^-14 by half of 2^-24."""
    from gshell_amd import nn
    dtype = TYPES[kind]
    u = torch.finfo(dtype).eps / 2
    z = column_inputs(-8.0, -3.0, dtype, N=512)
    w = torch.zeros(512, 8, dtype=dtype)
    w[:, 0] = z
    x = torch.zeros(M, 8, dtype=dtype)
    x[:, 0] = 1
    got = nn.linear(x.to(DEV), w.to(DEV), activation="gelu").cpu().double()
    ref, _ = tail("gelu", z.double(), 1.0)
    # the approximation shows where the rounding to the layer's type does not hide it: it moves a result by one step at most, and only next to a border between two
    err = (got - ref).abs()
    bar = (u + 2.0 ** -14 + 2 * W * z.double() ** 2 + 16 * W) * ref.abs() + (2.0 ** -25 if kind == "fp16" else 0)
    assert (err <= bar).all(), float((err / bar).max())


@pytest.mark.parametrize("M", [5, 130])
@pytest.mark.parametrize("beta", [1.0, 3.0, 100.0])
def test_fp32_softplus_is_relative_in_its_tail(beta, M):
    """exp2, the reciprocal (one step each), the polynomial (2^-26) and some ten roundings: 24 w of the result, wherever the exponent is; results below
    2^-126 are multiples of 2^-149."""
    from gshell_amd import nn
    z = column_inputs(-85.0, -2.0, torch.float32, N=768, scale=1 / beta)
    w = torch.zeros(768, 8)
    w[:, 0] = z
    x = torch.zeros(M, 8)
    x[:, 0] = 1
    got = nn.linear(x.to(DEV), w.to(DEV), activation="softplus", beta=beta).cpu().double()
    ref, _ = tail("softplus", z.double(), beta)
    assert ((got - ref).abs() <= 24 * W * ref + 2.0 ** -149).all(), float(((got - ref).abs() / ref).max() / W)


def test_softplus_ends():
    from gshell_amd import nn
    inf = float("inf")
    z = torch.tensor([inf, -inf, float("nan"), 3e38, -3e38, 0.0, 1e-30, -1e-30], device=DEV)
    for beta in (1.0, 100.0, 1e-3):
        w = torch.ones(1, 1, device=DEV)
        x = z[:, None].clone().requires_grad_(True)
        y = nn.linear(x, w, activation="softplus", beta=beta)
        dx, = torch.autograd.grad(y.sum(), x)
        y, dx = y[:, 0].detach().cpu().double(), dx[:, 0].cpu().double()
        ref, d = torch.logaddexp(torch.zeros(8, dtype=torch.float64), z.cpu().double() * beta) / beta, torch.sigmoid(z.cpu().double() * beta)
        assert torch.allclose(y, ref, rtol=1e-5, equal_nan=True), (beta, y, ref)
        assert torch.allclose(dx, d, rtol=1e-5, equal_nan=True), (beta, dx, d)
