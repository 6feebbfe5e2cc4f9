"""gshell_amd.nn.linear (csrc/linear.hip) against the formula in 64 bits.

Tolerances, per element, from the operations: u = eps / 2 of the layer's type (one rounding), w = 2^-24.  A product of K terms summed in 32 bits is off by at most
K w sum |x w| in the worst order (fp32 operands: the split leaves 2^-24 of every product besides); the activation has |act'| <= 1.13 and adds a few w of its own;
the result is rounded once.  In the backward pass gz carries the rounding of act' (fp16: 2^-11, next to bf16) and its own, 2 u at most relative to |g act'| -- and
what the forward sum's error moves act', |act''| <= max(1, beta / 4)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
W = 2.0 ** -24


def act64(z, act, beta):
    if act == "relu":
        return torch.relu(z), (z > 0).double()
    if act == "softplus":
        return torch.logaddexp(torch.zeros_like(z), z * beta) / beta, torch.sigmoid(z * beta)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def make(M, N, K, dtype, seed, bias=True, residual=True, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    x, w = (r(M, K) * scale).to(dtype), (r(N, K) / math.sqrt(max(K, 1))).to(dtype)
    return x, w, (r(N) * 0.1).to(dtype) if bias else None, r(M, N).to(dtype) if residual else None, r(M, N).to(dtype)


def check_all(x, w, b, r, g, act, beta, got, dtype):
    """got: y, dx, dw, db, dr on the CPU; x .. g on the CPU."""
    u = torch.finfo(dtype).eps / 2
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    za = xd.abs() @ wd.abs().t()
    if b is not None:
        z, za = z + b.double(), za + b.double().abs()
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    ez = (K + 16) * W * za + W * z.abs()
    y, d = act64(z, act, beta)
    ey = 1.13 * ez + 8 * W * (y.abs() + z.abs())
    if r is not None:
        y = y + r.double()
    ey = ey + (u + 2 * W) * y.abs() + 1e-30 + (6e-8 if dtype == torch.float16 else 0)
    assert torch.isfinite(got[0]).all() and ((got[0].double() - y).abs() <= ey).all(), float(((got[0].double() - y).abs() / ey).max())
    if len(got) == 1:
        return
    gd = g.double()
    gz = gd * d
    ed = {None: 0.0, "relu": 0.0, "softplus": beta / 4, "silu": 0.5, "gelu": 0.8}[act] * ez + (8 * W if act else 0.0)
    kept = 2.0 ** -11 if dtype == torch.bfloat16 and act not in (None, "relu") else W
    egz = gd.abs() * (ed + kept * d.abs() + (2.0 ** -25 if dtype == torch.bfloat16 and act else 0)) + ((u + W) * gz.abs() * 1.01 if act else 0) + (6e-8 if dtype == torch.float16 and act else 0)
    tiny = 6e-8 if dtype == torch.float16 else 1e-30
    for got_t, a, bb, ea, n in ((got[1], gz, wd, egz, N), (got[2], gz.t(), xd, egz.t(), M)):
        ref = a @ bb
        bar = ea @ bb.abs() + (n + 16) * W * (a.abs() @ bb.abs()) + (u + W) * ref.abs() + tiny
        assert torch.isfinite(got_t).all() and ((got_t.double() - ref).abs() <= bar).all(), float(((got_t.double() - ref).abs() / bar).max())
    k = 3
    if b is not None:
        ref = gz.sum(0)
        bar = egz.sum(0) + (M + 16) * W * gz.abs().sum(0) + (u + W) * ref.abs() + tiny
        assert ((got[k].double() - ref).abs() <= bar).all(), float(((got[k].double() - ref).abs() / bar).max())
        k += 1
    if r is not None:
        assert torch.equal(got[k], g)


def run(x, w, b, r, g, act, beta, train=True):
    from gshell_amd import nn
    leaf = [None if t is None else t.to(DEV).requires_grad_(train) for t in (x, w, b, r)]
    y = nn.linear(*leaf, activation=act, beta=beta)
    if not train:
        return [y.cpu()]
    grads = torch.autograd.grad(y, [t for t in leaf if t is not None], g.to(DEV))
    return [y.detach().cpu()] + [t.cpu() for t in grads]


SIZES = [(1, 1, 1), (1, 64, 64), (5, 3, 2), (17, 40, 24), (64, 128, 32), (130, 129, 33), (127, 256, 295), (300, 200, 8), (2, 1000, 777), (257, 16, 1031), (1000, 7, 515), (40, 520, 2050)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_and_gradients_over_sizes(kind, M, N, K):
    act = [None, "softplus", "silu", "gelu"][(M + N + K) % 4]
    ops = make(M, N, K, TYPES[kind], M * 7 + N)
    check_all(*ops, act, 1.0, run(*ops, act, 1.0), TYPES[kind])
    check_all(*ops, act, 1.0, run(*ops, act, 1.0, train=False), TYPES[kind])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act,beta", [(None, 1.0), ("softplus", 1.0), ("softplus", 100.0), ("silu", 1.0), ("gelu", 1.0)])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_epilogues(kind, act, beta, bias, residual):
    x, w, b, r, g = make(97, 72, 56, TYPES[kind], 3, bias, residual, 0.2 if beta > 1 else 1.0)
    check_all(x, w, b, r, g, act, beta, run(x, w, b, r, g, act, beta), TYPES[kind])


@pytest.mark.parametrize("kind", list(TYPES))
def test_relu_on_whole_numbers_is_exact(kind):
    """Small whole numbers: every sum is exact in 32 bits, so no pre-activation can round across zero, and zeros do occur."""
    g = torch.Generator().manual_seed(5)
    ri = lambda *s: torch.randint(-2, 3, s, generator=g).to(TYPES[kind])      # noqa: E731
    x, w, b, gy = ri(70, 24), ri(50, 24), ri(50), ri(70, 50)
    got = run(x, w, b, None, gy, "relu", 1.0)
    z = x.double() @ w.double().t() + b.double()
    assert (z == 0).any()
    gz = gy.double() * (z > 0)
    for a, ref in zip(got, (torch.relu(z), gz @ w.double(), gz.t() @ x.double(), gz.sum(0))):
        assert torch.equal(a.double(), ref)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K", [(4096, 64, 48), (20000, 40, 39), (3, 96, 4100), (16, 24, 9000)])
def test_long_contractions_shared_out_are_right_and_repeat(kind, M, N, K):
    ops = make(M, N, K, TYPES[kind], 11)
    first = run(*ops, "silu", 1.0)
    check_all(*ops, "silu", 1.0, first, TYPES[kind])
    again = run(*ops, "silu", 1.0)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("kind", list(TYPES))
def test_strided_views_and_leading_dimensions(kind):
    from gshell_amd import nn
    dtype = TYPES[kind]
    g = torch.Generator().manual_seed(8)
    big_x, big_w, big_r = (torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((33, 130), (50, 111), (33, 77)))
    x, w, r = big_x[:, 5:69], big_w[3:40, 7:71], big_r[:, 1:38]
    ref = nn.linear(x.contiguous(), w.contiguous(), None, r.contiguous(), "gelu")
    assert torch.equal(nn.linear(x, w, None, r, "gelu"), ref)
    assert torch.equal(nn.linear(x.t().contiguous().t(), w.t().contiguous().t(), None, r.t().contiguous().t(), "gelu"), ref)
    assert torch.equal(nn.linear(x.reshape(3, 11, 64), w, None, r.reshape(3, 11, 37), "gelu").reshape(33, 37), ref)
    row = nn.linear(x[0], w, None, r[0], "gelu")
    assert row.shape == (37,)
    # an expanded residual and an expanded gradient
    one = torch.randn(37, generator=g).to(dtype).to(DEV).requires_grad_(True)
    xs = x.detach().clone().requires_grad_(True)
    y = nn.linear(xs, w, None, one.expand(33, 37), "gelu")
    y.sum().backward()
    assert torch.allclose(one.grad.float(), torch.full((37,), 33.0, device=DEV))
    x2 = x.detach().clone().requires_grad_(True)
    nn.linear(x2, w, None, None, "gelu").backward(torch.ones(33, 37, dtype=dtype, device=DEV))
    assert torch.equal(xs.grad, x2.grad)


@pytest.mark.parametrize("kind", list(TYPES))
def test_empty_sizes(kind):
    from gshell_amd import nn
    dtype = TYPES[kind]
    z = lambda *s: torch.ones(*s, dtype=dtype, device=DEV, requires_grad=True)      # noqa: E731
    for M, N, K in ((0, 8, 8), (4, 0, 8), (4, 8, 0), (0, 0, 0)):
        x, w, b = z(M, K), z(N, K), z(N)
        y = nn.linear(x, w, b, activation="silu")
        assert y.shape == (M, N)
        y.backward(torch.ones_like(y))
        assert x.grad.shape == (M, K) and not x.grad.any()
        assert w.grad.shape == (N, K) and not w.grad.any()
        if K == 0:
            s = torch.sigmoid(torch.ones((), dtype=torch.float64))
            assert torch.allclose(y.double().cpu(), s.expand(M, N), rtol=0.01)
            assert b.grad.all()
        else:
            assert not b.grad.any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M", [1, 40, 300])
def test_infinities_and_nan_stay_in_their_rows(kind, M):
    dtype = TYPES[kind]
    x, w, _, _, _ = make(M, 70, 90, dtype, 4)
    w = w.abs() + 0.125
    x = x.abs() + 0.125
    x[0, 17] = float("inf")
    if M > 1:
        x[M - 1, 3] = float("nan")
        x[M // 2, 5], x[M // 2, 6] = float("inf"), float("-inf")
    got = run(x, w, None, None, None, None, 1.0, train=False)[0]
    assert (got[0] == float("inf")).all()
    if M > 1:
        assert got[M - 1].isnan().all() and got[M // 2].isnan().all()
        keep = [i for i in range(M) if i not in (0, M - 1, M // 2)]
        ref = x[keep].double() @ w.double().t()
        assert torch.allclose(got[keep].double(), ref, rtol=0.01)


def test_fp32_operands_keep_fp32_accuracy_over_their_range():
    """The split covers fp32's exponents: scaled by powers of two the products keep their relative accuracy (2^-24 each from the split, the rest from summing)."""
    x, w, _, _, _ = make(64, 96, 512, torch.float32, 21)
    for sx, sw in ((1.0, 1.0), (2.0 ** 60, 2.0 ** -70), (2.0 ** -60, 2.0 ** 40), (2.0 ** 100, 2.0 ** 10)):
        got = run(x * sx, w * sw, None, None, None, None, 1.0, train=False)[0].double() / (sx * sw)
        ref = x.double() @ w.double().t()
        bar = (512 + 16) * W * (x.double().abs() @ w.double().abs().t())
        assert ((got - ref).abs() <= bar).all()
        rms = ((got - ref).pow(2).mean() / ref.pow(2).mean()).sqrt()
        assert rms < 512 ** 0.5 * W, rms          # errors of 512 random signs add like their root
    top = torch.full((1, 4), 3.4e38)          # rounds to bf16's infinity: the sum is done again in fp32
    got = run(top, torch.tensor([[0.5, 0.25, 0.0, 0.125]]), None, None, None, None, 1.0, train=False)[0]
    assert torch.allclose(got.double(), torch.tensor([[3.4e38 * 0.875]], dtype=torch.float64), rtol=1e-6)


@pytest.mark.parametrize("act,beta", [("softplus", 3.0), ("silu", 1.0), ("gelu", 1.0)])
def test_gradients_against_differences(act, beta):
    """Central differences of the layer's own fp32 output: with h = 2^-6 the formula is off by h^2 / 6 of a third derivative (< 2 beta^2) and the outputs' roundings
    (2^-22 on values below 8) by 2^-22 / h."""
    from gshell_amd import nn
    g = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=g).to(DEV) * f for s, f in (((6, 9), 1.0), ((5, 9), 0.3), ((5,), 0.1)))
    h = 2.0 ** -6
    for k, t in enumerate((x, w, b)):
        leaf = [v.clone().requires_grad_(True) for v in (x, w, b)]
        nn.linear(*leaf, activation=act, beta=beta).sum().backward()
        for at in range(0, t.numel(), 4):
            lo, hi = [v.clone() for v in (x, w, b)], [v.clone() for v in (x, w, b)]
            lo[k].view(-1)[at] -= h
            hi[k].view(-1)[at] += h
            diff = (nn.linear(*hi, activation=act, beta=beta).double().sum() - nn.linear(*lo, activation=act, beta=beta).double().sum()) / (2 * h)
            third = 2 * beta ** 2 * (float(w.abs().max()) ** 3 * 5 if k == 0 else float(x.abs().max()) ** 3 * 6)
            assert abs(float(diff) - float(leaf[k].grad.view(-1)[at])) <= h * h / 6 * third + 30 * 2.0 ** -22 / h


def test_a_captured_step_replays():
    from gshell_amd import nn
    x, w, b, r, g = (t.to(DEV) for t in make(200, 96, 700, torch.bfloat16, 6))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))

    def step():
        y = nn.linear(x, w, b, r, "gelu")
        return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(make(200, 96, 700, torch.bfloat16, 60 + k)[0].to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in out]
        for a, b_ in zip(held, step()):
            assert torch.equal(a, b_)


def test_side_stream_and_module():
    from gshell_amd import nn
    torch.manual_seed(0)
    lin = nn.Linear(48, 80, activation="softplus", beta=100.0).to(DEV)
    plain = torch.nn.Linear(48, 80)
    plain.load_state_dict({k: v.cpu() for k, v in lin.state_dict().items()})
    x = torch.randn(33, 48, device=DEV) * 0.2
    y = lin(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y2 = lin(x)
    side.synchronize()
    assert torch.equal(y, y2)
    ref = torch.nn.functional.softplus(plain(x.cpu()).double(), beta=100)
    assert torch.allclose(y.detach().cpu().double(), ref, atol=1e-6)


def test_a_second_differentiation_raises():
    from gshell_amd import nn
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    gx, = torch.autograd.grad(nn.linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
