"""fp32 layers with infinities and NaN in their operands: the outputs that meet none keep their bits, the others are what 64-bit products give, and a step of nothing but NaN costs a few
times an ordinary one."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def step(x, w, b, g, act):
    from gshell_amd import nn
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = nn.linear(*leaf, activation=act)
    return [y.detach()] + list(torch.autograd.grad(y, leaf, g))


def same_kind(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a == INF, b == INF) and torch.equal(a == -INF, b == -INF)


@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("M,N,K", [(40, 24, 17), (300, 200, 100), (257, 129, 295), (5000, 72, 40)])
def test_only_what_meets_them_changes(M, N, K, act):
    gen = torch.Generator().manual_seed(M)
    x, w, b, g = (torch.randn(*s, generator=gen).to(DEV) for s in ((M, K), (N, K), (N,), (M, N)))
    clean = step(x, w, b, g, act)
    x2, g2 = x.clone(), g.clone()
    x2[3, 5] = INF
    x2[M - 1, K - 1], x2[M - 1, 0] = INF, -INF
    x2[M // 2, 1] = NAN
    g2[7, N - 1] = INF
    g2[M - 2, 2] = NAN
    got = step(x2, w, b, g2, act)
    rows = torch.ones(M, dtype=torch.bool, device=DEV)
    rows[[3, M // 2, M - 1]] = False
    assert torch.equal(got[0][rows], clean[0][rows])
    z = x2.double() @ w.double().t() + b.double()
    y = torch.where(z < 0, 0.0, z) if act else z
    assert same_kind(got[0].double(), y)
    # where the derivative is zero nothing passes, an infinity or NaN neither (relu of z <= 0; of a NaN it is 1)
    gz = torch.where(z <= 0, 0.0, g2.double()) if act else g2.double()
    dx = gz @ w.double()
    assert same_kind(got[1].double(), dx) and same_kind(got[3].double(), gz.sum(0))
    quiet = torch.ones(M, dtype=torch.bool, device=DEV)
    quiet[[3, 7, M // 2, M - 2, M - 1]] = False
    assert torch.equal(got[1][quiet], clean[1][quiet])
    dw = gz.t() @ x2.double()
    assert same_kind(got[2].double(), dw)
    fine = dw.isfinite()
    assert torch.allclose(got[2][fine].double(), dw[fine], rtol=1e-4, atol=1e-4 * M ** 0.5)
    fine = dx.isfinite()
    assert torch.allclose(got[1][fine].double(), dx[fine], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("M,N,K", [(32768, 256, 256), (4096, 1024, 1024)])
def test_nothing_but_nan_costs_a_few_times_an_ordinary_step(M, N, K):
    """The redone sums run on the fp32 matrix instruction, 16 / 6 of the six products' time and less well fed: 20 times is far above that, and far below a sum at a time (100 and more)."""
    gen = torch.Generator().manual_seed(1)
    x, w, b, g = (torch.randn(*s, generator=gen).to(DEV) for s in ((M, K), (N, K), (N,), (M, N)))

    def time(x, g):
        best = 1e9
        for _ in range(4):
            a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = step(x, w, b, g, "softplus")
            e.record()
            e.synchronize()
            best = min(best, a.elapsed_time(e))
        return best, out
    clean, _ = time(x, g)
    bad, out = time(torch.full_like(x, NAN), torch.full_like(g, NAN))
    assert all(t.isnan().all() for t in out)
    assert bad <= 20 * clean, (clean, bad)
