"""gshell_amd.optim.grad_norm / clip_grads / clip_grad_norm_ (csrc/gradnorm.hip) against the formulas in 64 bits.

The sums are in 64 bits, the norm is rounded once to fp32 (2^-24) on top of sums that are exact to 2^-40; the factor max_norm / (norm + 1e-6) takes two more roundings, the product one and the
element's type one: an output is off by (u + 5 * 2^-24) |out|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
W = 2.0 ** -24


def grads_of(sizes, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(dtype) for n in sizes]


def norm64(gs, p):
    flat = torch.cat([g.double().reshape(-1) for g in gs]) if gs else torch.zeros(1, dtype=torch.float64)
    return float(torch.linalg.vector_norm(flat, p)) if flat.numel() else 0.0


def check_clip(gs, max_norm, p, got_norm, got, extra=0.0):
    n = norm64(gs, p)
    assert abs(float(got_norm) - n) <= 2 * W * n
    coef = min(1.0, max_norm / (n + 1e-6))
    for g, o in zip(gs, got):
        ref = g.double() * coef
        u = torch.finfo(g.dtype).eps / 2
        assert ((o.cpu().double() - ref).abs() <= (u + 5 * W) * ref.abs() + (6e-8 if g.dtype == torch.float16 else 0)).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("p", [2.0, 1.0, float("inf")])
@pytest.mark.parametrize("sizes", [[1], [0], [0, 3, 0], [4096, 8192, 4097], [1, 2, 3, 5, 7, 20000, 33], [100003, 1]], ids=str)
def test_norm_and_clip(kind, p, sizes):
    from gshell_amd import optim
    gs = grads_of(sizes, TYPES[kind], 3)
    dev = [g.to(DEV) for g in gs]
    n = norm64(gs, p)
    assert abs(float(optim.grad_norm(dev, p)) - n) <= 2 * W * n
    for max_norm in (0.5, n, 2 * n + 1, float("inf"), 0.0):
        out = [torch.full_like(g, 9.0) for g in dev]
        check_clip(gs, max_norm, p, optim.clip_grads(dev, max_norm, p, out=out), out)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, gs))          # read only
        place = [g.clone() for g in dev]
        check_clip(gs, max_norm, p, optim.clip_grads(place, max_norm, p), place)
        assert all(torch.equal(a, b) for a, b in zip(place, out))


def test_more_tensors_than_one_launch_holds_of_mixed_types_and_odd_addresses():
    from gshell_amd import optim
    gen = torch.Generator().manual_seed(1)
    sizes = [int(v) for v in torch.randint(0, 3000, (307,), generator=gen)]
    gs, dev = [], []
    for k, n in enumerate(sizes):
        dtype = list(TYPES.values())[k % 3]
        base = torch.randn(n + 5, generator=gen).to(dtype)
        gs.append(base[k % 5:k % 5 + n])
        dev.append(base.to(DEV)[k % 5:k % 5 + n])
    first = optim.clip_grads(dev, 3.0)
    check_clip(gs, 3.0, 2.0, first, dev)
    again = [torch.empty_like(g, device=DEV) for g in gs]
    n2 = optim.clip_grads([g.to(DEV) for g in gs], 3.0, out=again)
    assert torch.equal(first, n2) and all(torch.equal(a, b) for a, b in zip(again, dev))


def test_neighbours_in_a_bucket_are_left_alone():
    from gshell_amd import optim
    flat = torch.randn(70000, device=DEV)
    held = flat.clone()
    parts = [flat[1:30001], flat[30003:66666]]
    optim.clip_grads(parts, 1.0)
    for a, b in ((0, 1), (30001, 30003), (66666, 70000)):
        assert torch.equal(flat[a:b], held[a:b])
    check_clip([held[1:30001].cpu(), held[30003:66666].cpu()], 1.0, 2.0, optim.grad_norm([held[1:30001], held[30003:66666]]), parts)


def test_squares_beyond_fp32_and_below():
    from gshell_amd import optim
    for scale in (1e25, 1e-30):
        gs = grads_of([5000, 17], torch.float32, 2, scale)
        n = norm64(gs, 2.0)
        assert abs(float(optim.grad_norm([g.to(DEV) for g in gs])) - n) <= 2 * W * n


@pytest.mark.parametrize("p", [2.0, 1.0, float("inf")])
def test_infinities_and_nan(p):
    from gshell_amd import optim
    for bad in (float("inf"), float("-inf"), float("nan")):
        gs = [g.to(DEV) for g in grads_of([300, 20000], torch.float32)]
        gs[1][777] = bad
        held = [g.clone() for g in gs]
        norm = optim.clip_grads(gs, 1.0, p)
        if math.isnan(bad):
            assert norm.isnan() and all(g.isnan().all() for g in gs)
        else:
            assert float(norm) == float("inf")
            assert not gs[0].any() and gs[1][777].isnan() and int((gs[1] != 0).sum()) == 1
        with pytest.raises(RuntimeError):
            ps = [torch.nn.Parameter(torch.zeros_like(h)) for h in held]
            for q, h in zip(ps, held):
                q.grad = h.clone()
            optim.clip_grad_norm_(ps, 1.0, p, error_if_nonfinite=True)
        assert all(torch.equal(q.grad, h) or h.isnan().any() for q, h in zip(ps, held))


def test_parameters_without_gradient_permuted_gradients_and_torchs_own():
    from gshell_amd import optim
    gen = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((40, 30), (7,), (12, 5), (3, 4, 5))]
    ref = [torch.nn.Parameter(torch.zeros_like(p)) for p in ps]
    for k in (0, 2, 3):
        g = torch.randn(ps[k].shape, generator=gen).to(DEV)
        ref[k].grad = g.clone()
        ps[k].grad = g.t().contiguous().t() if k == 2 else g.clone()
    assert not ps[2].grad.is_contiguous()
    version = ps[0].grad._version
    n = optim.clip_grad_norm_(ps, 1.5)
    m = torch.nn.utils.clip_grad_norm_(ref, 1.5)
    assert torch.allclose(n, m, rtol=1e-6) and ps[1].grad is None and ps[0].grad._version > version
    for a, b in zip(ps, ref):
        assert a.grad is None or torch.allclose(a.grad, b.grad, rtol=1e-6, atol=0)
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device=DEV))], 1.0)) == 0.0
    one = torch.nn.Parameter(torch.zeros(3, device=DEV))
    one.grad = torch.tensor([3.0, 0.0, 4.0], device=DEV)
    assert float(optim.clip_grad_norm_(one, 1.0)) == 5.0
    assert torch.allclose(one.grad, torch.tensor([0.6, 0.0, 0.8], device=DEV))


def test_a_captured_clip_replays():
    from gshell_amd import optim
    gs = [torch.randn(n, device=DEV) for n in (50000, 3, 4097)]
    out = [torch.empty_like(g) for g in gs]
    optim.clip_grads(gs, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grads(gs, 1.0, out=out)
    for _ in range(4):
        for g in gs:
            g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        held = [norm.clone()] + [o.clone() for o in out]
        want = [torch.empty_like(g) for g in gs]
        assert torch.equal(held[0], optim.clip_grads(gs, 1.0, out=want)) and all(torch.equal(a, b) for a, b in zip(held[1:], want))


def test_refusals_on_the_device():
    from gshell_amd import optim
    from gshell_amd._lib import GShellHipError
    g = torch.randn(6, 4, device=DEV)
    for bad in (g.to_sparse(), g.to_sparse_csr()):
        for call in (lambda: optim.grad_norm([g, bad]), lambda: optim.clip_grads([g, bad], 1.0)):      # noqa: B023
            with pytest.raises(GShellHipError, match="dense float32"):
                call()
    t = torch.empty(4, 6, device=DEV).t()
    a = torch.empty(12, 2, device=DEV)
    for grads, out, what in (([g, g.clone()], [t, t], "same output twice"), ([t, t], None, "same output twice"), ([g], [g.half()], "an output is"), ([g], [g.cpu()], "HBM"),
                             ([g], [torch.empty(4, 6, device=DEV)], "an output is"), ([g, g], None, "shares memory"), ([a[:, 0], a[:, 0]], None, "same output twice")):
        before = g.clone()
        with pytest.raises(GShellHipError, match=what):
            optim.clip_grads(grads, 1.0, out=out)
        assert torch.equal(g, before)


def test_views_of_one_tensor_clip_apart():
    """Columns of one matrix: not contiguous, each written from a copy; whole numbers over a power of two are exact."""
    from gshell_amd import optim
    a = torch.zeros(16, 3, device=DEV)
    a[:, 0], a[:, 2] = 3.0, 4.0
    n = optim.clip_grads([a[:, 0], a[:, 2]], 10.0)          # 4 * 5
    assert float(n) == 20.0
    want = torch.tensor([1.5, 0.0, 2.0], device=DEV).expand(16, 3)
    assert torch.allclose(a, want, rtol=4 * 2.0 ** -24, atol=0)
