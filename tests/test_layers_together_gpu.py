"""Embedding, dense layers, the gradient's clipping and the optimiser as one training step; and the calls of gshell_amd.nn and gshell_amd.optim that only a whole program makes:
two streams, two graphs, one weight in two layers, masked gradients that are not finite, results of more than 2^31 elements."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
W = 2.0 ** -24
V, D, F, C = 300, 48, 64, 24          # rows of the table, widths


class Net(torch.nn.Module):
    def __init__(self, dtype=torch.float32):
        super().__init__()
        from gshell_amd import nn
        torch.manual_seed(11)
        self.table = nn.Embedding(V, D, padding_idx=0, scale=math.sqrt(D), dtype=dtype)
        self.up, self.down = nn.Linear(D, F, activation="gelu", dtype=dtype), nn.Linear(F, D, dtype=dtype)
        self.head = nn.Linear(D, C, activation="softplus", beta=2.0, dtype=dtype)
        with torch.no_grad():
            self.table.weight.mul_(D ** -0.5)

    def forward(self, ids):
        e = self.table(ids)
        return self.head(self.down(self.up(e), residual=e))


def plain64(net, ids, g):
    """Output and gradients of Net by torch, in 64 bits on the CPU."""
    p = {n: q.detach().cpu().double().requires_grad_(True) for n, q in net.named_parameters()}
    fn = torch.nn.functional
    e = fn.embedding(ids.cpu(), p["table.weight"], padding_idx=0) * math.sqrt(D)
    h = fn.gelu(fn.linear(e, p["up.weight"], p["up.bias"]))
    y = fn.softplus(fn.linear(fn.linear(h, p["down.weight"], p["down.bias"]) + e, p["head.weight"], p["head.bias"]), beta=2.0, threshold=60)
    y.backward(g.cpu().double())
    return y.detach(), {n: q.grad for n, q in p.items()}


def near(a, ref, bar):
    a = a.detach().cpu().double()
    assert float((a - ref).norm()) <= bar * float(ref.norm()), float((a - ref).norm() / ref.norm())


@pytest.mark.parametrize("shape", [(1,), (7,), (5, 61), (40, 128)], ids=str)
def test_a_training_step(shape):
    """A product of K terms in 32 bits is off by at most (K + 16) w |x| |w|, in norms (64 + 16) w sqrt(64) of the result for weights without a direction: 4e-5.  A gradient here
    comes through six of them at most, with act' <= 1.13, and two sums over the tokens, which add their own number of terms times w: 1e-3 holds all of it."""
    from gshell_amd import optim
    net = Net().to(DEV)
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, V, shape, generator=gen).to(DEV)
    g = torch.randn(*shape, C, generator=gen).to(DEV)
    params = list(net.parameters())
    start = [p.detach().clone() for p in params]
    opt = optim.HipAdam(params, lr=1e-2)
    y = net(ids)
    y.backward(g)
    ref, grads = plain64(net, ids, g)
    near(y, ref, 1e-3)
    for n, p in net.named_parameters():
        near(p.grad, grads[n], 1e-3)
    assert not net.table.weight.grad[0].any()
    before = [p.grad.clone() for p in params]
    total = math.sqrt(sum(float(b.double().pow(2).sum()) for b in before))
    n = optim.clip_grad_norm_(params, 0.5 * total)
    assert abs(float(n) - total) <= 2 * W * total
    for p, b in zip(params, before):          # the factor has the rounding of the norm and its own, the product one more
        assert ((p.grad.double() - b.double() * 0.5).abs() <= 6 * W * b.double().abs() + 1e-6 / total).all()
    opt.step()
    other = [torch.nn.Parameter(s) for s in start]
    for o, p in zip(other, params):
        o.grad = p.grad.clone()
    torch.optim.Adam(other, lr=1e-2, fused=True).step()
    for o, p in zip(other, params):
        assert torch.equal(o, p)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_captured_step_replays(kind):
    from gshell_amd import optim
    net = Net(TYPES[kind]).to(DEV)
    params = list(net.parameters())
    ids = torch.randint(0, V, (33, 70), device=DEV)
    g = torch.randn(33, 70, C, device=DEV).to(TYPES[kind])

    def step():
        y = net(ids)
        grads = torch.autograd.grad(y, params, g)
        norm = optim.clip_grads(grads, 1.0)
        return [y.detach(), norm, *grads]
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
        ids.random_(0, V)
        with torch.no_grad():
            for p in params:
                p.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in out]
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def _layer(dtype, seed, M=700, N=130, K=1100):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=gen) / 8).to(dtype).to(DEV)      # noqa: E731
    return r(M, K).requires_grad_(True), r(N, K).requires_grad_(True), r(N).requires_grad_(True), r(M, N)


@pytest.mark.parametrize("kind", list(TYPES))
def test_two_streams_at_once(kind):
    from gshell_amd import nn, optim
    sets = [_layer(TYPES[kind], s) for s in (1, 2)]

    def step(x, w, b, g):
        y = nn.linear(x, w, b, activation="silu")
        grads = torch.autograd.grad(y, [x, w, b], g)
        return [y.detach(), optim.clip_grads(grads, 0.1), *grads]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for result in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[k]))


@pytest.mark.parametrize("kind", list(TYPES))
def test_two_graphs_replayed_in_turn(kind):
    from gshell_amd import nn, optim
    sets = [_layer(TYPES[kind], s) for s in (3, 4)]
    ids = [torch.randint(0, 130, (3000,), device=DEV) for _ in sets]

    def step(k):
        x, w, b, g = sets[k]
        y = nn.linear(x, w, b, activation="gelu")
        grads = torch.autograd.grad(y, [x, w, b], g)
        table = torch.autograd.grad(nn.embedding(ids[k], w), w, x.detach().reshape(-1)[:1100].expand(3000, 1100))
        return [y.detach(), optim.clip_grads([*grads, *table], 0.1), *grads, *table]
    want = [step(k) for k in (0, 1)]
    want = [[t.clone() for t in w] for w in want]
    torch.cuda.synchronize()
    graphs, out = [torch.cuda.CUDAGraph() for _ in sets], []
    for k, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            out.append(step(k))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(out[k], want[k]))
            for t in out[k]:
                t.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("kind", list(TYPES))
def test_one_weight_in_two_layers_and_as_its_own_input(kind):
    """Small whole numbers: every sum is exact in 32 bits, and in the layer's type where it is below 2^8 (bf16), so the gradients are."""
    from gshell_amd import nn
    gen = torch.Generator().manual_seed(9)
    w = torch.zeros(40, 40)
    w[torch.arange(40), torch.randperm(40, generator=gen)] = 1.0
    w[torch.arange(40), torch.randperm(40, generator=gen)] += 1.0
    x = torch.randint(-1, 2, (50, 40), generator=gen).float()
    g = torch.zeros(50, 40)
    g[torch.arange(50), torch.randint(0, 40, (50,), generator=gen)] = 1.0
    dev = [t.to(TYPES[kind]).to(DEV).requires_grad_(True) for t in (x, w)]
    ref = [t.double().requires_grad_(True) for t in (x, w)]
    y = nn.linear(nn.linear(*dev), dev[1])
    got = torch.autograd.grad(y, dev, g.to(y))
    yr = ref[0] @ ref[1].t() @ ref[1].t()
    assert torch.equal(y.cpu().double(), yr)
    for a, b in zip(got, torch.autograd.grad(yr, ref, g.double())):
        assert float(b.abs().max()) < 256 and torch.equal(a.cpu().double(), b)
    y = nn.linear(dev[1], dev[1], residual=dev[1])
    yr = ref[1] @ ref[1].t() + ref[1]
    assert torch.equal(torch.autograd.grad(y, dev[1], g[:40].to(y))[0].cpu().double(), torch.autograd.grad(yr, ref[1], g[:40].double())[0])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K", [(1, 30, 20), (40, 70, 50), (600, 260, 130)])
def test_what_relu_masks_passes_nothing(kind, M, N, K):
    """Gradients that are infinite or NaN where the derivative is zero leave no trace: the same bits as with zeros there (whole numbers: every order of the sums is exact)."""
    from gshell_amd import nn
    gen = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randint(-2, 3, s, generator=gen).to(TYPES[kind]).to(DEV)      # noqa: E731
    x, w, b, g = r(M, K).requires_grad_(True), r(N, K).requires_grad_(True), r(N).requires_grad_(True), r(M, N)
    y = nn.linear(x, w, b, activation="relu")
    off = y.detach() == 0
    assert off.any()
    clean, dirty = g.masked_fill(off, 0.0), g.masked_fill(off, float("inf"))
    dirty[off & (torch.arange(N, device=DEV) % 2 == 0)] = float("nan")
    want = torch.autograd.grad(y, [x, w, b], clean, retain_graph=True)
    got = torch.autograd.grad(y, [x, w, b], dirty)
    for a, c in zip(got, want):
        assert torch.isfinite(c).all() and torch.equal(a, c)


@pytest.mark.parametrize("kind,M,N", [("bf16", 2 ** 21 + 5, 1030), ("bf16", 2 ** 20 + 1, 2056), ("fp32", 2 ** 20 + 3, 2051)])
def test_layers_of_more_than_2_to_the_31_outputs(kind, M, N):
    """Rows near both ends; a gradient that is zero but in the last rows, so that a 64-bit sum over those is the whole."""
    from gshell_amd import nn
    dtype, K, last = TYPES[kind], 8, 100
    assert M * N > 2 ** 31
    u = torch.finfo(dtype).eps / 2
    x = (torch.randint(-4, 5, (M, K), device=DEV) / 4).to(dtype).requires_grad_(True)
    w = (torch.randint(-4, 5, (N, K), device=DEV) / 4).to(dtype).requires_grad_(True)
    y = nn.linear(x, w, activation="softplus")
    for rows in (slice(0, 50), slice(M // 2, M // 2 + 50), slice(M - last, M)):
        z = x[rows].double() @ w.double().t()
        ref = torch.logaddexp(torch.zeros_like(z), z)
        assert ((y[rows].double() - ref).abs() <= (u + 32 * W) * ref).all()          # |z| <= 8: the exponent's rounding is 16 w at most
    g = torch.zeros_like(y)
    g[-last:] = torch.randint(-2, 3, (last, N), device=DEV).to(dtype)
    dx, dw = torch.autograd.grad(y, [x, w], g)
    gz = g[-last:].double() * torch.sigmoid(x[-last:].double() @ w.double().t())
    # gz: act' (2^-11 as fp16 keeps it, next to bf16) and its own rounding; sums of N and of `last` terms; the result's rounding
    per = 2 * u + 32 * W if dtype == torch.bfloat16 else 32 * W
    assert not dx[:-last].any()
    for got, a, b, n in ((dx[-last:], gz, w.double(), N), (dw, gz.t(), x[-last:].double(), last)):
        ref = a @ b
        assert ((got.double() - ref).abs() <= (per + (n + 16) * W) * (a.abs() @ b.abs()) + (u + W) * ref.abs()).all()


def test_one_row_of_more_columns_than_the_kernel_for_few_rows_takes():
    from gshell_amd import nn
    N = 2 ** 27 + 9
    w = (torch.arange(N, device=DEV) % 1000).float()[:, None]
    y = nn.linear(torch.tensor([[2.0], [3.0]], device=DEV), w)
    assert torch.equal(y[0], 2.0 * w[:, 0]) and torch.equal(y[1], 3.0 * w[:, 0])


def test_a_lookup_of_more_than_2_to_the_31_elements():
    from gshell_amd import nn
    T, D_, last = 2 ** 20 + 1, 2056, 64
    table = torch.randint(-50, 51, (10, D_), device=DEV).to(torch.bfloat16).requires_grad_(True)
    ids = torch.randint(0, 10, (T,), device=DEV)
    y = nn.embedding(ids, table)
    for rows in (slice(0, 50), slice(T - last, T)):
        assert torch.equal(y[rows], table[ids[rows]])
    g = torch.zeros_like(y)
    g[-last:] = torch.randint(-2, 3, (last, D_), device=DEV).to(torch.bfloat16)
    dw, = torch.autograd.grad(y, table, g)
    ref = torch.zeros(10, D_, dtype=torch.float64, device=DEV).index_add_(0, ids[-last:], g[-last:].double())
    assert torch.equal(dw.double(), ref)          # whole numbers of 128 at most


def test_tokens_of_a_table_by_the_tens_of_millions():
    """More chunks of the sorted list than one side of the grid that joins them has; sums of whole numbers below 2^24 are exact."""
    from gshell_amd import nn
    T = 2 ** 25 + 100
    table = torch.zeros(3, 1, device=DEV, requires_grad=True)
    ids = torch.randint(0, 3, (T,), device=DEV)
    g = torch.randint(-1, 2, (T, 1), device=DEV).float()
    dw, = torch.autograd.grad(nn.embedding(ids, table), table, g)
    assert torch.equal(dw[:, 0].double(), torch.stack([g[ids == k].double().sum() for k in range(3)]))


def test_a_gradient_of_more_than_2_to_the_31_elements():
    from gshell_amd import optim
    g = torch.zeros(2 ** 31 + 5, dtype=torch.bfloat16, device=DEV)
    g[0], g[2 ** 31 - 1], g[-1] = 2.0, 10.0, -11.0
    assert float(optim.clip_grads([g], 1.5)) == 15.0          # 4 + 100 + 121
    for at, v in ((0, 0.2), (2 ** 31 - 1, 1.0), (-1, -1.1)):
        assert abs(float(g[at]) - v) <= 2 ** -8 * abs(v)
    assert int(torch.count_nonzero(g.view(torch.int16)).item()) == 3


@pytest.mark.timeout(120)
def test_the_trainer_clips_by_the_joint_norm(monkeypatch):
    from gshell_amd import train, workload
    tr = workload.build(res=16, n_samples=2, batch=1, train_res=(64, 64), fit_steps=60)
    target = workload.make_targets(tr, [0], (64, 64))
    tr.it = 1000
    tr.FLAGS.clip_max_norm = 1e-3
    seen = []

    def spy(params, max_norm, **kw):
        other = [torch.nn.Parameter(p.detach()) for p in params]
        for o, p in zip(other, params):
            o.grad = None if p.grad is None else p.grad.clone()
        ours, torchs = train_clip(params, max_norm, **kw), torch.nn.utils.clip_grad_norm_(other, max_norm)
        seen.append((ours, torchs, [(p.grad, o.grad) for p, o in zip(params, other) if p.grad is not None]))
        return ours
    train_clip = train.clip_grad_norm_
    monkeypatch.setattr(train, "clip_grad_norm_", spy)
    tr.step(target)
    (ours, torchs, grads), = seen
    # torch sums squares in 32 bits, tensor by tensor in a tree: a few hundred roundings at most
    assert float(ours) > 1e-3 and abs(float(ours) - float(torchs)) <= 512 * W * float(torchs)
    assert len(grads) > 3
    for a, b in grads:
        assert ((a - b).abs() <= 1024 * W * b.abs()).all()


def test_torch_func_says_that_it_is_not_taken_part_in():
    from gshell_amd import nn
    x, w = torch.randn(5, 8, device=DEV), torch.randn(4, 8, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda q: nn.linear(q, w).sum())(x)
    ids, table = torch.arange(4, device=DEV), torch.randn(6, 3, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: nn.embedding(ids, t).sum())(table)


def test_forward_mode_and_vmap_raise():
    import torch.autograd.forward_ad as fa
    from gshell_amd import nn
    x, w = torch.randn(5, 8, device=DEV), torch.randn(4, 8, device=DEV)
    with fa.dual_level():
        with pytest.raises(NotImplementedError):
            nn.linear(fa.make_dual(x, torch.ones_like(x)), w)
        with pytest.raises(NotImplementedError):
            nn.embedding(torch.arange(3, device=DEV), fa.make_dual(w, torch.ones_like(w)))
        assert torch.equal(nn.linear(x, w), nn.linear(x, w))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: nn.linear(q, w))(x[:, None])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: nn.embedding(torch.arange(3, device=DEV), q))(w[None])
