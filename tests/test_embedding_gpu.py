"""gshell_amd.nn.embedding (csrc/embedding.hip) against the formula in 64 bits.

A looked-up value is scaled in 32 bits and rounded once.  A row's gradient is a 32-bit sum of n values, scaled, rounded once: at most n 2^-24 sum |g| + (u + 2^-23) |sum|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
W = 2.0 ** -24


def check_one(ids, V, D, dtype, scale, pad, seed=0):
    from gshell_amd import nn
    gen = torch.Generator().manual_seed(seed)
    u = torch.finfo(dtype).eps / 2
    w = torch.randn(V, D, generator=gen).to(dtype)
    g = torch.randn(ids.shape + (D,), generator=gen).to(dtype)
    wd = w.to(DEV).requires_grad_(True)
    y = nn.embedding(ids.to(DEV), wd, scale, pad)
    dw, = torch.autograd.grad(y, wd, g.to(DEV))
    ref = w[ids].double() * scale
    assert y.shape == ref.shape and ((y.detach().cpu().double() - ref).abs() <= (u + W) * ref.abs() + (6e-8 if dtype == torch.float16 else 0)).all()
    flat, gf = ids.reshape(-1).long(), g.reshape(-1, D).double().clone()
    if pad is not None:
        gf[flat == pad] = 0
    d = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat, gf) * scale
    a = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat, gf.abs()) * abs(scale)
    n = torch.bincount(flat, minlength=V)[:, None].double()
    bar = n * W * a + (u + 2 * W) * d.abs() + (6e-8 if dtype == torch.float16 else 0)
    dw = dw.cpu().double()
    assert ((dw - d).abs() <= bar).all(), float(((dw - d).abs() / (bar + 1e-300)).max())
    assert not dw[n[:, 0] == 0].any()
    return y, dw


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 5, 8), (7, 3, 5), (31, 100, 64), (33, 2, 65), (64, 70, 1), (257, 511, 7), (2048, 300, 33), (2049, 512, 12), (3000, 513, 260), (5000, 70000, 40),
                                   (70001, 9, 16), (20000, 40, 300)])
def test_over_sizes(kind, T, V, D):
    gen = torch.Generator().manual_seed(T + V)
    check_one(torch.randint(0, V, (T,), generator=gen), V, D, TYPES[kind], 0.5 if T % 2 else 1.0, [None, 0, V - 1][T % 3], T)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T", [40, 2000, 5000])
@pytest.mark.parametrize("what", ["one row", "two rows", "ends of chunks", "sorted", "reversed", "last row"])
def test_runs(kind, T, what):
    V, D = 37, 20
    at = torch.arange(T)
    ids = {"one row": torch.full((T,), 17), "two rows": at % 2, "ends of chunks": torch.clamp(at // 32, max=V - 1), "sorted": (at * V) // T, "reversed": V - 1 - (at * V) // T,
           "last row": torch.full((T,), V - 1)}[what]
    check_one(ids, V, D, TYPES[kind], 2.0, None, T)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T", [40, 2000, 5000])
@pytest.mark.parametrize("what", ["one row", "two rows", "ends of chunks", "sorted", "reversed", "last row"])
@pytest.mark.parametrize("V,D", [(1500, 20), (1500, 270)])
def test_runs_in_larger_tables(kind, T, what, V, D):
    at = torch.arange(T)
    ids = {"one row": torch.full((T,), 17), "two rows": at % 2, "ends of chunks": torch.clamp(at // 32, max=V - 1), "sorted": (at * V) // T, "reversed": V - 1 - (at * V) // T,
           "last row": torch.full((T,), V - 1)}[what]
    check_one(ids, V, D, TYPES[kind], 2.0, None, T)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (9, 160, 1), (5000, 160, 1), (5000, 161, 1), (700, 80, 32), (700, 160, 32), (700, 161, 32), (9000, 160, 64), (9000, 10, 1024), (300, 5, 2048), (40, 1, 9000),
                                   (100000, 2, 3), (131072, 72, 33)])
def test_around_what_counts_as_few_rows(kind, T, V, D):
    gen = torch.Generator().manual_seed(T + V)
    check_one(torch.randint(-1, V + 1, (T,), generator=gen).clamp_(0, V - 1), V, D, TYPES[kind], 0.5, V // 2 if V > 2 else None, T)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("T,V,D", [(3000, 70001, 520), (3000, 9000, 4100), (5000, 4200000, 4)])
def test_large_tables(kind, T, V, D):
    gen = torch.Generator().manual_seed(T)
    check_one(torch.randint(0, V // 3, (T,), generator=gen) * 3, V, D, TYPES[kind], 2.0, 0, T)


def test_shapes_types_of_ids_and_repeatability():
    from gshell_amd import nn
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 50, (4, 9, 11), generator=gen)
    y, d = check_one(ids, 50, 24, torch.bfloat16, 3.0, 4)
    y2, d2 = check_one(ids.int(), 50, 24, torch.bfloat16, 3.0, 4)
    assert torch.equal(y, y2) and torch.equal(d, d2)
    y3, d3 = check_one(ids.transpose(0, 2).contiguous().transpose(0, 2), 50, 24, torch.bfloat16, 3.0, 4)
    assert torch.equal(y, y3) and torch.equal(d, d3)
    big = torch.randn(50, 60, device=DEV)
    view = big[:, 3:40]
    assert torch.equal(nn.embedding(ids.to(DEV), view), view[ids.to(DEV)])
    assert torch.equal(nn.embedding(ids.to(DEV), big.t()), big.t()[ids.to(DEV).clamp(max=49)])
    assert nn.embedding(torch.tensor(7, device=DEV), big).shape == (60,)
    # an expanded gradient
    w = big.clone().requires_grad_(True)
    nn.embedding(ids.to(DEV), w).sum().backward()
    assert torch.equal(w.grad[:, 0].cpu(), torch.bincount(ids.reshape(-1), minlength=50).float())


@pytest.mark.parametrize("T", [100, 5000])
def test_ids_outside_of_the_table_read_nothing(T):
    from gshell_amd import nn
    V, D = 20, 8
    ids = torch.arange(T) % V
    bad = torch.zeros(T, dtype=torch.bool)
    for at, v in ((0, -1), (3, V), (T - 1, 2 ** 62), (T // 2, -2 ** 63)):
        ids[at], bad[at] = v, True
    w = torch.randn(V, D).to(DEV).requires_grad_(True)
    y = nn.embedding(ids.to(DEV), w)
    dw, = torch.autograd.grad(y, w, torch.ones(T, D, device=DEV))
    y = y.detach().cpu()
    assert y[bad].isnan().all() and torch.equal(y[~bad], w.detach().cpu()[ids[~bad]])
    assert torch.equal(dw[:, 0].cpu(), torch.bincount(ids[~bad], minlength=V).float())


def test_empty_sizes():
    from gshell_amd import nn
    for T, V, D in ((0, 5, 4), (3, 5, 0), (0, 0, 4), (0, 5, 0)):
        w = torch.randn(V, D, device=DEV, requires_grad=True)
        y = nn.embedding(torch.zeros(T, dtype=torch.int64, device=DEV), w)
        assert y.shape == (T, D)
        dw, = torch.autograd.grad(y, w, torch.ones_like(y))
        assert dw.shape == (V, D) and not dw.any()


def test_padding_row_keeps_its_value_and_nan_stays_in_its_row():
    from gshell_amd import nn
    w = torch.randn(6, 16)
    w[2] = float("nan")
    wd = w.to(DEV).requires_grad_(True)
    ids = torch.tensor([0, 2, 5, 0, 5], device=DEV)
    g = torch.randn(5, 16)
    g[2, 3] = float("inf")
    y = nn.embedding(ids, wd, padding_idx=0)
    dw, = torch.autograd.grad(y, wd, g.to(DEV))
    assert torch.equal(y[0].detach().cpu(), w[0]) and y[1].isnan().all()
    dw = dw.cpu()
    assert not dw[0].any() and torch.equal(dw[2], g[1]) and dw[5, 3] == float("inf") and torch.isfinite(dw[5, [0, 1, 2, 4, 5]]).all()


@pytest.mark.parametrize("T", [500, 6000])
def test_a_captured_step_replays(T):
    from gshell_amd import nn
    ids = torch.randint(0, 90, (T,), device=DEV)
    w = torch.randn(90, 48, device=DEV).to(torch.float16).requires_grad_(True)
    g = torch.randn(T, 48, device=DEV).to(torch.float16)

    def step():
        y = nn.embedding(ids, w, 0.5, 3)
        return [y.detach(), torch.autograd.grad(y, w, g)[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        ids.copy_(torch.randint(0, 90, (T,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in out]
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_module():
    from gshell_amd import nn
    m = nn.Embedding(30, 12, padding_idx=1, scale=4.0).to(DEV)
    assert set(m.state_dict()) == {"weight"} and not m.weight[1].any()
    ids = torch.tensor([[1, 2], [29, 2]], device=DEV)
    y = m(ids)
    assert torch.equal(y, m.weight[ids] * 4.0)
    y.sum().backward()
    assert float(m.weight.grad[2, 0]) == 8.0 and not m.weight.grad[1].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [300, 520, 24])
@pytest.mark.parametrize("seed", range(4))
def test_runs_of_lengths_around_a_chunk(kind, D, seed):
    """Sorted, the tokens lie in runs of lengths around the 32 of a chunk and its multiples, at every offset to the chunks' borders; the padding row is one of the long ones."""
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.tensor([1, 2, 3, 30, 31, 32, 33, 34, 63, 64, 65, 95, 96, 97, 200])[torch.randint(0, 15, (60 if seed else 30,), generator=gen)]
    if seed == 2:
        lengths[0] = 32
    if seed == 3:
        lengths = torch.cat([lengths, torch.tensor([700])])
    V = len(lengths) * 2 + 1
    ids = torch.repeat_interleave(torch.arange(len(lengths)) * 2 + (seed & 1), lengths)
    ids = ids[torch.randperm(len(ids), generator=gen)]
    check_one(ids, V, D, TYPES[kind], 1.0, int(ids[0]) if seed == 3 else None, seed)
