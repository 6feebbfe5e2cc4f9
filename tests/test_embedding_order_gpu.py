"""The order in which nn.embedding's gradient is summed goes by the sizes and the ids alone, not by where the gradient lies."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [130, 240, 256, 258, 384, 480, 512, 516, 600, 1024])          # bytes of a row
def test_a_gradient_that_is_a_view_gives_the_same_bits(dtype, size):
    from gshell_amd import nn
    es = torch.tensor([], dtype=dtype).element_size()
    D, V, T = size // es, 3000, 6000
    gen = torch.Generator().manual_seed(size)
    ids = (torch.rand(T, generator=gen) ** 3 * V).long().clamp(max=V - 1)          # runs of many lengths, across borders of every kind
    ids[:700] = 5
    ids[700:760] = 11
    ids, weight = ids.to(DEV), torch.zeros(V, D, dtype=dtype, device=DEV, requires_grad=True)
    g = torch.randn(T, D, generator=gen).to(dtype).to(DEV)

    def gradient(g):
        return torch.autograd.grad(nn.embedding(ids, weight), weight, g)[0]
    first = gradient(g)
    assert torch.equal(first, gradient(g))
    for before, behind in ((1, 0), (2, 1), (4, 4), (8, 0), (3, 8)):
        big = torch.randn(T, before + D + behind, generator=gen).to(dtype).to(DEV)
        big[:, before:before + D] = g
        view = big[:, before:before + D]
        assert not view.is_contiguous() and torch.equal(first, gradient(view)), (before, behind)
    flat = torch.empty(T * D + 1, dtype=dtype, device=DEV)
    flat[1:] = g.reshape(-1)
    assert torch.equal(first, gradient(flat[1:].view(T, D)))
