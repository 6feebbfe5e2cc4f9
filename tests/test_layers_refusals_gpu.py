"""Calls of gshell_amd.nn and gshell_amd.optim with tensors that are not what they look like: refused before anything is written, or taken for what is in them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_clip_refuses_outputs_whose_elements_share_a_place_before_it_writes():
    from gshell_amd import optim
    from gshell_amd._lib import GShellHipError
    one = torch.full((4, 3), 2.0, device=DEV)
    row = torch.ones(5, device=DEV).expand(4, 5)
    for grads, out in (([one, row], None), ([one, row.contiguous()], [torch.zeros_like(one), row])):
        version = one._version
        with pytest.raises(GShellHipError, match="share"):
            optim.clip_grads(grads, 0.5, out=out)
        assert (one == 2).all() and one._version == version and (out is None or not out[0].any())
    got = [torch.zeros_like(one), torch.zeros(4, 5, device=DEV)]          # a gradient may be such a view
    norm = optim.clip_grads([one, row], 1.0, out=got)
    assert abs(float(norm) - 68 ** 0.5) < 1e-5 and torch.allclose(got[1], row / 68 ** 0.5, rtol=1e-5)


def test_tensors_that_outlived_a_transform():
    """What a function under torch.func.grad kept of its argument is an ordinary tensor again once that is over."""
    from gshell_amd import nn
    kept = []

    def f(t):
        kept.append(t)
        return (t * t).sum()
    x, w = torch.randn(5, 8, device=DEV), torch.randn(4, 8, device=DEV)
    torch.func.grad(f)(x)
    torch.func.grad(f)(w)
    assert torch.equal(nn.linear(kept[0], kept[1], activation="relu"), nn.linear(x, w, activation="relu"))
    leaf = w.clone().requires_grad_(True)
    y = nn.linear(kept[0], leaf, activation="relu")
    other = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0], torch.autograd.grad(nn.linear(x, other, activation="relu").sum(), other)[0])
    ids = torch.tensor([3, 0, 3], device=DEV)
    assert torch.equal(nn.embedding(ids, kept[1]), w[ids])
