"""Gradients of some of nn.linear's operands alone (a frozen weight, a frozen input): the same products, and so the same bits, as in the whole backward pass; db's sum
has the order of the launch that takes it along."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("M,N,K", [(20, 40, 24), (1000, 520, 300), (777, 129, 1031), (4096, 256, 264)])
def test_gradients_of_some_operands(M, N, K, act, dtype):
    from gshell_amd import nn
    gen = torch.Generator().manual_seed(M)
    x, w, b, r, g = (torch.randn(*s, generator=gen).to(dtype).to(DEV) for s in ((M, K), (N, K), (N,), (M, N), (M, N)))
    w = w / 16

    def grads(wanted):
        leaf = [t.clone().requires_grad_(k in wanted) for k, t in enumerate((x, w, b, r))]
        y = nn.linear(*leaf, activation=act)
        return dict(zip(wanted, torch.autograd.grad(y, [leaf[k] for k in wanted], g)))
    whole = grads((0, 1, 2, 3))
    for n in (1, 2, 3):
        for wanted in itertools.combinations(range(4), n):
            for k, t in grads(wanted).items():
                if k == 2:          # db is summed with dW, beside a product or by itself, in three orders: each is off by (M + 16) 2^-24 sum |gz|, then rounded once
                    gz = g.double().abs().sum(0) * 1.13
                    rounded = 0 if dtype == torch.float32 else torch.finfo(dtype).eps * (1 + 2.0 ** -10)
                    assert ((t - whole[k]).double().abs() <= 2 * (M + 16) * 2.0 ** -24 * gz * 1.01 + rounded * whole[k].double().abs()).all()
                else:
                    assert torch.equal(t, whole[k]), (wanted, k)
