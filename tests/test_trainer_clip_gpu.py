"""Trainer.step clips whatever torch's clipping takes: fp32 gradients on the GPU by the framework's kernels, other lists by torch."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.timeout(120)
@pytest.mark.parametrize("extra", ["float64", "cpu", "float16"])
def test_parameters_of_other_kinds_beside_the_reconstructions(extra):
    from gshell_amd import workload
    tr = workload.build(res=16, n_samples=2, batch=1, train_res=(64, 64), fit_steps=60)
    target = workload.make_targets(tr, [0], (64, 64))
    tr.it = 1000
    tr.FLAGS.clip_max_norm = 1e-3
    p = torch.nn.Parameter(torch.ones(7, dtype={"float64": torch.float64, "float16": torch.float16}.get(extra, torch.float32), device="cpu" if extra == "cpu" else DEV))
    p.grad = torch.full_like(p, 0.25)
    tr.mat_params.append(p)          # clipped with the others, stepped by whoever added it
    tr.step(target)
    assert 0 < float(p.grad.abs().max()) < 0.25
    total = torch.stack([q.grad.double().norm().cpu() for q in list(tr.geometry.parameters()) + list(tr.mat_params) if q.grad is not None]).norm()
    assert abs(float(total) - 1e-3) <= 2e-5
