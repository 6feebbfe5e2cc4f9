"""What gshell_amd.nn refuses, before anything reaches a GPU."""
import pytest
import torch

from gshell_amd import nn
from gshell_amd._lib import GShellHipError


def _ops(dtype=torch.float32):
    return torch.zeros(4, 8, dtype=dtype), torch.zeros(6, 8, dtype=dtype)


@pytest.mark.parametrize("kw,what", [
    (dict(activation="tanh"), "activation"),
    (dict(activation="softplus", beta=0.0), "beta"),
    (dict(activation="softplus", beta=float("nan")), "beta"),
    (dict(activation="softplus", beta=float("inf")), "beta"),
    (dict(bias=torch.zeros(5)), "bias"),
    (dict(bias=torch.zeros(6, 1)), "bias"),
    (dict(bias=torch.zeros(6, dtype=torch.float16)), "bias"),
    (dict(residual=torch.zeros(6)), "residual"),
    (dict(residual=torch.zeros(4, 6, dtype=torch.bfloat16)), "residual"),
    (dict(), "HBM"),
])
def test_linear_refuses(kw, what):
    with pytest.raises(GShellHipError, match=what):
        nn.linear(*_ops(), **kw)


def test_linear_refuses_operands():
    x, w = _ops()
    for a, b in ((x, w[:, :7]), (x, w[0]), (torch.zeros(()), w), (x.double(), w.double()), (x.long(), w.long()), (x, w.half())):
        with pytest.raises(GShellHipError):
            nn.linear(a, b)


def test_linear_module_has_torchs_parameters():
    lin = nn.Linear(8, 6, activation="gelu")
    assert set(lin.state_dict()) == set(torch.nn.Linear(8, 6).state_dict())
    with pytest.raises(GShellHipError):
        nn.Linear(8, 6, activation="tanh")
    with pytest.raises(GShellHipError, match="HBM"):
        lin(torch.zeros(3, 8))


def test_linear_c_entry_refuses_bad_arguments():
    """Host-side checks of the C entry points: no device call is reached."""
    from gshell_amd import _lib
    from gshell_amd._lib import c_float, c_int, c_int64, c_void_p
    L = _lib.lib()
    n, p = c_void_p(0), c_void_p(256)
    i = c_int64

    def fwd(M=4, N=4, K=4, dtype=0, act=0, beta=1.0, x=p, y=p, ldy=4):
        return L.gs_linear_fwd(x, i(4), p, i(4), n, n, i(0), i(M), i(N), i(K), c_int(dtype), c_int(act), c_float(beta), y, i(ldy), n, n, i(0), n)
    for kw in (dict(M=-1), dict(N=1 << 31), dict(dtype=3), dict(act=5), dict(act=2, beta=0.0), dict(x=n), dict(y=n), dict(ldy=3), dict(M=1, N=1, K=100000)):
        assert fwd(**kw) != 0 and b"gs_linear" in L.gs_last_error(), kw
    assert fwd(M=0) == 0
    assert L.gs_linear_fwd_workspace_bytes(i(-1), i(1), i(1), c_int(0)) == -1
    assert L.gs_linear_bwd_workspace_bytes(i(1), i(1), i(1), c_int(9), c_int(0), c_int(1), c_int(1), c_int(1)) == -1
