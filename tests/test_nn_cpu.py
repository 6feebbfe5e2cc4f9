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
    assert L.gs_linear_fwd_workspace_bytes(p, i(8), p, i(8), i(-1), i(1), i(1), c_int(0)) == -1
    assert L.gs_linear_bwd_workspace_bytes(p, i(8), c_int(0), p, i(8), p, i(8), i(1), i(1), i(1), c_int(9), c_int(1), c_int(1), c_int(1)) == -1


def test_embedding_refuses():
    w, ids = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    for a, b, kw, what in ((ids, w[0], {}, "weight"), (ids, w.double(), {}, "weight"), (ids.float(), w, {}, "ids"), (ids.to(torch.int16), w, {}, "ids"),
                           (ids, w, dict(padding_idx=5), "padding_idx"), (ids, w, dict(padding_idx=-1), "padding_idx"), (ids, w, {}, "HBM")):
        with pytest.raises(GShellHipError, match=what):
            nn.embedding(a, b, **kw)
    assert set(nn.Embedding(5, 4).state_dict()) == {"weight"}


def test_embedding_c_entry_refuses_bad_arguments():
    from gshell_amd import _lib
    from gshell_amd._lib import c_float, c_int, c_int64, c_void_p
    L, i, n, p = _lib.lib(), c_int64, c_void_p(0), c_void_p(256)
    for T, V, D, dtype, ids in ((-1, 4, 4, 0, p), (4, 1 << 31, 4, 0, p), (4, 4, -1, 0, p), (4, 4, 4, 3, p), (4, 4, 4, 0, n)):
        assert L.gs_embedding_fwd(ids, c_int(1), p, i(4), i(T), i(V), i(D), c_int(dtype), c_float(1), p, n) != 0
        assert L.gs_embedding_bwd(ids, c_int(1), p, i(4), i(T), i(V), i(D), i(-1), c_int(dtype), c_float(1), p, p, i(1 << 40), n) != 0
    assert L.gs_embedding_bwd(p, c_int(1), p, i(4), i(4), i(4), i(4), i(-1), c_int(0), c_float(1), p, p, i(16), n) != 0 and b"workspace" in L.gs_last_error()
    assert L.gs_embedding_bwd_workspace_bytes(i(-1), i(4), i(4)) == -1
    assert L.gs_embedding_fwd(n, c_int(1), n, i(4), i(0), i(4), i(4), c_int(0), c_float(1), n, n) == 0


def test_clip_refuses():
    from gshell_amd import optim
    g = [torch.zeros(4), torch.zeros(5)]
    for kw, what in ((dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"), (dict(max_norm=1.0, norm_type=3.0), "norm_type"),
                     (dict(max_norm=1.0, out=[g[0]]), "outputs"), (dict(max_norm=1.0, out=[torch.zeros(4), torch.zeros(6)]), "output"),
                     (dict(max_norm=1.0, out=[torch.zeros(4), torch.zeros(5).half()]), "output"), (dict(max_norm=1.0), "HBM")):
        with pytest.raises(GShellHipError, match=what):
            optim.clip_grads(g, **kw)
    with pytest.raises(GShellHipError, match="float32"):
        optim.grad_norm([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(GShellHipError, match="float32"):
        optim.grad_norm([torch.zeros(4, 4).to_sparse()])
    assert float(optim.clip_grads([], 1.0)) == 0.0 and float(optim.grad_norm([])) == 0.0


@pytest.mark.parametrize("written,read,fine", [
    ([(0, 50), (49, 51)], None, False), ([(0, 9), (0, 9)], None, False), ([(10, 10), (0, 11)], None, False), ([(0, 10)], [(5, 10)], False),
    ([(0, 10), (50, 10)], [(0, 10), (55, 10)], False), ([(50, 10), (0, 10)], [(50, 10), (45, 10)], False), ([(0, 100)], [(99, 100)], False),
    ([(0, 50), (50, 50)], None, True), ([(0, 50), (20, 0), (50, 50)], None, True), ([(0, 10)], [(10, 10)], True), ([(10, 10)], [(0, 10)], True),
    ([(0, 10), (50, 10)], [(0, 10), (60, 10)], True), ([(5, 0)], [(5, 0)], True), ([(5, 0), (0, 20)], [(3, 0), (0, 20)], True),
])
def test_clip_refuses_shared_memory(written, read, fine):
    """(address, elements of 4 bytes) of the outputs and of the gradients: the C entry's check on the host.  A list that passes is stopped by its workspace's size."""
    import ctypes
    from gshell_amd import _lib
    L, n = _lib.lib(), len(written)
    base = 1 << 20
    at = lambda v: (ctypes.c_void_p * n)(*[base + 4 * a for a, _ in v])      # noqa: E731
    call = lambda ws: L.gs_grad_norm(n, at(read or written), at(written), (ctypes.c_int64 * n)(*[z for _, z in written]), (ctypes.c_int32 * n)(), 0, 1.0, 256, 256, ws, 0)      # noqa: E731
    if fine:
        assert call(0) != 0 and b"workspace" in L.gs_last_error()
    else:
        assert call(1 << 30) != 0 and b"shares memory" in L.gs_last_error()


def test_clip_c_entry_refuses_bad_arguments():
    import ctypes
    from gshell_amd import _lib
    from gshell_amd._lib import c_float, c_int, c_int64, c_void_p
    L, n, p = _lib.lib(), c_void_p(0), c_void_p(256)

    def call(ptr=256, numel=4, dtype=0, kind=0, max_norm=1.0, norm=p, ws=1 << 20, out=256):
        return L.gs_grad_norm(c_int(1), (ctypes.c_void_p * 1)(ptr), (ctypes.c_void_p * 1)(out), (ctypes.c_int64 * 1)(numel), (ctypes.c_int32 * 1)(dtype), c_int(kind),
                              c_float(max_norm), norm, p, c_int64(ws), n)
    for kw in (dict(ptr=None), dict(out=None), dict(numel=-1), dict(dtype=3), dict(dtype=-1), dict(kind=3), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(norm=n), dict(ws=8)):
        assert call(**kw) != 0 and b"gs_grad_norm" in L.gs_last_error(), kw
    assert L.gs_grad_norm_workspace_bytes(c_int(-1)) == -1


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_linear_workspace_sizes(dtype):
    """The plan of a call is made on the host: sizes from nothing to the largest, none negative, and for ordinary layers no more than a few times their operands."""
    from gshell_amd import _lib
    L = _lib.lib()
    es = 4 if dtype == 0 else 2
    for M in (0, 1, 2, 31, 32, 33, 64, 1000, 4096, 131072, (1 << 31) - 1):
        for N in (0, 1, 7, 8, 64, 1000, 4096, 65536):
            for K in (0, 1, 8, 295, 777, 4096, 65536):
                for ld, at in ((K, 0), (K + 3, 2)):
                    fwd = L.gs_linear_fwd_workspace_bytes(1024 + at, ld, 2048, K, M, N, K, dtype)
                    bwd = L.gs_linear_bwd_workspace_bytes(4096, N, 1, 1024 + at, ld, 2048, K, M, N, K, dtype, 1, 1, 1)
                    assert fwd >= 0 and bwd >= 0, (M, N, K)
                    if max(M, N, K) < 5000:
                        assert fwd <= 8 * es * (M * K + N * K + M * N) + (64 << 20) and bwd <= 8 * es * (M * K + N * K + M * N) + (160 << 20), (M, N, K, fwd, bwd)


def test_linear_backward_c_entry_refuses_bad_arguments():
    from gshell_amd import _lib
    L, p = _lib.lib(), 256

    def bwd(g=p, ldg=4, x=p, ldx=4, w=p, ldw=4, M=4, N=4, K=4, dtype=0, dx=p, dw=p, db=p, ws=p, ws_bytes=1 << 30):
        return L.gs_linear_bwd(g, ldg, 0, x, ldx, w, ldw, M, N, K, dtype, dx, dw, db, ws, ws_bytes, 0)
    for kw in (dict(g=0), dict(ldg=-1), dict(x=0), dict(ldx=-4), dict(w=0), dict(ldw=-4), dict(M=-1), dict(K=1 << 31), dict(dtype=1, N=1 << 21), dict(dtype=3), dict(ws_bytes=0, dtype=1), dict(ws=257)):
        assert bwd(**kw) != 0 and b"gs_linear_bwd" in L.gs_last_error(), kw


def test_modules_say_what_they_are_and_a_table_can_be_given():
    rows = torch.arange(12.0).view(3, 4)
    table = nn.Embedding.from_pretrained(rows, padding_idx=-1, scale=0.5)
    assert table.weight.data_ptr() == rows.data_ptr() and not table.weight.requires_grad and table.padding_idx == 2 and table.scale == 0.5 and torch.equal(rows, torch.arange(12.0).view(3, 4))
    assert nn.Embedding.from_pretrained(rows, freeze=False).weight.requires_grad and "scale=0.5" in repr(table) and "activation=gelu" in repr(nn.Linear(2, 3, activation="gelu"))
    with pytest.raises(GShellHipError, match="rows"):
        nn.Embedding.from_pretrained(rows[0])
