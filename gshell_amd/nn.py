"""Layers for networks that the fused SDF network (geometry/mlp.py) and the hash table (render/mlptexture.py) do not cover, on hand-written HIP kernels:

  linear(x, weight, bias, residual, activation)   y = act(x W^T + b) + r with its backward pass   (csrc/linear.hip)
  Linear                                          torch.nn.Linear with that epilogue; same parameter names, same initialisation
  embedding(ids, weight, scale, padding_idx)      y_t = scale W[id_t], gradient by sorted ids             (csrc/embedding.hip)
  Embedding                                       torch.nn.Embedding's parameters and initialisation, with the scale

bf16, fp16 and fp32; every sum is 32-bit; a call's sums are taken in a fixed order, so the same inputs give the same bits.  All operands live in HBM: there is no CPU
fallback.  A call launches on the current stream of its operands' device and keeps nothing between calls.  Gradients can be taken once
(a second differentiation raises).  Under torch.autocast the operators run in their operands' own type.

A backward pass that is captured into a graph must be the only live graph of its leaves: drop the outputs of eager passes over the same parameters first."""
import torch

from . import _lib
from ._lib import GShellHipError, c_float, c_int, c_int64, c_void_p, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "softplus": 2, "silu": 3, "gelu": 4}


def _p(t):
    return c_void_p(0 if t is None else t.data_ptr())


class _on:
    """The operands' device as the current one, without the context manager's cost where it is already."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return c_void_p(torch.cuda.current_stream(self.index).cuda_stream)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)
        return False


def _rows(t):
    """`t` [rows, n] with contiguous rows, and the stride between them (a copy only where a row's elements are apart)."""
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t, t.stride(0)


def _workspace(nbytes, device):
    if nbytes < 0:
        raise GShellHipError("linear: sizes are 0 .. 2^31 - 1")
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear_forward(x, weight, bias, residual, act, beta, want_dact):
    M, K = x.shape
    N = weight.shape[0]
    x, ldx = _rows(x)
    w, ldw = _rows(weight)
    b = None if bias is None else bias.contiguous()
    r, ldr = (None, 0) if residual is None else _rows(residual)
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    dact = torch.empty((M, N), dtype=torch.float16 if x.dtype == torch.bfloat16 else torch.float32, device=x.device) if want_dact and act else None
    L = _lib.lib()
    with _on(x.device) as stream:
        code = _DTYPES[x.dtype]
        need = L.gs_linear_fwd_workspace_bytes(_p(x), c_int64(ldx), _p(w), c_int64(ldw), c_int64(M), c_int64(N), c_int64(K), c_int(code))
        ws = _workspace(need, x.device)
        check(L.gs_linear_fwd(_p(x), c_int64(ldx), _p(w), c_int64(ldw), _p(b), _p(r), c_int64(ldr), c_int64(M), c_int64(N), c_int64(K), c_int(code), c_int(act),
                              c_float(beta), _p(y), c_int64(N), _p(dact), _p(ws), c_int64(need), stream), "gs_linear_fwd")
    return y, dact


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, beta):
        need = ctx.needs_input_grad
        y, dact = _linear_forward(x, weight, bias, residual, act, beta, need[0] or need[1] or need[2])
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, dact)
        ctx.sizes = (x.shape[0], weight.shape[0], x.shape[1])
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight, dact = ctx.saved_tensors
        M, N, K = ctx.sizes
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_x or want_w or want_b:
            gr, ldg = _rows(g)
            x, ldx = _rows(x) if x is not None else (None, 0)
            weight, ldw = _rows(weight) if weight is not None else (None, 0)
            new = lambda *shape: torch.empty(shape, dtype=g.dtype, device=g.device)      # noqa: E731
            dx, dw, db = new(M, K) if want_x else None, new(N, K) if want_w else None, new(N) if want_b else None
            L = _lib.lib()
            with _on(g.device) as stream:
                code = _DTYPES[g.dtype]
                need = L.gs_linear_bwd_workspace_bytes(_p(gr), c_int64(ldg), c_int(dact is not None), _p(x), c_int64(ldx), _p(weight), c_int64(ldw), c_int64(M), c_int64(N), c_int64(K),
                                                       c_int(code), c_int(want_x), c_int(want_w), c_int(want_b))
                ws = _workspace(need, g.device)
                check(L.gs_linear_bwd(_p(gr), c_int64(ldg), _p(dact), _p(x), c_int64(ldx), _p(weight), c_int64(ldw), c_int64(M), c_int64(N), c_int64(K), c_int(code),
                                      _p(dx), _p(dw), _p(db), _p(ws), c_int64(need), stream), "gs_linear_bwd")
        return dx, dw, db, g if want_r else None, None, None


def linear(x, weight, bias=None, residual=None, activation=None, beta=1.0):
    """act(x W^T + b) + r: x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    activation: None, "relu", "softplus" (log(1 + exp(beta z)) / beta), "silu" or "gelu" (erf form).  The residual is added behind the activation and has the
    output's shape (an expanded view may stand for it).  All operands have one type (float32, bfloat16, float16) and one device; x, weight and residual may be views whose rows are
    any stride apart.  fp32 operands keep fp32's accuracy.  Where the gradient is taken of an activation, act'(z) is kept for the backward pass: 2 bytes an output
    for bf16, 4 for the others."""
    if activation not in ACTIVATIONS:
        raise GShellHipError(f"linear: activation {activation!r} is not one of {sorted(k for k in ACTIVATIONS if k)} or None")
    act = ACTIVATIONS[activation]
    beta = float(beta)
    if act == 2 and not 0.0 < beta < 1e30:
        raise GShellHipError(f"linear: softplus needs a positive finite beta, got {beta}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise GShellHipError(f"linear: x [..., K] and weight [N, K] are wanted, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    shape = x.shape[:-1] + (N,)
    if bias is not None and bias.shape != (N,):
        raise GShellHipError(f"linear: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != shape:
        raise GShellHipError(f"linear: residual must have the output's shape {tuple(shape)}, got {tuple(residual.shape)}")
    if x.dtype not in _DTYPES:
        raise GShellHipError(f"linear: float32, bfloat16 or float16 operands are wanted, got {x.dtype}")
    operands = (("x", x), ("weight", weight), ("bias", bias), ("residual", residual))
    for name, t in operands:
        if t is not None and t.dtype != x.dtype:
            raise GShellHipError(f"linear: {name} is {t.dtype}, x is {x.dtype}")
    for name, t in operands:
        if t is None:
            continue
        if not t.is_cuda:
            raise GShellHipError(f"linear: {name} must live in HBM (got device {t.device}); the HIP path has no CPU fallback")
        if t.device != x.device:
            raise GShellHipError(f"linear: {name} is on {t.device}, x on {x.device}")
    x2 = x if x.dim() == 2 else x.reshape(-1, K) if K else x.reshape(x.shape[:-1].numel(), 0)
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(x2.shape[0], N)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for _, t in operands):
        y = _LinearFn.apply(x2, weight, bias, r2, act, beta)
    else:
        y, _ = _linear_forward(x2, weight, bias, r2, act, beta, False)
    return y if x.dim() == 2 else y.reshape(shape)


class Linear(torch.nn.Linear):
    """torch.nn.Linear (same parameters, initialisation and state_dict) with an activation, and a residual that a call may hand over."""

    def __init__(self, in_features, out_features, bias=True, activation=None, beta=1.0, device=None, dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        if activation not in ACTIVATIONS:
            raise GShellHipError(f"Linear: activation {activation!r} is not one of {sorted(k for k in ACTIVATIONS if k)} or None")
        self.activation, self.beta = activation, beta

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual, self.activation, self.beta)

    def extra_repr(self):
        return super().extra_repr() + f", activation={self.activation}"


_ID_TYPES = {torch.int64: 1, torch.int32: 0}


def _lookup(ids, weight, scale):
    w, ldw = _rows(weight)
    V, D = w.shape
    y = torch.empty((ids.numel(), D), dtype=w.dtype, device=w.device)
    with _on(w.device) as stream:
        check(_lib.lib().gs_embedding_fwd(_p(ids), c_int(_ID_TYPES[ids.dtype]), _p(w), c_int64(ldw), c_int64(ids.numel()), c_int64(V), c_int64(D), c_int(_DTYPES[w.dtype]),
                                          c_float(scale), _p(y), stream), "gs_embedding_fwd")
    return y


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rest = (weight.shape, scale, padding_idx)
        return _lookup(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        (V, D), scale, padding_idx = ctx.rest
        g, ldg = _rows(g)
        T = ids.numel()
        dw = torch.empty((V, D), dtype=g.dtype, device=g.device)
        L = _lib.lib()
        with _on(g.device) as stream:
            need = L.gs_embedding_bwd_workspace_bytes(c_int64(T), c_int64(V), c_int64(D))
            ws = _workspace(need, g.device)
            check(L.gs_embedding_bwd(_p(ids), c_int(_ID_TYPES[ids.dtype]), _p(g), c_int64(ldg), c_int64(T), c_int64(V), c_int64(D), c_int64(padding_idx), c_int(_DTYPES[g.dtype]),
                                     c_float(scale), _p(dw), _p(ws), c_int64(need), stream), "gs_embedding_bwd")
        return None, dw, None, None


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids]: ids int64 or int32 of any shape, weight [V, D] (float32, bfloat16, float16) -> ids.shape + [D].

    The gradient sums a row's tokens in their order in 32 bits: the same bits every time.  The row `padding_idx` gets none.  Ids are not looked at on the host: one outside
    of [0, V) gives a row of NaN and has no gradient (negative ids do not count from the end)."""
    if weight.dim() != 2 or weight.dtype not in _DTYPES:
        raise GShellHipError(f"embedding: a weight [V, D] of float32, bfloat16 or float16 is wanted, got {tuple(weight.shape)} {weight.dtype}")
    if ids.dtype not in _ID_TYPES:
        raise GShellHipError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    if max(ids.numel(), *weight.shape) >= (1 << 31) - 1:
        raise GShellHipError("embedding: sizes are 0 .. 2^31 - 2")
    if padding_idx is None:
        padding_idx = -1
    elif not 0 <= padding_idx < weight.shape[0]:
        raise GShellHipError(f"embedding: padding_idx {padding_idx} is not a row of the table of {weight.shape[0]}")
    scale = float(scale)
    for name, t in (("ids", ids), ("weight", weight)):
        if not t.is_cuda:
            raise GShellHipError(f"embedding: {name} must live in HBM (got device {t.device}); the HIP path has no CPU fallback")
    if ids.device != weight.device:
        raise GShellHipError(f"embedding: ids are on {ids.device}, the weight on {weight.device}")
    flat = ids.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        y = _EmbeddingFn.apply(flat, weight, scale, int(padding_idx))
    else:
        y = _lookup(flat, weight, scale)
    return y if ids.dim() == 1 else y.view(ids.shape + (weight.shape[1],))


class Embedding(torch.nn.Embedding):
    """torch.nn.Embedding (same parameter, initialisation and state_dict) whose rows come out scaled."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)
