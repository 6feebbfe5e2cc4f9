"""Layers for networks that the fused SDF network (geometry/mlp.py) and the hash table (render/mlptexture.py) do not cover, on hand-written HIP kernels:

  linear(x, weight, bias, residual, activation)   y = act(x W^T + b) + r with its backward pass   (csrc/linear.hip)
  Linear                                          torch.nn.Linear with that epilogue; same parameter names, same initialisation
  embedding(ids, weight, scale, padding_idx)      y_t = scale W[id_t], gradient without atomics           (csrc/embedding.hip)
  Embedding                                       torch.nn.Embedding's parameters and initialisation, with the scale

bf16, fp16 and fp32; every sum is 32-bit; a call's sums are taken in a fixed order, so the same inputs give the same bits.  All operands live in HBM: there is no CPU
fallback.  A call launches on the current stream of its operands' device and keeps nothing between calls.  Gradients can be taken once
(a second differentiation, forward-mode differentiation and torch.func's transforms raise).  Under torch.autocast the operators run in their operands' own type.

A backward pass that is captured into a graph must be the only live graph of its leaves: drop the outputs of eager passes over the same parameters first."""
import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import GShellHipError, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "softplus": 2, "silu": 3, "gelu": 4}
# The calls below are short next to what Python spends around them, and a backward pass runs in a thread of its own, where every Python object comes from another core's
# cache: plain numbers and addresses go to the C functions (_lib.PLAIN_CALLS), what a backward pass needs is worked out in the forward pass, and the current device is changed
# only where it is another one.
_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _at(t):
    return 0 if t is None else t.data_ptr()


def _within(t):
    """What a tensor that outlived a transform of torch.func holds (it has no storage of its own), any other one as it is."""
    for held in (lambda: t, lambda: t.view_as(t)):
        try:
            held().data_ptr()
            return held()
        except RuntimeError:
            pass
    return t


def _rows(t):
    """`t` [rows, n] with contiguous rows, and the stride between them (a copy only where a row's elements are apart)."""
    ld, step = t.stride()
    if step != 1 and t.shape[1] > 1:
        t = t.contiguous()
        ld = t.stride(0)
    return t, ld


def _linear_forward(x, weight, bias, residual, act, beta, want_dact):
    M, K = x.shape
    N = weight.shape[0]
    x, ldx = _rows(x)
    w, ldw = _rows(weight)
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    r, ldr = (None, 0) if residual is None else _rows(residual)
    y = x.new_empty((M, N))
    code = _DTYPES[x.dtype]
    dact = x.new_empty((M, N), dtype=torch.float16 if code == 1 else torch.float32) if want_dact and act else None
    L = _lib.lib()
    xp, wp = x.data_ptr(), w.data_ptr()
    need = L.gs_linear_fwd_workspace_bytes(xp, ldx, wp, ldw, M, N, K, code)
    if need < 0:
        raise GShellHipError("linear: sizes are 0 .. 2^31 - 1, of 16-bit rows (in and out) 0 .. 2^21 - 1")
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    device = x.get_device()
    args = (xp, ldx, wp, ldw, _at(b), _at(r), ldr, M, N, K, code, act, beta, y.data_ptr(), N, _at(dact), _at(ws), need, _stream_of(device))
    if _current_device() == device:
        rc = L.gs_linear_fwd(*args)
    else:
        with torch.cuda.device(device):
            rc = L.gs_linear_fwd(*args)
    if rc:
        check(rc, "gs_linear_fwd")
    return y, dact


_once_differentiable = torch.autograd.function.once_differentiable
# Function.apply without what it does for torch.func's transforms, which these layers do not take part in: where one is active the usual apply is called, and says so.
_transforms_active = torch._C._are_functorch_transforms_active


def _linear_backward(ctx, g):
    if torch.is_grad_enabled():          # create_graph: the results carry a node that says that they cannot be differentiated again
        return _once_differentiable(_linear_backward)(ctx, g)
    x, weight, dact = ctx.saved_tensors
    M, K, N, code, want_x, want_w, want_b, want_r, L = ctx.rest
    dx = dw = db = None
    if want_x or want_w or want_b:
        gr, ldg = _rows(g)
        xp = ldx = wp = ldw = xo = wo = bo = 0
        if want_w:
            x, ldx = _rows(x)
            xp = x.data_ptr()
            dw = gr.new_empty((N, K))
            wo = dw.data_ptr()
        if want_x:
            weight, ldw = _rows(weight)
            wp = weight.data_ptr()
            dx = gr.new_empty((M, K))
            xo = dx.data_ptr()
        if want_b:
            db = gr.new_empty(N)
            bo = db.data_ptr()
        gp, dp = gr.data_ptr(), _at(dact)
        need = L.gs_linear_bwd_workspace_bytes(gp, ldg, dact is not None, xp, ldx, wp, ldw, M, N, K, code, want_x, want_w, want_b)
        if need < 0:
            raise GShellHipError("linear: sizes are 0 .. 2^31 - 1, of 16-bit rows (in and out) 0 .. 2^21 - 1")
        ws = gr.new_empty(need, dtype=torch.uint8) if need else None
        device = gr.get_device()
        args = (gp, ldg, dp, xp, ldx, wp, ldw, M, N, K, code, xo, wo, bo, _at(ws), need, _stream_of(device))
        if _current_device() == device:
            rc = L.gs_linear_bwd(*args)
        else:
            with torch.cuda.device(device):
                rc = L.gs_linear_bwd(*args)
        if rc:
            check(rc, "gs_linear_bwd")
    return dx, dw, db, g if want_r else None, None, None


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, beta):
        want_x, want_w, want_b, want_r, _, _ = ctx.needs_input_grad
        y, dact = _linear_forward(x, weight, bias, residual, act, beta, want_x or want_w or want_b)
        ctx.save_for_backward(x if want_w else None, weight if want_x else None, dact)
        ctx.rest = (*x.shape, weight.shape[0], _DTYPES[x.dtype], want_x, want_w, want_b, want_r, _lib.lib())
        return y

    backward = staticmethod(_linear_backward)


_linear_apply = super(torch.autograd.Function, _LinearFn).apply


def _linear_refuse(x, weight, bias, residual, activation, beta):
    """What is wrong with a call's operands, said in full."""
    if activation not in ACTIVATIONS:
        raise GShellHipError(f"linear: activation {activation!r} is not one of {sorted(k for k in ACTIVATIONS if k)} or None")
    if activation == "softplus" and not 0.0 < beta < 1e30:
        raise GShellHipError(f"linear: softplus needs a positive finite beta, got {beta}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise GShellHipError(f"linear: x [..., K] and weight [N, K] are wanted, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None and bias.shape != (N,):
        raise GShellHipError(f"linear: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + (N,):
        raise GShellHipError(f"linear: residual must have the output's shape {tuple(x.shape[:-1]) + (N,)}, got {tuple(residual.shape)}")
    if x.dtype not in _DTYPES:
        raise GShellHipError(f"linear: float32, bfloat16 or float16 operands are wanted, got {x.dtype}")
    operands = [(n, t) for n, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)) if t is not None]
    for name, t in operands:
        if t.dtype != x.dtype:
            raise GShellHipError(f"linear: {name} is {t.dtype}, x is {x.dtype}")
    for name, t in operands:
        if not t.is_cuda:
            raise GShellHipError(f"linear: {name} must live in HBM (got device {t.device}); the HIP path has no CPU fallback")
        if t.device != x.device:
            raise GShellHipError(f"linear: {name} is on {t.device}, x on {x.device}")
    raise GShellHipError("linear: these operands are not supported")


def linear(x, weight, bias=None, residual=None, activation=None, beta=1.0):
    """act(x W^T + b) + r: x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    activation: None, "relu", "softplus" (log(1 + exp(beta z)) / beta), "silu" or "gelu" (erf form).  The residual is added behind the activation and has the
    output's shape (an expanded view may stand for it).  All operands have one type (float32, bfloat16, float16) and one device; x, weight and residual may be views whose rows are
    any stride apart.  fp32 operands of 2^-112 and above keep fp32's accuracy; fp32 outputs that meet infinities or NaN are summed a second time, which costs
    up to eleven times the product.  Where the gradient is taken of an activation, act'(z) is kept for the backward pass: 2 bytes an output
    for bf16, 4 for the others; where it is exactly zero (relu of z <= 0) nothing passes, an infinite gradient neither.  16-bit layers round
    the gradient times act' to their type before the products of dx and dW, as torch's do."""
    act = ACTIVATIONS.get(activation)
    beta = float(beta)
    dtype, device, xs, ws = x.dtype, x.get_device(), x.shape, weight.shape
    ok = act is not None and (act != 2 or 0.0 < beta < 1e30) and len(ws) == 2 and len(xs) >= 1 and xs[-1] == ws[1] and dtype in _DTYPES and x.is_cuda \
        and weight.dtype is dtype and weight.get_device() == device
    grad = ok and (x.requires_grad or weight.requires_grad)
    if ok and bias is not None:
        ok = bias.dim() == 1 and bias.shape[0] == ws[0] and bias.dtype is dtype and bias.get_device() == device
        grad = grad or bias.requires_grad
    flat = len(xs) == 2
    if ok and residual is not None:
        ok = residual.shape == xs[:-1] + ws[:1] and residual.dtype is dtype and residual.get_device() == device
        grad = grad or residual.requires_grad
    if not ok:
        _linear_refuse(x, weight, bias, residual, activation, beta)
    if not flat:
        rows = xs[:-1].numel()
        x = x.reshape(rows, ws[1])
        residual = None if residual is None else residual.reshape(rows, ws[0])
    try:
        if grad and torch.is_grad_enabled() or _forward_ad._current_level >= 0:          # (forward-mode differentiation is refused there)
            y = (_LinearFn.apply if _transforms_active() else _linear_apply)(x, weight, bias, residual, act, beta)
        else:
            y = _linear_forward(x, weight, bias, residual, act, beta, False)[0]
    except RuntimeError:
        inner = [t if t is None else _within(t) for t in (x, weight, bias, residual)]
        if _transforms_active() or all(a is b for a, b in zip(inner, (x, weight, bias, residual))):
            raise
        y = linear(*inner, activation, beta)
    return y if flat else y.reshape(xs[:-1] + ws[:1])


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
    T = ids.numel()
    y = w.new_empty((T, D))
    device = w.get_device()
    args = (ids.data_ptr(), _ID_TYPES[ids.dtype], w.data_ptr(), ldw, T, V, D, _DTYPES[w.dtype], scale, y.data_ptr(), _stream_of(device))
    if _current_device() == device:
        rc = _lib.lib().gs_embedding_fwd(*args)
    else:
        with torch.cuda.device(device):
            rc = _lib.lib().gs_embedding_fwd(*args)
    if rc:
        check(rc, "gs_embedding_fwd")
    return y


def _embedding_backward(ctx, g):
    if torch.is_grad_enabled():
        return _once_differentiable(_embedding_backward)(ctx, g)
    ids, = ctx.saved_tensors
    kind, T, V, D, padding_idx, code, scale, need, call = ctx.rest
    g, ldg = _rows(g)
    dw = g.new_empty((V, D))
    ws = g.new_empty(need, dtype=torch.uint8)
    device = g.get_device()
    args = (ids.data_ptr(), kind, g.data_ptr(), ldg, T, V, D, padding_idx, code, scale, dw.data_ptr(), ws.data_ptr(), need, _stream_of(device))
    if _current_device() == device:
        rc = call(*args)
    else:
        with torch.cuda.device(device):
            rc = call(*args)
    if rc:
        check(rc, "gs_embedding_bwd")
    return None, dw, None, None


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        T, (V, D), L = ids.numel(), weight.shape, _lib.lib()
        ctx.rest = (_ID_TYPES[ids.dtype], T, V, D, padding_idx, _DTYPES[weight.dtype], scale, L.gs_embedding_bwd_workspace_bytes(T, V, D), L.gs_embedding_bwd)
        return _lookup(ids, weight, scale)

    backward = staticmethod(_embedding_backward)


_embedding_apply = super(torch.autograd.Function, _EmbeddingFn).apply


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids]: ids int64 or int32 of any shape, weight [V, D] (float32, bfloat16, float16) -> ids.shape + [D].

    The gradient sums a row's tokens in 32 bits, in an order that the sizes and the ids alone decide: the same bits every time.  The row `padding_idx` gets none.  Ids are not looked at on the host: one outside
    of [0, V) gives a row of NaN and has no gradient (negative ids do not count from the end)."""
    if weight.dim() != 2 or weight.dtype not in _DTYPES:
        raise GShellHipError(f"embedding: a weight [V, D] of float32, bfloat16 or float16 is wanted, got {tuple(weight.shape)} {weight.dtype}")
    if ids.dtype not in _ID_TYPES:
        raise GShellHipError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    V, D = weight.shape
    if max(ids.numel(), V, D) >= (1 << 31) - 1:
        raise GShellHipError("embedding: sizes are 0 .. 2^31 - 2")
    if padding_idx is None:
        padding_idx = -1
    elif not 0 <= padding_idx < V:
        raise GShellHipError(f"embedding: padding_idx {padding_idx} is not a row of the table of {V}")
    if not (ids.is_cuda and weight.is_cuda and ids.get_device() == weight.get_device()):
        for name, t in (("ids", ids), ("weight", weight)):
            if not t.is_cuda:
                raise GShellHipError(f"embedding: {name} must live in HBM (got device {t.device}); the HIP path has no CPU fallback")
        raise GShellHipError(f"embedding: ids are on {ids.device}, the weight on {weight.device}")
    flat = ids if ids.is_contiguous() else ids.contiguous()
    try:
        if weight.requires_grad and torch.is_grad_enabled() or _forward_ad._current_level >= 0:
            y = (_EmbeddingFn.apply if _transforms_active() else _embedding_apply)(flat, weight, float(scale), int(padding_idx))
        else:
            y = _lookup(flat, weight, float(scale))
    except RuntimeError:
        inner = _within(flat), _within(weight)
        if _transforms_active() or inner[0] is flat and inner[1] is weight:
            raise
        y = embedding(*inner, scale, None if padding_idx < 0 else padding_idx)
    return y if ids.dim() == 1 else y.view(ids.shape + (D,))


class Embedding(torch.nn.Embedding):
    """torch.nn.Embedding (same parameter, initialisation and state_dict) whose rows come out scaled."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings, freeze=True, padding_idx=None, scale=1.0):
        """A table with the rows of `embeddings` [V, D], which it shares; frozen unless told otherwise."""
        if embeddings.dim() != 2:
            raise GShellHipError(f"Embedding: rows [V, D] are wanted, got {tuple(embeddings.shape)}")
        table = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        table.weight = torch.nn.Parameter(embeddings, requires_grad=not freeze)
        return table

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return super().extra_repr() + f", scale={self.scale}"
