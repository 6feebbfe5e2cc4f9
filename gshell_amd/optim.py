"""torch.optim.Adam with its step as ONE HIP launch over all parameter tensors (csrc/adam.hip: gs_adam_step).

Same constructor, parameter groups, schedulers and state_dict as torch.optim.Adam(fused=True) -- the state is the fused optimiser's
(`step` a float32 device scalar per parameter, `exp_avg`, `exp_avg_sq`), so checkpoints move freely between the two -- and the same
arithmetic (ATen/native/cuda/fused_adam_utils.cuh).  The reference trains with torch.optim.Adam (train_gshelltet_deepfashion.py:372-383).

And the gradient's global norm with clipping by it, two HIP launches over all tensors (csrc/gradnorm.hip: gs_grad_norm): grad_norm, clip_grads, clip_grad_norm_."""
import ctypes
from array import array

import torch

from . import _lib
from ._lib import c_int, check, stream

CONTRACT = 1          # rounding of the moment updates that reproduces ATen's fused kernel bit for bit on gfx950 (tests/test_adam_gpu.py)


class HipAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, **kw):
        for k, bad in (("weight_decay", 0), ("amsgrad", False), ("maximize", False), ("capturable", False), ("differentiable", False)):
            if kw.pop(k, bad) != bad:
                raise NotImplementedError(f"HipAdam: {k} is not used by the reference's optimisers and is not implemented")
        kw.pop("fused", None)
        kw.pop("foreach", None)
        super().__init__(params, lr=lr, betas=betas, eps=eps, fused=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        by_key = {}
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse or p.dtype != torch.float32 or not p.is_cuda:
                    raise _lib.GShellHipError("HipAdam: dense fp32 parameters in HBM only")
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["_host_step"] = None
                if st.get("_host_step") is None:          # fresh state or one loaded from a checkpoint: read the counter once
                    st["_host_step"] = float(st["step"])
                    # a checkpoint written by torch's default (non-fused) Adam keeps `step` on the CPU: the kernel writes the counter through
                    # this pointer, so it has to be a float32 scalar on the parameter's device
                    if st["step"].device != p.device or st["step"].dtype != torch.float32:
                        st["step"] = st["step"].detach().to(device=p.device, dtype=torch.float32)
                    for name in ("exp_avg", "exp_avg_sq"):
                        if st[name].device != p.device or st[name].dtype != torch.float32:
                            st[name] = st[name].detach().to(device=p.device, dtype=torch.float32).contiguous()
                st["_host_step"] += 1.0
                if not (p.is_contiguous() and st["exp_avg"].is_contiguous() and st["exp_avg_sq"].is_contiguous()):
                    raise _lib.GShellHipError("HipAdam: parameters and their moments must be contiguous")
                key = (p.device, tuple(group["betas"]), group["eps"], st["_host_step"])          # a loaded state may carry betas as a list
                by_key.setdefault(key, []).append((p, p.grad if p.grad.is_contiguous() else p.grad.contiguous(), st, float(group["lr"])))
        L = _lib.lib()
        for (dev, betas, eps, step_value), items in by_key.items():
            n = len(items)
            vp = ctypes.c_void_p * n
            keep = [g for _, g, _, _ in items]          # contiguous copies must outlive the launch call
            with torch.cuda.device(dev):
                check(L.gs_adam_step(c_int(n), vp(*[p.data_ptr() for p, _, _, _ in items]), vp(*[g.data_ptr() for g in keep]),
                                     vp(*[st["exp_avg"].data_ptr() for _, _, st, _ in items]), vp(*[st["exp_avg_sq"].data_ptr() for _, _, st, _ in items]),
                                     vp(*[st["step"].data_ptr() for _, _, st, _ in items]), (ctypes.c_int64 * n)(*[p.numel() for p, _, _, _ in items]),
                                     (ctypes.c_double * n)(*[lr for _, _, _, lr in items]), ctypes.c_double(betas[0]), ctypes.c_double(betas[1]),
                                     ctypes.c_double(eps), ctypes.c_double(step_value), c_int(CONTRACT), stream()), "gs_adam_step")
            # the kernel writes the parameters through raw pointers: tell autograd (saved-tensor checks, and every cache keyed on a parameter's
            # version such as the packed SDF-network weights, see them as modified in place)
            torch.autograd.graph.increment_version([p for p, _, _, _ in items])
        return loss

    def state_dict(self):
        sd = super().state_dict()
        sd["state"] = {k: {n: v for n, v in st.items() if n != "_host_step"} for k, st in sd["state"].items()}      # torch's keys only
        return sd

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        for st in self.state.values():
            st["_host_step"] = None


_GRAD_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_stream_of, _group_tensors = torch._C._cuda_getCurrentRawStream, torch._C._group_tensors_by_device_and_dtype
_NORM_TYPES = {2.0: 0, 1.0: 1, float("inf"): 2}


def _norm_code(norm_type, what):
    code = _NORM_TYPES.get(float(norm_type))
    if code is None:
        raise _lib.GShellHipError(f"{what}: norm_type is 2, 1 or inf, got {norm_type}")
    return code


def takes(tensors):
    """Whether the calls below take these gradients: dense float32, bfloat16 or float16, in HBM and on one device, none of them twice."""
    return len({t.get_device() for t in tensors}) <= 1 and all(t.layout is torch.strided and t.is_cuda and t.dtype in _GRAD_TYPES for t in tensors) \
        and len({t.data_ptr() for t in tensors if t.numel()}) == sum(1 for t in tensors if t.numel())


def _refuse_grads(tensors, what):
    for t in tensors:
        if t.layout is not torch.strided or t.dtype not in _GRAD_TYPES:
            raise _lib.GShellHipError(f"{what}: dense float32, bfloat16 or float16 tensors are wanted, got {t.dtype} ({t.layout})")
    for t in tensors:
        if not t.is_cuda:
            raise _lib.GShellHipError(f"{what}: tensors must live in HBM (got device {t.device}); the HIP path has no CPU fallback")
        if t.device != tensors[0].device:
            raise _lib.GShellHipError(f"{what}: tensors are on {tensors[0].device} and on {t.device}")


def _check_grads(tensors, what, out=None):
    """Type codes of `tensors` (and of `out`): dense, on one device, of known types -- on the host, before anything is launched."""
    # Where all are alike one call a list tells (as torch's own optimisers sort their tensors).  A call for both lists would not: it lets the second one's lie on the CPU.
    kinds = list(_group_tensors([tensors], False))
    if len(kinds) == 1 and kinds[0][1] in _GRAD_TYPES and kinds[0][0].type == "cuda" and (out is None or list(_group_tensors([out], False)) == kinds):
        return [_GRAD_TYPES[kinds[0][1]]] * len(tensors)
    types = [_GRAD_TYPES.get(t.dtype) for t in tensors]
    every = tensors if out is None else tensors + out
    devices = {t.get_device() for t in every if t.layout is torch.strided and t.is_cuda}
    if None in types or len(devices) != 1 or not all([t.layout is torch.strided and t.is_cuda for t in every]):
        _refuse_grads(every, what)
    return types


def _dense(tensors, what):
    """Whether each of `tensors` is contiguous; refuses sparse ones."""
    try:
        whole = [t.is_contiguous() for t in tensors]
    except RuntimeError:          # compressed layouts have no such thing
        whole = [False]
    if not all(whole) and any(t.layout is not torch.strided for t in tensors):
        _refuse_grads(tensors, what)
    return whole


def _launch_norm(src, dst, types, max_norm, code):
    """gs_grad_norm over contiguous tensors (dst None: the norm alone)."""
    n, like = len(src), src[0]
    L = _lib.lib()
    need = L.gs_grad_norm_workspace_bytes(n)
    dev = like.get_device()
    norm = like.new_empty((), dtype=torch.float32)
    ws = like.new_empty(need, dtype=torch.uint8)
    at, numel, kinds = array("q", [t.data_ptr() for t in src]), array("q", [t.numel() for t in src]), array("i", types)
    to = None if dst is None else at if dst is src else array("q", [t.data_ptr() for t in dst])
    args = (n, at.buffer_info()[0], None if to is None else to.buffer_info()[0], numel.buffer_info()[0], kinds.buffer_info()[0], code, max_norm, norm.data_ptr(), ws.data_ptr(),
            need, _stream_of(dev))
    if torch._C._cuda_getDevice() == dev:
        rc = L.gs_grad_norm(*args)
    else:
        with torch.cuda.device(dev):
            rc = L.gs_grad_norm(*args)
    if rc:
        check(rc, "gs_grad_norm")
    return norm


def grad_norm(tensors, norm_type=2.0):
    """The norm (2, 1 or inf) of all elements of `tensors` together, one fp32 value on their device; summed in 64 bits."""
    code = _norm_code(norm_type, "grad_norm")
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.zeros(())
    types = _check_grads(tensors, "grad_norm")
    return _launch_norm([t if c else t.detach().contiguous() for t, c in zip(tensors, _dense(tensors, "grad_norm"))], None, types, 0.0, code)


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """out[k] = grads[k] * min(1, max_norm / (norm + 1e-6)) -> norm, one fp32 value on the device.  Without `out`, in place.

    `out`: tensors of the gradients' shapes and types; one may be its gradient's own place, otherwise no output shares memory with a gradient or another output (such a
    call is refused; of outputs that are not contiguous the same one twice, and expanded views).  A norm that is NaN makes every output NaN, one that is infinite makes finite elements zero."""
    code = _norm_code(norm_type, "clip_grads")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.GShellHipError(f"clip_grads: max_norm must not be negative or NaN, got {max_norm}")
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    out = grads if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    if out is not grads:
        if len(out) != len(grads):
            raise _lib.GShellHipError(f"clip_grads: {len(grads)} gradients and {len(out)} outputs")
        for g, o in zip(grads, out):
            if o.dtype != g.dtype or not o.is_same_size(g):
                raise _lib.GShellHipError(f"clip_grads: an output is {tuple(o.shape)} {o.dtype}, its gradient {tuple(g.shape)} {g.dtype}")
    if not grads:
        return torch.zeros(())
    types = _check_grads(grads, "clip_grads", None if out is grads else out)
    whole = _dense(grads, "clip_grads")
    src = grads if all(whole) else [g if c else g.detach().contiguous() for g, c in zip(grads, whole)]
    if out is not grads:
        whole = _dense(out, "clip_grads")
    if all(whole):
        norm = _launch_norm(src, src if out is grads else out, types, max_norm, code)
    else:          # outputs that are not contiguous are written from copies, one after the other
        apart = [o.data_ptr() for o, c in zip(out, whole) if not c]
        if len(set(apart)) != len(apart):
            raise _lib.GShellHipError("clip_grads: the same output twice")
        if any(n > 1 and step == 0 for o, c in zip(out, whole) if not c for n, step in zip(o.shape, o.stride())):
            raise _lib.GShellHipError("clip_grads: elements of an output share a place (an expanded view)")
        dst = src if out is grads else [o if c else torch.empty_like(o, memory_format=torch.contiguous_format) for o, c in zip(out, whole)]
        norm = _launch_norm(src, dst, types, max_norm, code)
        for o, d in zip(out, dst):
            if d is not o:
                o.detach().copy_(d)
    torch.autograd.graph.increment_version(out)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ over parameters whose gradients live on one device: clips their .grad in place, returns the norm before (one fp32 value).

    `error_if_nonfinite` waits for the norm and raises before anything is scaled."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the norm of order {float(norm_type)} is not finite, so the gradients cannot be clipped")
    return clip_grads(grads, max_norm, norm_type)
