"""The norm of all gradients of a model, and gradients cut back to a limit: what a training step does between its backward pass and its optimizer.

    norm = clip_grad_norm([p.grad for p in model.parameters()], 1.0)

CUDA tensors of one device are read by one kernel and scaled by a second one (csrc/gradients/grad_norm.cu), up to 512 tensors each, on the device's current
stream; nothing is read by the host, and the calls can be captured into a graph. CPU tensors take the same formulas in torch.
Squares are added in fp32 within one access of 16 bytes, or in 64 bits where fp32 does not hold them, and in 64 bits from there on, in an order that depends on sizes, types and
addresses only: the same tensors give the same bits. The norm is infinite only where an element is, or where it is itself beyond fp32.

Where gradients are split over ranks, each with its own (the slices of a sharded optimizer, experts that live on one rank), `comm` adds up the squares of all of them.

The original has no such operators: its API ends at the collectives (reference include/dccl/dccl.hpp:143-420).
"""
import ctypes

import torch

from .._lib import lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_ENTRIES = ("dccl_grad_parts", "dccl_grad_squares", "dccl_grad_total", "dccl_grad_clip")
_EPS = 1e-6             # as torch.nn.utils.clip_grad_norm_ adds it, and csrc/gradients/grad_norm.cu
_native = None


def _ext():
    """The host side of the operators on CUDA tensors (csrc/torch/gradient_ops.cpp), compiled where that has not been done yet."""
    global _native
    if _native is None:
        from ..parallel import backend_build
        L = lib()
        if not hasattr(L, "dccl_grad_clip"):
            raise RuntimeError("libdccl.so was built without CUDA; the device kernels are missing")
        ext = backend_build.load(compile=True)
        ext.gradient_ops_bind(*(ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRIES))
        _native = ext
    return _native


def _check(what, name, tensors):
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: %s must be tensors" % (what, name))
        if t.dtype not in _DTYPES or t.layout is not torch.strided:
            raise TypeError("%s: one of %s is %s, %s; strided float16, bfloat16 and float32 are taken" % (what, name, t.dtype, t.layout))
        if t.device.type not in ("cuda", "cpu"):
            raise ValueError("%s: one of %s is on %s; CUDA and CPU tensors are taken" % (what, name, t.device))
        if t.device != tensors[0].device:
            raise ValueError("%s: %s on %s and on %s" % (what, name, tensors[0].device, t.device))


def _is_dense(t):
    return torch.ops.aten.is_non_overlapping_and_dense.default(t) and not t.is_neg()


def _dense(t):
    """The same values where a kernel can read them."""
    return t if _is_dense(t) else t.detach().resolve_neg().contiguous()


def _squares(what, tensors, comm):
    """The sum of all squares, float64, over the ranks of `comm` too."""
    total = _ext().grad_norm([_dense(t) for t in tensors], True) if tensors[0].is_cuda else None
    if total is NotImplemented:
        raise TypeError("%s takes plain tensors: none that stand for others" % what)
    if total is None:           # on the CPU, or something observes the call
        total = torch.zeros((), dtype=torch.float64, device=tensors[0].device)
        for t in tensors:
            total = total + t.detach().double().square().sum()
    return total if comm is None else comm.all_reduce(total, torch.empty_like(total), op="sum")


def grad_norm(tensors, comm=None):
    """``sqrt(sum of all squares)`` of the tensors (None among them is left out), a float32 tensor of no dimensions on their device. With `comm`, of those of all its
    ranks; a rank that has none passes an empty tensor."""
    if type(tensors) is list and comm is None and tensors and isinstance(tensors[0], torch.Tensor) and tensors[0].is_cuda:
        out = _ext().grad_norm(tensors, False)
        if isinstance(out, torch.Tensor):
            return out
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else [t for t in tensors if t is not None]
    _check("grad_norm", "tensors", tensors)
    if not tensors:
        if comm is not None:
            raise ValueError("grad_norm: no tensors, and other ranks wait for their squares; pass an empty one")
        return torch.zeros(())
    with torch.no_grad():
        return _squares("grad_norm", tensors, comm).sqrt().float()


def clip_grad_norm(tensors, max_norm, out=None, comm=None):
    """The tensors (None among them is left out) times ``min(1, max_norm / (norm + 1e-6))``, rounded once, in place or into the tensors of `out` (of the
    same shapes and types, or float32). Returns the norm before, a float32 tensor of no dimensions on their device, which the host need not read; with `comm`, it is
    that of the tensors of all its ranks, as in ``grad_norm``. A norm that is not finite makes the tensors zeros and NaN, as
    ``torch.nn.utils.clip_grad_norm_`` does; where nothing has to change nothing is written in place.

    What is written must not share memory with any other of the tensors."""
    if (type(tensors) is list and comm is None and tensors and isinstance(tensors[0], torch.Tensor) and tensors[0].is_cuda and isinstance(max_norm, (int, float))
            and (out is None or type(out) is list)):
        norm = _ext().clip_grad_norm(tensors, out, max_norm, None)
        if isinstance(norm, torch.Tensor):
            return norm
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if out is None:
        to = tensors = [t for t in tensors if t is not None]
    else:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(tensors):
            raise ValueError("clip_grad_norm: %d tensors and %d of out" % (len(tensors), len(out)))
        to = [o for t, o in zip(tensors, out) if t is not None]
        tensors = [t for t in tensors if t is not None]
        _check("clip_grad_norm", "out", to)
    _check("clip_grad_norm", "tensors", tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("clip_grad_norm: max_norm is %r" % max_norm)
    if not tensors:
        return grad_norm(tensors, comm)
    for t, o in zip(tensors, to):
        if t.shape != o.shape or t.device != o.device or o.dtype not in (t.dtype, torch.float32):
            raise ValueError("clip_grad_norm: a tensor %s of %s on %s, and for it %s of %s on %s" % (tuple(t.shape), t.dtype, t.device, tuple(o.shape), o.dtype, o.device))
        if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
            raise ValueError("clip_grad_norm: a tensor that would be written is expanded")
    if len({o.data_ptr() for o in to if o.numel()}) < sum(o.numel() > 0 for o in to):
        raise ValueError("clip_grad_norm: what is written shares memory with another of the tensors")
    with torch.no_grad():
        total = _squares("clip_grad_norm", tensors, comm)
        if total.is_cuda:
            ins = [_dense(t) for t in tensors]
            outs = [i if o is t else o if _is_dense(o) and o.stride() == i.stride() else torch.empty_like(i, dtype=o.dtype)
                    for t, i, o in zip(tensors, ins, to)]
            norm = _ext().clip_grad_norm(ins, outs, max_norm, total)
            if norm is False:
                raise ValueError("clip_grad_norm: what is written shares memory with another of the tensors")
            if norm is NotImplemented:
                raise TypeError("clip_grad_norm takes plain tensors: none that stand for others")
            if norm is not None:
                for o, w in zip(to, outs):
                    if w is not o:
                        o.copy_(w)
                return norm
        norm = total.sqrt()
        factor = (max_norm / (norm + _EPS)).clamp(max=1.0).float()
        for t, o in zip(tensors, to):
            o.copy_(t.float() * factor)
        return norm.float()
