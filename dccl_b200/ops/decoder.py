"""Operators of a decoder block: what stands between its attention, its collectives and its matrix products.

    ====================  ==============================================================================
    function              computes
    ====================  ==============================================================================
    rms_norm              n = x / rms(x) * weight
    residual_norm         y = x + scale * gate * norm(branch), n = rms_norm(y): the end of one sub-block
                          and the entry of the next, in one pass
    rotary                queries and keys turned by their positions
    rotary_frequencies    the frequencies it takes, also those stretched to longer contexts
    gated_linear          act(x Wg^T) * (x Wu^T): the two projections of a gated feed-forward layer
    ====================  ==============================================================================

All are differentiable. CUDA tensors run kernels on the current stream of their device (csrc/decoder/residual_norm.cu, rotary.cu,
gated_linear.cu) in float16, bfloat16 or float32 (gated_linear: not float32): one for a call, of gated_linear up to three (rows that do not start
on 16 bytes are copied, and parts of a sum joined), and in the backward pass two at most for a norm, one for rotary and two to five for gated_linear. Sums and
statistics are fp32 and every result is rounded once. CPU tensors take the same formulas in torch, so the same model code is tested without a
GPU. Inputs may have any strides; what a kernel cannot read in place is copied first. A call allocates its outputs and its workspace from
torch's allocator and nothing else, so it can be captured into a graph. There are no atomics: the order of a sum depends on sizes and, in a
norm, on whether rows start on 16 bytes, so the same inputs in memory that lies alike give the same bits.

Under a mode of torch's (other than the one behind ``torch.device``), a tracer, or with a subclass of Tensor, the same kernels run as operators
of torch's dispatcher (``torch.ops.dccl``), which those see and record. Fake and transformed tensors are refused.

The original has no such operators: its API ends at the collectives (reference include/dccl/dccl.hpp:143-420).
"""
import ctypes
import math
import threading

import torch

from .._lib import lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# as csrc/decoder/decoder_ops.hpp has them
_MAX_WIDTH, _MAX_PAIRS, _MAX_TOKEN, _MAX_DIMENSION = 32768, 1024, 1 << 24, 1 << 30

_ENTRIES = ("dccl_residual_norm", "dccl_residual_norm_workspace", "dccl_residual_norm_backward", "dccl_rotary", "dccl_gated_linear_workspace", "dccl_gated_linear_pads",
            "dccl_gated_linear", "dccl_gated_linear_backward")
_native = None


def _ext():
    """The host side of the operators on CUDA tensors (csrc/torch/decoder_ops.cpp), compiled where that has not been done yet."""
    global _native
    if _native is None:
        from ..parallel import backend_build
        L = lib()
        if not hasattr(L, "dccl_residual_norm"):
            raise RuntimeError("libdccl.so was built without CUDA; the device kernels are missing")
        ext = backend_build.load(compile=True)
        ext.decoder_ops_bind(*(ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRIES))
        _native = ext
    return _native


# ---------------------------------------------------------------------------------------------- calls that something observes

_SCHEMAS = {"residual_norm": "Tensor x, Tensor? branch, Tensor weight, float eps, Tensor? post_weight, Tensor? gate, float scale",
            "rotary": "Tensor q, Tensor? k, Tensor freqs, Tensor? positions, int first, bool interleaved, float scale",
            "gated_linear": "Tensor x, Tensor w_gate, Tensor w_up, int activation"}
_registered, _registering = {}, threading.Lock()


def _run(name, args):
    """The kernels from inside of a registered operator, where nothing observes them any more."""
    if name == "rotary":
        q, k, freqs, positions, first, interleaved, scale = args
        args = q, k, freqs, first if positions is None else positions, interleaved, scale
    out = getattr(_ext(), name)(*args)
    if out is None or out is NotImplemented:
        raise RuntimeError("%s: a registered operator got tensors that are not plain" % name)
    return list(out) if isinstance(out, tuple) else [out]


def _register(name):
    """`name` as an operator of torch's dispatcher, dccl::name, and its gradient as another, so that modes see them and tracers record them. The
    gradient runs the forward pass again: what that keeps is not among the results that a tracer could hand over."""
    def forward(*args):
        with torch._C.DisableTorchFunction(), torch.no_grad():
            return _run(name, args)

    def backward(grads, *rest):
        *args, needed = rest
        with torch._C.DisableTorchFunction(), torch.enable_grad():
            args = [a.detach().contiguous().requires_grad_(n) if isinstance(a, torch.Tensor) else a for a, n in zip(args, needed)]
            outs = [(o, g) for o, g in zip(_run(name, args), grads) if g is not None]
            leaves = [a for a, n in zip(args, needed) if n]
            found, seen = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs], allow_unused=True), []
            for leaf, g in zip(leaves, found):      # results of an operator are tensors of their own
                seen.append(torch.zeros_like(leaf) if g is None else g.clone() if any(g is s for s in seen) else g)
            return seen

    run = torch.library.custom_op("dccl::" + name, forward, mutates_args=(), device_types="cuda", schema="(%s) -> Tensor[]" % _SCHEMAS[name])
    run_back = torch.library.custom_op("dccl::%s_backward" % name, backward, mutates_args=(), device_types="cuda",
                                       schema="(Tensor?[] grads, %s, bool[] needed) -> Tensor[]" % _SCHEMAS[name])

    def setup(ctx, inputs, output):
        ctx.set_materialize_grads(False)
        ctx.others = [None if isinstance(a, torch.Tensor) else (a,) for a in inputs]
        ctx.save_for_backward(*(a for a in inputs if isinstance(a, torch.Tensor)))

    def gradients(ctx, grads):
        needed = list(ctx.needs_input_grad)
        if all(g is None for g in grads) or not any(needed):
            return (None,) * len(needed)
        tensors = iter(ctx.saved_tensors)
        found = iter(run_back(list(grads), *(next(tensors) if o is None else o[0] for o in ctx.others), needed))
        return tuple(next(found) if n else None for n in needed)

    run.register_autograd(gradients, setup_context=setup)
    return run


def _observed(name, *args):
    """The call through torch's dispatcher, which tells whoever follows it."""
    if name == "rotary":
        q, k, freqs, positions, interleaved, scale = args
        args = (q, k, freqs) + ((positions, 0) if isinstance(positions, torch.Tensor) else (None, positions)) + (interleaved, float(scale))
    with _registering:
        if name not in _registered:
            _registered[name] = _register(name)
    out = _registered[name](*args)
    return out[0] if len(out) == 1 else tuple(out)


def _refuse(what):
    """The tensors are of the right types and shapes, and still none that a kernel can read."""
    raise TypeError("%s takes plain tensors: no subclass that replaces their operations, no functorch transform, no complex conjugate" % what)


def _check_like(what, name, t, shape, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: %s must be a tensor" % (what, name))
    if t.shape != shape:
        raise ValueError("%s: %s has shape %s, not %s" % (what, name, tuple(t.shape), tuple(shape)))
    if t.dtype not in dtypes:
        raise TypeError("%s: %s is %s, not %s" % (what, name, t.dtype, " or ".join(str(d) for d in dict.fromkeys(dtypes))))
    if t.device != device:
        raise ValueError("%s: %s is on %s, not on %s" % (what, name, t.device, device))


def _check_activations(what, name, x, dims):
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s: %s must be a tensor" % (what, name))
    if x.dtype not in _DTYPES:
        raise TypeError("%s: %s is %s, not float16, bfloat16 or float32" % (what, name, x.dtype))
    if x.dim() not in dims:
        raise ValueError("%s: %s has %d dimensions" % (what, name, x.dim()))
    if x.device.type not in ("cuda", "cpu"):
        raise ValueError("%s: %s is on %s; CUDA and CPU tensors are taken" % (what, name, x.device))


# ---------------------------------------------------------------------------------------------- norms

def _check_gate(x, gate):
    """A gate of one row ([width], or ones in front of it), or one per entry of the first dimensions of x: x's own sizes and then ones."""
    width, shape = x.shape[-1], tuple(gate.shape)
    ok = shape == (width,)
    if not ok and len(shape) == x.dim() and shape[-1] == width:
        lead, k = tuple(x.shape[:-1]), 0
        while k < len(lead) and shape[k] == lead[k]:
            k += 1
        ok = all(s == 1 for s in shape[k:-1])
    if not ok:
        raise ValueError("residual_norm: gate has shape %s; for x of %s it is [%d], or has x's leading sizes followed by ones" % (shape, tuple(x.shape), width))
    _check_like("residual_norm", "gate", gate, gate.shape, (x.dtype, torch.float32), x.device)


def _norm_on_cpu(x, branch, weight, post, gate, eps, scale):
    def rms(v):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)

    v = x.float()
    if branch is not None:
        p = branch.float()
        if post is not None:
            p = rms(p) * post.float()
        if gate is not None:
            p = p * gate.float()
        v = v + (scale * p if scale != 1.0 else p)
    return v.to(x.dtype), (rms(v) * weight.float()).to(x.dtype)


def _norm(what, x, branch, weight, post, gate, eps, scale):
    if isinstance(x, torch.Tensor) and x.is_cuda:
        out = _ext().residual_norm(x, branch, weight, eps, post, gate, scale)
        if out is None:
            return _observed("residual_norm", x, branch, weight, float(eps), post, gate, float(scale))
        if out is not NotImplemented:
            return out
    _check_activations(what, "x", x, range(1, 65))
    width = x.shape[-1]
    if not 0 < width <= _MAX_WIDTH:
        raise ValueError("%s: rows of %d elements; 1 to %d are taken" % (what, width, _MAX_WIDTH))
    vectors = (x.dtype, torch.float32)
    _check_like(what, "weight", weight, x.shape[-1:], vectors, x.device)
    if branch is not None:
        _check_like(what, "branch", branch, x.shape, (x.dtype,), x.device)
    if post is not None:
        _check_like(what, "post_weight", post, x.shape[-1:], vectors, x.device)
    if gate is not None:
        _check_gate(x, gate)
    eps, scale = float(eps), float(scale)
    if x.is_cuda:
        if x.numel() // width >= 1 << 31:
            raise ValueError("%s: %d rows; fewer than 2^31 are taken" % (what, x.numel() // width))
        out = _ext().residual_norm(x, branch, weight, eps, post, gate, scale)
        if out is None:
            return _observed("residual_norm", x, branch, weight, eps, post, gate, scale)
        return out if out is not NotImplemented else _refuse(what)
    y, n = _norm_on_cpu(x, branch, weight, post, gate, eps, scale)
    return n if branch is None else (y, n)


def rms_norm(x, weight, eps=1e-5):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension. `weight` has x's type, or float32."""
    return _norm("rms_norm", x, None, weight, None, None, eps, 1.0)


def residual_norm(x, branch, weight, eps=1e-5, post_weight=None, gate=None, scale=1.0):
    """The end of a sub-block and the entry of the next one: returns ``(y, n)`` with

        y = x + scale * gate * p        p = branch, or rms_norm(branch, post_weight) where that is given
        n = rms_norm(y, weight)

    `branch` is what the sub-block computed, of x's shape and type. `gate` is one row ([width]), or one row per entry of x's leading
    dimensions ([batch, 1, width] for one gate per sequence). `weight`, `post_weight` and `gate` have x's type, or float32. n
    comes from y before y is rounded. x and branch are kept for the backward pass and must not be overwritten before it. In backward an output that nothing used costs nothing; with scale 1 and neither gate
    nor post_weight, x and branch get the same tensor as their gradient, as from a sum."""
    if branch is None:
        raise TypeError("residual_norm: branch must be a tensor (rms_norm has none)")
    return _norm("residual_norm", x, branch, weight, post_weight, gate, eps, scale)


# ---------------------------------------------------------------------------------------------- rotary positions

def _turn_on_cpu(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    v, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :pairs], v[..., pairs:])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat([turned.to(x.dtype), rest], -1)


def rotary(q, k, freqs, positions=None, interleaved=False, scale=1.0):
    """Rotary positions: pair j of every head's elements turned by ``position * freqs[j]`` radians. Returns the turned q and k (q
    alone where k is None), laid out in memory as they came.

    q, k: [batch, seq, heads, head_dim] or [seq, heads, head_dim] of one type, with any strides (``t.transpose(1, 2)`` of a
        tensor with the heads in front) and head counts of their own.
    freqs: float64 [pairs] (``rotary_frequencies``). The first 2 * pairs elements of a head turn, the others are passed on.
    positions: None (0, 1, ...), the first position of every sequence as an integer, or an int32 or int64 tensor [seq] or [batch, seq].
    interleaved: pair j is (2j, 2j + 1) and not (j, pairs + j).
    scale: factor of the turned elements, as stretched contexts use it."""
    if isinstance(q, torch.Tensor) and q.is_cuda:
        out = _ext().rotary(q, k, freqs, 0 if positions is None else positions, interleaved, scale)
        if out is None:
            return _observed("rotary", q, k, freqs, 0 if positions is None else positions, interleaved, scale)
        if out is not NotImplemented:
            return out
    _check_activations("rotary", "q", q, (3, 4))
    dim = q.shape[-1]
    if k is not None:
        _check_activations("rotary", "k", k, (q.dim(),))
        _check_like("rotary", "k", k, q.shape[:-2] + (k.shape[-2], dim), (q.dtype,), q.device)
    if not isinstance(freqs, torch.Tensor) or freqs.dim() != 1 or not 0 < 2 * freqs.shape[0] <= dim:
        raise ValueError("rotary: freqs is a tensor [pairs] with 1 to head_dim / 2 pairs")
    if freqs.shape[0] > _MAX_PAIRS:
        raise ValueError("rotary: %d pairs; up to %d are taken" % (freqs.shape[0], _MAX_PAIRS))
    _check_like("rotary", "freqs", freqs, freqs.shape, (torch.float64,), q.device)
    if freqs.requires_grad:
        raise ValueError("rotary: freqs has no gradient")
    batch, seq = q.shape[:2] if q.dim() == 4 else (1, q.shape[0])
    if isinstance(positions, torch.Tensor):
        if positions.shape != (seq,) and (q.dim() == 3 or positions.shape != (batch, seq)):
            raise ValueError("rotary: positions has shape %s for %d sequences of %d" % (tuple(positions.shape), batch, seq))
        _check_like("rotary", "positions", positions, positions.shape, (torch.int64, torch.int32), q.device)
    elif positions is None:
        positions = 0
    elif isinstance(positions, bool) or not isinstance(positions, int):
        raise TypeError("rotary: positions is None, an integer or a tensor of integers")
    elif not -2 ** 62 < positions < 2 ** 62:
        raise ValueError("rotary: position %d" % positions)
    else:
        positions = int(positions)
    scale, interleaved = float(scale), bool(interleaved)
    if not q.is_cuda:
        at = positions if isinstance(positions, torch.Tensor) else torch.arange(positions, positions + seq, device=q.device)
        angle = (at.double().unsqueeze(-1) * freqs).unsqueeze(-2)
        cos, sin = (angle.cos() * scale).float(), (angle.sin() * scale).float()
        q = _turn_on_cpu(q, cos, sin, interleaved)
        return q if k is None else (q, _turn_on_cpu(k, cos, sin, interleaved))
    if (q.shape[-2] + (0 if k is None else k.shape[-2])) * dim > _MAX_TOKEN or seq >= 1 << 31:
        raise ValueError("rotary: a token has more than 2^24 elements, or a sequence 2^31 tokens")
    out = _ext().rotary(q, k, freqs, positions, interleaved, scale)
    if out is None:
        return _observed("rotary", q, k, freqs, positions, interleaved, scale)
    return out if out is not NotImplemented else _refuse("rotary")


def rotary_frequencies(rotary_dim, theta=10000.0, scaling=None, factor=1.0, original_length=None, slow=1.0, fast=None, device=None):
    """Radians per position of the rotary_dim / 2 pairs: ``theta ** (-2 j / rotary_dim)``, float64. For contexts `factor` times as long as
    the `original_length` that the model was trained on, `scaling` names how the frequencies change:

    ``"linear"``   all divided by the factor (position interpolation)
    ``"theta"``    theta grows so that the slowest pair is divided by the factor and the fastest is kept
    ``"turns"``    pairs that turn less than `slow` times in the original length are divided by the factor, those above `fast` (4) kept, and
                   between the two the frequency is mixed in proportion to the turns
    ``"yarn"``     the same, mixed in proportion to the index of the pair between those that turn `fast` (32) and `slow` times (Peng et al.,
                   "YaRN: Efficient Context Window Extension of Large Language Models", 2023); it goes with ``scale=0.1 * log(factor) + 1`` in ``rotary``"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim is even, at least 2")
    if factor < 1 or theta <= 1:
        raise ValueError("rotary_frequencies: the factor is at least 1 and theta above 1")
    pairs = rotary_dim // 2
    index = torch.arange(pairs, dtype=torch.float64, device=device)
    if scaling == "theta":
        if pairs == 1:
            raise ValueError("rotary_frequencies: one pair has no slowest and fastest")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(theta) ** (-index / pairs)
    if scaling is None or scaling == "theta":
        return f
    if scaling == "linear":
        return f / factor
    if scaling not in ("turns", "yarn"):
        raise ValueError("rotary_frequencies: scaling %r" % (scaling,))
    if not original_length or original_length <= 0:
        raise ValueError("rotary_frequencies: scaling %r needs original_length" % scaling)
    fast = (4.0 if scaling == "turns" else 32.0) if fast is None else fast
    if not 0 < slow < fast:
        raise ValueError("rotary_frequencies: 0 < slow < fast")
    if scaling == "turns":
        keep = (f * (original_length / (2 * math.pi)) - slow) / (fast - slow)
    else:
        def pair_of(turns):         # the (fractional) pair that turns this often
            return pairs * math.log(original_length / (2 * math.pi * turns)) / math.log(theta)

        first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        keep = 1 - (index - first) / max(last - first, 0.001)
    keep = keep.clamp(0, 1)
    return f * (keep + (1 - keep) / factor)


# ---------------------------------------------------------------------------------------------- gated linear

_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}        # csrc/decoder/decoder_ops.hpp


def _activate_on_cpu(g, activation):
    if activation == "silu":
        return torch.nn.functional.silu(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if activation == "gelu_tanh" else "none")


def gated_linear(x, w_gate, w_up, activation="silu"):
    """``act(x @ w_gate.T) * (x @ w_up.T)``: x [..., width], the weights [ffn, width], all of one type; `activation` is "silu", "gelu" or
    "gelu_tanh". Both products stay in fp32 up to the one rounding of the result.

    On the GPU x is float16 or bfloat16. The gradients of the two products are rounded to that type once, to be multiplied again: in float16
    they overflow above 65504, and dx and the weights' gradients are 1.4 times as far off as their own rounding alone would put them. For the
    backward pass the call keeps the two products in fp32 (8 bytes per element of the result): from 16 bits their rounding would come on top of
    the one that their gradients need. A product that does not end in time (nine seconds) leaves NaN, and the next call on its device raises."""
    if isinstance(x, torch.Tensor) and x.is_cuda and isinstance(activation, str):
        h = _ext().gated_linear(x, w_gate, w_up, _ACTIVATIONS.get(activation, -1))
        if h is None:
            return _observed("gated_linear", x, w_gate, w_up, _ACTIVATIONS[activation])
        if h is not NotImplemented:
            return h
    _check_activations("gated_linear", "x", x, range(1, 65))
    width = x.shape[-1]
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2:
        raise TypeError("gated_linear: w_gate must be a tensor [ffn, width]")
    ffn = w_gate.shape[0]
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        _check_like("gated_linear", name, w, (ffn, width), (x.dtype,), x.device)
    if not width or not ffn:
        raise ValueError("gated_linear: weights of shape %s" % ((ffn, width),))
    if not isinstance(activation, str) or activation not in _ACTIVATIONS:
        raise ValueError("gated_linear: activation %r is none of %s" % (activation, ", ".join(_ACTIVATIONS)))
    if not x.is_cuda:
        v = x.float()
        return (_activate_on_cpu(v @ w_gate.float().t(), activation) * (v @ w_up.float().t())).to(x.dtype)
    if x.dtype is torch.float32:
        raise TypeError("gated_linear: float32 is taken on the CPU only; the tensor cores multiply float16 and bfloat16")
    if max(x.numel() // width, width, ffn) >= _MAX_DIMENSION:
        raise ValueError("gated_linear: a dimension of 2^30 or more")
    _refuse("gated_linear")
