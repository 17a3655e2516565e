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

All are differentiable. CUDA tensors run one kernel per call on the current stream of their device (csrc/kernels/residual_norm.cu,
rotary.cu, gated_linear.cu) in float16, bfloat16 or float32 (gated_linear: not float32); sums and statistics are fp32 and every result is rounded once. CPU tensors take
the same formulas in torch, so the same model code is tested without a GPU. Inputs may have any strides; what a kernel cannot
read in place is copied first. A call allocates its outputs and its workspace from torch's allocator and nothing else, so it can be
captured into a graph; a gradient has the same bits whenever its inputs do (no atomics).

The original has no such operators: its API ends at the collectives (reference include/dccl/dccl.hpp:143-420).
"""
import ctypes
import math

import torch

from .._lib import lib
from ..comm import DcclError, current_stream_handle, dtype_of

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_WEIGHT_F32, _POST_F32, _GATE_F32 = 1, 2, 4          # csrc/kernels/decoder_ops.hpp
_MAX_WIDTH, _MAX_PAIRS = 32768, 1024                 # kNormMaxWidth of csrc/kernels/residual_norm.cu, kRotaryPairs of rotary.cu


def _ptr(t):
    return None if t is None else t.data_ptr()


def _done(rc, what):
    if rc != 0:
        raise DcclError(1, what)


def _records(*tensors):
    """Whether autograd has to see a call with these inputs."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


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

def _gates(x, gate):
    """Rows of gates (0: none), each of which covers as many consecutive rows of x."""
    if gate is None:
        return 0
    n = 1
    if gate.dim() > 1:
        for s in gate.shape[:-1]:
            n *= s
    return n


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


def _f32_flags(x, weight, post, gate):
    if x.dtype is torch.float32:
        return 0
    return ((_WEIGHT_F32 if weight.dtype is torch.float32 else 0) | (_POST_F32 if post is not None and post.dtype is torch.float32 else 0)
            | (_GATE_F32 if gate is not None and gate.dtype is torch.float32 else 0))


def _norm_forward(x, branch, weight, post, gate, eps, scale, keep):
    """(y, n, rstd, rstd_post); y is x where there is no branch, the last two are None unless `keep`."""
    width = x.shape[-1]
    rows = x.numel() // width
    n = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y = torch.empty_like(n) if branch is not None else x
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
    rstd_post = torch.empty(rows, dtype=torch.float32, device=x.device) if keep and post is not None else None
    if rows:
        device, gates = x.get_device(), _gates(x, gate)
        _done(lib().dccl_residual_norm(device, dtype_of(x), rows, width, x.data_ptr(), _ptr(branch), weight.data_ptr(), _ptr(post), _ptr(gate), rows // gates if gates else 0,
                                       _f32_flags(x, weight, post, gate), eps, scale, y.data_ptr() if branch is not None else None, n.data_ptr(), _ptr(rstd), _ptr(rstd_post),
                                       current_stream_handle(device)), "residual_norm")
    return y, n, rstd, rstd_post


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, post, gate, eps, scale):
        y, n, rstd, rstd_post = _norm_forward(x, branch, weight, post, gate, eps, scale, True)
        ctx.scale, ctx.has_branch = scale, branch is not None
        ctx.set_materialize_grads(False)
        # of a plain sum y is enough; otherwise the branch is needed anyway, and with x it gives y before its rounding
        full = branch is not None and (post is not None or gate is not None or scale != 1.0)
        ctx.save_for_backward(x if full else y, branch if full else None, weight, post, gate, rstd, rstd_post)
        return (y, n) if branch is not None else n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        y, branch, weight, post, gate, rstd, rstd_post = ctx.saved_tensors
        dy, dn = grads if ctx.has_branch else (None, grads[0])
        if dy is None and dn is None:
            return (None,) * 7
        dy, dn = (None if g is None else g.contiguous() for g in (dy, dn))
        need = ctx.needs_input_grad
        width = y.shape[-1]
        rows = y.numel() // width
        dx = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        dbranch = torch.empty_like(dx) if branch is not None else dx if ctx.has_branch else None
        dweight = torch.empty_like(weight) if need[2] and dn is not None else None
        dpost = torch.empty_like(post) if post is not None and need[3] else None
        dgate = torch.empty_like(gate) if gate is not None and need[4] else None
        if rows:
            device, gates = y.get_device(), _gates(y, gate)
            L, dtype = lib(), dtype_of(y)
            size = L.dccl_residual_norm_workspace(device, rows, width, gates, post is not None, branch is not None)
            work = torch.empty(size // 4, dtype=torch.float32, device=y.device)
            _done(L.dccl_residual_norm_backward(device, dtype, rows, width, _ptr(dy), _ptr(dn), y.data_ptr(), _ptr(branch), weight.data_ptr(), _ptr(post), _ptr(gate),
                                                rows // gates if gates else 0, _f32_flags(y, weight, post, gate), ctx.scale, rstd.data_ptr(), _ptr(rstd_post), dx.data_ptr(),
                                                _ptr(dbranch) if branch is not None else None, _ptr(dweight), _ptr(dpost), _ptr(dgate), work.data_ptr(), size,
                                                current_stream_handle(device)), "residual_norm backward")
        else:
            for g in (dweight, dpost, dgate):
                if g is not None:
                    g.zero_()
        return dx, dbranch, dweight, dpost, dgate, None, None


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
    if not x.is_cuda:
        y, n = _norm_on_cpu(x, branch, weight, post, gate, eps, scale)
        return n if branch is None else (y, n)
    x, branch, weight, post, gate = (None if t is None else t.contiguous() for t in (x, branch, weight, post, gate))
    if _records(x, branch, weight, post, gate):
        return _ResidualNorm.apply(x, branch, weight, post, gate, eps, scale)
    y, n, _, _ = _norm_forward(x, branch, weight, post, gate, eps, scale, False)
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
    comes from y before y is rounded. In backward an output that nothing used costs nothing; with scale 1 and neither gate
    nor post_weight, x and branch get the same tensor as their gradient, as from a sum."""
    if branch is None:
        raise TypeError("residual_norm: branch must be a tensor (rms_norm has none)")
    return _norm("residual_norm", x, branch, weight, post_weight, gate, eps, scale)


# ---------------------------------------------------------------------------------------------- rotary positions

class _Heads(ctypes.Structure):
    """DcclHeads of csrc/kernels/decoder_ops.hpp."""
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p)] + [(n, ctypes.c_longlong) for n in ("ib", "is_", "ih", "ob", "os", "oh")] + [("heads", ctypes.c_int)]


_NO_HEADS = _Heads()


def _heads(x, out):
    """x and out as [batch, seq, heads, dim] by their strides; of three dimensions the batch is missing."""
    if x is None:
        return _NO_HEADS
    i, o = x.stride(), out.stride()
    if x.dim() == 3:
        return _Heads(x.data_ptr(), out.data_ptr(), 0, i[0], i[1], 0, o[0], o[1], x.shape[1])
    return _Heads(x.data_ptr(), out.data_ptr(), i[0], i[1], i[2], o[0], o[1], o[2], x.shape[2])


def _turn(q, k, freqs, positions, interleaved, scale, back):
    outs = []
    for x in (q, k):
        outs.append(None if x is None else torch.empty_like(x))
    like = q if q is not None else k
    batch, seq = (1, like.shape[0]) if like.dim() == 3 else like.shape[:2]
    if batch and seq:
        device = like.get_device()
        at, wide, pb, ps, first = None, 0, 0, 0, 0
        if isinstance(positions, torch.Tensor):
            at, wide = positions.data_ptr(), positions.dtype is torch.int64
            pb, ps = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
        else:
            first = positions
        _done(lib().dccl_rotary(device, dtype_of(like), batch, seq, like.shape[-1], freqs.shape[0], interleaved, back, ctypes.byref(_heads(q, outs[0])),
                                ctypes.byref(_heads(k, outs[1])), freqs.data_ptr(), at, wide, pb, ps, first, scale, current_stream_handle(device)), "rotary")
    return outs


def _dense_head(x):
    return x if x is None or x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, freqs, positions, interleaved, scale):
        tensor = isinstance(positions, torch.Tensor)
        ctx.save_for_backward(freqs, positions if tensor else None)
        ctx.first, ctx.interleaved, ctx.scale = None if tensor else positions, interleaved, scale
        ctx.set_materialize_grads(False)
        q, k = _turn(q, k, freqs, positions, interleaved, scale, 0)
        return q if k is None else (q, k)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        freqs, positions = ctx.saved_tensors
        dq, dk = (None if not need else _dense_head(g) for g, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is not None or dk is not None:
            dq, dk = _turn(dq, dk, freqs, ctx.first if positions is None else positions, ctx.interleaved, ctx.scale, 1)
        return dq, dk, None, None, None, None


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
    scale, interleaved = float(scale), bool(interleaved)
    if not q.is_cuda:
        at = positions if isinstance(positions, torch.Tensor) else torch.arange(positions, positions + seq)
        angle = (at.double().unsqueeze(-1) * freqs).unsqueeze(-2)
        cos, sin = (angle.cos() * scale).float(), (angle.sin() * scale).float()
        q = _turn_on_cpu(q, cos, sin, interleaved)
        return q if k is None else (q, _turn_on_cpu(k, cos, sin, interleaved))
    if (q.shape[-2] + (0 if k is None else k.shape[-2])) * dim > 1 << 24:
        raise ValueError("rotary: a token has more than 2^24 elements")
    q, k, freqs = _dense_head(q), _dense_head(k), freqs.contiguous()
    if _records(q, k):
        return _Rotary.apply(q, k, freqs, positions, interleaved, scale)
    q, k = _turn(q, k, freqs, positions, interleaved, scale, 0)
    return q if k is None else (q, k)


def rotary_frequencies(rotary_dim, theta=10000.0, scaling=None, factor=1.0, original_length=None, slow=1.0, fast=None, device=None):
    """Radians per position of the rotary_dim / 2 pairs: ``theta ** (-2 j / rotary_dim)``, float64. For contexts `factor` times as long as
    the `original_length` that the model was trained on, `scaling` names how the frequencies change:

    ``"linear"``   all divided by the factor (position interpolation)
    ``"theta"``    theta grows so that the slowest pair is divided by the factor and the fastest is kept
    ``"turns"``    pairs that turn less than `slow` times in the original length are divided by the factor, those above `fast` (4) kept, and
                   between the two the frequency is mixed in proportion to the turns
    ``"yarn"``     the same, mixed in proportion to the index of the pair between those that turn `fast` (32) and `slow` times; it goes
                   with ``scale=0.1 * log(factor) + 1`` in ``rotary``"""
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

_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}        # csrc/kernels/decoder_ops.hpp


def _gated_work(x, w_gate, w_up, backward):
    """(workspace or None, its bytes) of a call."""
    aligned = (x.data_ptr() | w_gate.data_ptr() | w_up.data_ptr()) % 16 == 0
    size = lib().dccl_gated_linear_workspace(x.get_device(), x.numel() // x.shape[-1], x.shape[-1], w_gate.shape[0], aligned, backward)
    _done(-1 if size < 0 else 0, "gated_linear")
    return (torch.empty(size, dtype=torch.uint8, device=x.device) if size else None), size


def _gated_forward(x, w_gate, w_up, act, keep):
    """(h, g, u): g and u are the two products in fp32, in rows of a multiple of four elements, or None unless `keep`."""
    width, ffn = x.shape[-1], w_gate.shape[0]
    tokens = x.numel() // width
    h = torch.empty(x.shape[:-1] + (ffn,), dtype=x.dtype, device=x.device)
    g = u = None
    stride = -(-ffn // 4) * 4
    if keep:
        g, u = (torch.empty(tokens, stride, dtype=torch.float32, device=x.device) for _ in range(2))
    if tokens:
        device = x.get_device()
        work, size = _gated_work(x, w_gate, w_up, False)
        _done(lib().dccl_gated_linear(device, dtype_of(x), tokens, width, ffn, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), act, h.data_ptr(), _ptr(g), _ptr(u), stride,
                                      _ptr(work), size, current_stream_handle(device)), "gated_linear")
    return h, g, u


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        h, g, u = _gated_forward(x, w_gate, w_up, act, True)
        ctx.act = act
        ctx.save_for_backward(x, w_gate, w_up, g, u)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        dh = dh.contiguous()
        dx = torch.empty_like(x) if need[0] else None
        dw_gate, dw_up = (torch.empty_like(w_gate), torch.empty_like(w_up)) if need[1] or need[2] else (None, None)
        width, ffn = x.shape[-1], w_gate.shape[0]
        tokens = x.numel() // width
        if tokens:
            device = x.get_device()
            work, size = _gated_work(x, w_gate, w_up, True)
            _done(lib().dccl_gated_linear_backward(device, dtype_of(x), tokens, width, ffn, dh.data_ptr(), g.data_ptr(), u.data_ptr(), g.shape[1], x.data_ptr(), w_gate.data_ptr(),
                                                   w_up.data_ptr(), ctx.act, _ptr(dx), _ptr(dw_gate), _ptr(dw_up), _ptr(work), size, current_stream_handle(device)),
                  "gated_linear backward")
        elif dw_gate is not None:
            dw_gate.zero_(), dw_up.zero_()
        return dx, dw_gate if need[1] else None, dw_up if need[2] else None, None


def _activate_on_cpu(g, activation):
    if activation == "silu":
        return torch.nn.functional.silu(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if activation == "gelu_tanh" else "none")


def gated_linear(x, w_gate, w_up, activation="silu"):
    """``act(x @ w_gate.T) * (x @ w_up.T)``: x [..., width], the weights [ffn, width], all of one type; `activation` is "silu", "gelu" or
    "gelu_tanh". Both products stay in fp32 up to the one rounding of the result.

    On the GPU x is float16 or bfloat16. For the backward pass the call keeps the two products in fp32 (8 bytes per element of the result):
    from 16 bits their rounding would come on top of the one that their gradients need to be multiplied again."""
    _check_activations("gated_linear", "x", x, range(1, 65))
    width = x.shape[-1]
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2:
        raise TypeError("gated_linear: w_gate must be a tensor [ffn, width]")
    ffn = w_gate.shape[0]
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        _check_like("gated_linear", name, w, (ffn, width), (x.dtype,), x.device)
    if not width or not ffn:
        raise ValueError("gated_linear: weights of shape %s" % ((ffn, width),))
    if activation not in _ACTIVATIONS:
        raise ValueError("gated_linear: activation %r is none of %s" % (activation, ", ".join(_ACTIVATIONS)))
    if not x.is_cuda:
        v = x.float()
        return (_activate_on_cpu(v @ w_gate.float().t(), activation) * (v @ w_up.float().t())).to(x.dtype)
    if x.dtype is torch.float32:
        raise TypeError("gated_linear: float32 is taken on the CPU only; the tensor cores multiply float16 and bfloat16")
    if max(x.numel() // width, width, ffn) >= 1 << 30:
        raise ValueError("gated_linear: a dimension of 2^30 or more")
    act = _ACTIVATIONS[activation]
    x, w_gate, w_up = x.contiguous(), w_gate.contiguous(), w_up.contiguous()
    if _records(x, w_gate, w_up):
        return _GatedLinear.apply(x, w_gate, w_up, act)
    return _gated_forward(x, w_gate, w_up, act, False)[0]
