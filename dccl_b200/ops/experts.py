"""Operators of a mixture of experts: which experts a token goes to, its way there and back, and the experts' products.

    ====================  ==============================================================================
    function              computes
    ====================  ==============================================================================
    route                 the experts of each token and their weights, from a router's logits
    expert_plan           where each token's copies go when they are put in the order of the experts
    dispatch              rows in that order, one for each expert of each token
    expert_linear         act(x W_e^T) for the rows of every expert e
    combine               the weighted sum of each token's rows
    ====================  ==============================================================================

One layer is::

    weights, experts = route(x @ router.T, k)
    plan = expert_plan(experts, num_experts)
    h = expert_linear(dispatch(x, plan), w_in, plan, activation="gelu")
    y = combine(expert_linear(h, w_out, plan), plan, weights)

Nothing of it is read by the host: how many rows an expert has stays on the device, every size is known before (a row for each of a token's experts, whether
it has one or not), and the layer can be captured into a graph. All but expert_plan are differentiable. CUDA tensors run kernels on the current
stream of their device (csrc/experts/route.cu, exchange.cu, grouped.cu) in float16, bfloat16 or float32 (expert_linear: not float32): one for a call and
one for its backward pass. expert_linear has up to three (rows that do not start on 16 bytes are copied, and a product of few tiles is cut along what it sums over and
joined), and in the backward pass one for the activation's gradient and one or two for each of the others. Sums are fp32 and every
result is rounded once. CPU tensors take the same formulas in torch. Inputs may have any strides; what a kernel cannot read in place is copied first. A call
allocates its outputs and its workspace from torch's allocator and nothing else. There are no atomics: the same inputs give the same bits.

Calls that a mode of torch's, a tracer or a subclass of Tensor observes run as operators of torch's dispatcher, as those of ``dccl_b200.ops.decoder`` do.
Fake and transformed tensors are refused.

The original has no such operators: its API ends at the collectives (reference include/dccl/dccl.hpp:143-420).
"""
import ctypes
import itertools
import math
import operator

import torch

from .._lib import lib
from . import _registered
from .decoder import _ACTIVATIONS, _DTYPES, _activate_on_cpu, _check_activations, _check_like, _refuse

# as csrc/experts/expert_ops.hpp has them
_MAX_EXPERTS, _MAX_CHOSEN, _MAX_GROUPS, _MAX_WIDTH, _MAX_PLACES = 1024, 32, 32, 1 << 20, 1 << 30

_ENTRIES = ("dccl_route", "dccl_route_backward", "dccl_expert_plan", "dccl_dispatch", "dccl_combine", "dccl_combine_backward", "dccl_expert_linear_workspace",
            "dccl_expert_linear_pads", "dccl_expert_linear", "dccl_expert_linear_backward")
_native = None


def _ext():
    """The host side of the operators on CUDA tensors (csrc/torch/expert_ops.cpp), compiled where that has not been done yet."""
    global _native
    if _native is None:
        from ..parallel import backend_build
        L = lib()
        if not hasattr(L, "dccl_route"):
            raise RuntimeError("libdccl.so was built without CUDA; the device kernels are missing")
        ext = backend_build.load(compile=True)
        ext.expert_ops_bind(*(ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRIES))
        _native = ext
    return _native


_SCHEMAS = {"route": "Tensor logits, int k, bool sigmoid, Tensor? bias, int groups, int top_groups, bool top2, bool renormalize, float scale",
            "expert_plan": "Tensor experts, int num_experts",
            "dispatch": "Tensor x, Tensor rows, Tensor starts, bool whole",
            "combine": "Tensor rows, Tensor places, Tensor starts, Tensor? weights, bool whole",
            "expert_linear": "Tensor x, Tensor weight, Tensor starts, int activation"}


def _compute(name, args):
    """The kernels from inside of a registered operator, where nothing observes them any more."""
    out = getattr(_ext(), name)(*args)
    if out is None or out is NotImplemented:
        raise RuntimeError("%s: a registered operator got tensors that are not plain" % name)
    return list(out) if isinstance(out, tuple) else [out]


def _kernel(name, *args):
    """The call on CUDA tensors; NotImplemented where the arguments do not fit, and somebody has to say why."""
    out = getattr(_ext(), name)(*args)
    return _registered.call(name, _SCHEMAS[name], _compute, args) if out is None else out


def _integer(what, name, v, low, high):
    """`v` as an int: of any class of integers, and what sizes are while something traces."""
    try:
        n = None if isinstance(v, bool) else operator.index(v)
    except TypeError:
        n = None
    if n is None:
        raise TypeError("%s: %s must be an integer" % (what, name))
    if not low <= n <= high:
        raise ValueError("%s: %s is %d; %d to %d are taken" % (what, name, n, low, high))
    return n


# ---------------------------------------------------------------------------------------------- routing

def _route_on_cpu(logits, k, sigmoid, bias, groups, top_groups, top2, renormalize, scale):
    experts_of = logits.shape[-1]
    z = logits.reshape(-1, experts_of).float()
    with torch.no_grad():
        exact = z.detach().double()
        there = exact > -math.inf
        score = exact
        if bias is not None or (groups > 1 and top2):
            top = torch.where(there, exact, -math.inf).amax(-1, keepdim=True)
            score = torch.sigmoid(exact) if sigmoid else torch.exp(exact - top) / torch.where(there, torch.exp(exact - top), 0.0).sum(-1, keepdim=True)
            if bias is not None:
                score = score + bias.double()
        score = torch.where(there & (score > -math.inf), score, -math.inf)          # NaN is not chosen
        if groups > 1:
            by_group = score.view(-1, groups, experts_of // groups)
            best = by_group.sort(dim=-1, descending=True).values[..., :2]
            of_group = best[..., 0]
            if top2 and best.shape[-1] > 1:
                of_group = of_group + torch.where(best[..., 1] > -math.inf, best[..., 1], 0.0)
            at = of_group.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
            score = torch.where(torch.zeros_like(of_group, dtype=torch.bool).scatter(-1, at, True).unsqueeze(-1), by_group, -math.inf).flatten(1)
        value, at = score.sort(dim=-1, descending=True, stable=True)
        chosen = value[:, :k] > -math.inf
        experts = torch.where(chosen, at[:, :k], -1)
        poisoned = z.isnan().any(-1, keepdim=True) if not sigmoid else torch.zeros_like(chosen[:, :1])
    picked = z.gather(-1, experts.clamp(min=0))
    if renormalize:
        # shares of the chosen: of a softmax their own, of sigmoids that of their logarithms
        of = torch.where(chosen, torch.nn.functional.logsigmoid(picked) if sigmoid else picked, -math.inf)
        of = torch.where(chosen.any(-1, keepdim=True), of, 0.0)
        weights = torch.softmax(of, -1)
    elif sigmoid:
        weights = torch.sigmoid(picked)
    else:
        open_ = torch.where((z == -math.inf).all(-1, keepdim=True), 0.0, z)
        weights = torch.softmax(open_, -1).gather(-1, experts.clamp(min=0))
    weights = torch.where(chosen, torch.where(poisoned, math.nan, weights), 0.0) * scale
    lead = logits.shape[:-1]
    return weights.view(*lead, k), experts.int().view(*lead, k)


def route(logits, k, scores="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """The `k` best of each token's experts, the best first: (weights, experts), float32 and int32 [..., k], of logits [..., experts].

    scores: ``"softmax"`` over the experts, or the ``"sigmoid"`` of each.
    bias: float32 [experts], added to the scores for the choice alone, as it is used to balance the experts' load; it has no gradient.
    groups, top_groups, group_score: the experts in `groups` equal runs, of which the `top_groups` with the best score stay: the group's best expert
        (``"max"``), or the sum of its two best (``"top2"``).
    renormalize: the weights of a token add up to `scale`; otherwise they are the scores times `scale`.

    Of equal scores the expert with the lower number is chosen, and of equal groups likewise. Which experts are chosen is decided as if the scores were exact to 64
    bits. An expert whose logit is minus infinity or NaN is not chosen, nor one whose bias makes its score minus infinity. Where fewer than k are left, the number is -1 and
    the weight 0: a token of padding is one whose logits are all minus infinity. A NaN among the logits (or plus infinity) makes a softmax NaN, and with it all weights of its
    token; where scores are compared and not logits (with a bias, or ``"top2"``), such a token has no experts. The experts are kept for the backward pass and must not be
    overwritten before it."""
    top2, sigmoid = group_score == "top2", scores == "sigmoid"
    if isinstance(logits, torch.Tensor) and logits.is_cuda and scores in ("softmax", "sigmoid") and group_score in ("max", "top2"):
        out = _kernel("route", logits, k, sigmoid, bias, groups, top_groups, top2, bool(renormalize), scale)
        if out is not NotImplemented:
            return out
    _check_activations("route", "logits", logits, range(1, 65))
    n = logits.shape[-1]
    if not 0 < n <= _MAX_EXPERTS:
        raise ValueError("route: %d experts; 1 to %d are taken" % (n, _MAX_EXPERTS))
    if scores not in ("softmax", "sigmoid"):
        raise ValueError("route: scores %r is neither softmax nor sigmoid" % (scores,))
    if group_score not in ("max", "top2"):
        raise ValueError("route: group_score %r is neither max nor top2" % (group_score,))
    groups = _integer("route", "groups", groups, 1, _MAX_GROUPS)
    top_groups = _integer("route", "top_groups", top_groups, 1, groups)
    if n % groups:
        raise ValueError("route: %d experts do not split into %d groups" % (n, groups))
    k = _integer("route", "k", k, 1, min(_MAX_CHOSEN, top_groups * (n // groups)))
    if bias is not None:
        _check_like("route", "bias", bias, (n,), (torch.float32,), logits.device)
    scale = float(scale)
    if not logits.is_cuda:
        return _route_on_cpu(logits, k, sigmoid, bias, groups, top_groups, top2, bool(renormalize), scale)
    if logits.numel() // n * k > _MAX_PLACES:
        raise ValueError("route: %d tokens of %d experts; up to 2^30 are taken" % (logits.numel() // n, k))
    out = _kernel("route", logits, k, sigmoid, bias, groups, top_groups, top2, bool(renormalize), scale)
    return out if out is not NotImplemented else _refuse("route")


# ---------------------------------------------------------------------------------------------- the order of the experts

class ExpertPlan:
    """Where the copies of tokens go in the order of the experts: ``rows`` int32 [..., k], the row of each (-1: none), ``counts`` int32 [experts], how many rows each
    expert has, and ``starts`` int32 [experts + 1], where its rows begin; starts[-1] rows are used.

    A plan may also be made of other tensors, or be given others: one from which places over an expert's capacity are dropped has -1 in ``rows`` for them. No two places have the
    same row, and rows that none has are nobody's, wherever they lie; ``dispatch`` and the gradient of ``combine`` fill all rows of such a plan with zeros first. (The tensors
    of a plan by ``expert_plan`` are not changed where torch does not count it: in place in inference mode, or through ``.data``.)"""
    __slots__ = ("rows", "counts", "starts", "_made")

    def __init__(self, rows, counts, starts, _made=None):
        self.rows, self.counts, self.starts, self._made = rows, counts, starts, _made

    def __setstate__(self, state):          # of a copy, of which it is not known who changes its tensors; or of a plan from before there was _made
        for name in ("rows", "counts", "starts"):
            setattr(self, name, state[1][name])
        self._made = None

    @property
    def num_experts(self):
        return self.counts.shape[0]

    @property
    def _whole(self):
        """Whether each of the rows that are used has a place: in what ``expert_plan`` made, as long as nobody changes it."""
        return (self._made is not None and all(t is m for t, m in zip((self.rows, self.starts), self._made))
                and all(t.is_inference() or t._version == 0 for t in self._made))


def _exchange(name, plan, *args):
    """_kernel with the plan's rows and starts, and what the host side tells by whether it is whole."""
    out = getattr(_ext(), name)(*args, plan._made)
    return _registered.call(name, _SCHEMAS[name], _compute, (*args, plan._whole)) if out is None else out


def _check_chosen(what, name, t):
    if t.dim() < 1 or not 1 <= t.shape[-1] <= _MAX_CHOSEN:
        raise ValueError("%s: %s has shape %s; it is [..., k] with k of 1 to %d" % (what, name, tuple(t.shape), _MAX_CHOSEN))
    if t.numel() > _MAX_PLACES:
        raise ValueError("%s: %d places; up to 2^30 are taken" % (what, t.numel()))


def expert_plan(experts, num_experts):
    """The order of the experts, of int32 or int64 numbers [..., k] as ``route`` gives them: an ``ExpertPlan``. The rows of one expert keep the order of the tokens, and
    of a token's places. A number outside of 0 to num_experts - 1 (-1, as a rule) has no row: its place gets nothing and gives nothing. A token may name an expert
    more than once."""
    if isinstance(experts, torch.Tensor) and experts.is_cuda:
        out = _kernel("expert_plan", experts, num_experts)
        if out is not NotImplemented:
            return ExpertPlan(*out, out[::2])
    if not isinstance(experts, torch.Tensor):
        raise TypeError("expert_plan: experts must be a tensor")
    if experts.dtype not in (torch.int32, torch.int64):
        raise TypeError("expert_plan: experts is %s, not int32 or int64" % experts.dtype)
    if experts.device.type not in ("cuda", "cpu"):
        raise ValueError("expert_plan: experts is on %s; CUDA and CPU tensors are taken" % experts.device)
    num_experts = _integer("expert_plan", "num_experts", num_experts, 1, _MAX_EXPERTS)
    _check_chosen("expert_plan", "experts", experts)
    if experts.is_cuda:
        out = _kernel("expert_plan", experts, num_experts)
        return ExpertPlan(*out, out[::2]) if out is not NotImplemented else _refuse("expert_plan")
    flat = experts.reshape(-1).long()
    there = (flat >= 0) & (flat < num_experts)
    order = torch.where(there, flat, num_experts).argsort(stable=True)
    rows = torch.empty_like(flat).scatter_(0, order, torch.arange(flat.numel(), device=flat.device))
    counts = torch.bincount(flat[there], minlength=num_experts)
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return ExpertPlan(torch.where(there, rows, -1).int().view(experts.shape), counts.int(), starts.int())


def _check_plan(what, plan, device):
    if not isinstance(plan, ExpertPlan):
        raise TypeError("%s: plan must be an ExpertPlan" % what)
    _check_like(what, "plan.rows", plan.rows, plan.rows.shape, (torch.int32,), device)
    _check_chosen(what, "plan.rows", plan.rows)
    _check_starts(what, plan.starts, device)


def _check_starts(what, starts, device):
    if not isinstance(starts, torch.Tensor) or starts.dim() != 1 or not 2 <= starts.shape[0] <= _MAX_EXPERTS + 1:
        raise ValueError("%s: where the experts' rows start is a tensor [experts + 1]" % what)
    _check_like(what, "starts", starts, starts.shape, (torch.int32,), device)


def _check_width(what, width):
    if not 0 < width <= _MAX_WIDTH:
        raise ValueError("%s: rows of %d elements; 1 to %d are taken" % (what, width, _MAX_WIDTH))


def dispatch(x, plan):
    """x [..., width] copied into the order of the experts: [tokens * k, width]. Rows that nobody has, behind the last expert's as a rule, are zeros. The gradient of a token
    is the sum of those of its rows."""
    if isinstance(x, torch.Tensor) and x.is_cuda and isinstance(plan, ExpertPlan):
        out = _ext().dispatch(x, plan.rows, plan.starts, plan._made)
        if out is not None and out is not NotImplemented:
            return out
    _check_activations("dispatch", "x", x, range(1, 65))
    _check_plan("dispatch", plan, x.device)
    if x.shape[:-1] != plan.rows.shape[:-1]:
        raise ValueError("dispatch: x has shape %s, and the plan is for tokens [%s]" % (tuple(x.shape), ", ".join(str(s) for s in plan.rows.shape[:-1])))
    _check_width("dispatch", x.shape[-1])
    if x.is_cuda:
        out = _exchange("dispatch", plan, x, plan.rows, plan.starts)
        return out if out is not NotImplemented else _refuse("dispatch")
    flat, k = plan.rows.reshape(-1).long(), plan.rows.shape[-1]
    places = ((flat >= 0) & (flat < flat.numel())).nonzero().squeeze(-1)
    return x.new_zeros(flat.numel(), x.shape[-1]).index_copy(0, flat[places], x.reshape(-1, x.shape[-1])[places // k])


def combine(rows, plan, weights=None):
    """The sum of each token's rows, times `weights` [..., k] (float32, or of the rows' type) where they are given: [..., width] of rows [tokens * k, width]. A place
    without a row adds nothing, whatever its weight, and its weight's gradient is 0; rows that nobody has are not read, and their gradient is 0."""
    if isinstance(rows, torch.Tensor) and rows.is_cuda and isinstance(plan, ExpertPlan):
        out = _ext().combine(rows, plan.rows, plan.starts, weights, plan._made)
        if out is not None and out is not NotImplemented:
            return out
    _check_activations("combine", "rows", rows, (2,))
    _check_plan("combine", plan, rows.device)
    if rows.shape[0] != plan.rows.numel():
        raise ValueError("combine: %d rows, and the plan has %d places" % (rows.shape[0], plan.rows.numel()))
    _check_width("combine", rows.shape[1])
    if weights is not None:
        _check_like("combine", "weights", weights, plan.rows.shape, (torch.float32, rows.dtype), rows.device)
    if rows.is_cuda:
        out = _exchange("combine", plan, rows, plan.rows, plan.starts, weights)
        return out if out is not NotImplemented else _refuse("combine")
    at = plan.rows.long()
    there = (at >= 0) & (at < at.numel())
    of = rows if not at.numel() else torch.where(there.unsqueeze(-1), rows[torch.where(there, at, 0).reshape(-1)].view(*at.shape, -1), 0.0)
    of = of.float().view(*at.shape, rows.shape[1])
    if weights is not None:
        of = of * torch.where(there, weights.float(), 0.0).unsqueeze(-1)
    return of.sum(-2).to(rows.dtype)


# ---------------------------------------------------------------------------------------------- the experts' products

def expert_linear(rows, weight, plan, activation=None):
    """``act(x @ weight[e].T)`` for the rows x of every expert e: [n, out] of rows [n, width] in the order of the experts and weight [experts, out, width] of one type.
    `plan` is an ``ExpertPlan``, or the int32 tensor [experts + 1] that says where the experts' rows start; `activation` is None, "silu", "gelu" or
    "gelu_tanh". Products stay in fp32 up to the one rounding of the result. Rows that nobody has, before the first expert's and behind the last one's, are not
    read; their results and gradients are zeros: ``expert_linear(rows, weight[2:5], plan.starts[2:6])`` multiplies the rows of three experts. Starts are taken as if they lay
    within [0, n] and none before those ahead of it: no row is of two experts, and one whose end lies before its start has none.

    On the GPU rows and weights are float16 or bfloat16. With an activation the gradient of the product is rounded to that type once, to be multiplied
    again, and the call keeps the product in fp32 for it (4 bytes per element of the result), as ``gated_linear`` does. A product that does not end in time (nine
    seconds) leaves NaN, and the next call on its device raises."""
    starts = plan.starts if isinstance(plan, ExpertPlan) else plan
    act = -1 if activation is None else _ACTIVATIONS.get(activation) if isinstance(activation, str) else None
    if isinstance(rows, torch.Tensor) and rows.is_cuda and act is not None:
        out = _kernel("expert_linear", rows, weight, starts, act)
        if out is not NotImplemented:
            return out
    _check_activations("expert_linear", "rows", rows, (2,))
    if not isinstance(weight, torch.Tensor) or weight.dim() != 3:
        raise TypeError("expert_linear: weight must be a tensor [experts, out, width]")
    experts, out_width, width = weight.shape
    _check_like("expert_linear", "weight", weight, (experts, out_width, rows.shape[1]), (rows.dtype,), rows.device)
    if not 0 < experts <= _MAX_EXPERTS:
        raise ValueError("expert_linear: %d experts; 1 to %d are taken" % (experts, _MAX_EXPERTS))
    _check_width("expert_linear", width)
    _check_width("expert_linear", out_width)
    _check_starts("expert_linear", starts, rows.device)
    if starts.shape[0] != experts + 1:
        raise ValueError("expert_linear: weights of %d experts, and starts of %d" % (experts, starts.shape[0] - 1))
    if act is None:
        raise ValueError("expert_linear: activation %r is none of %s" % (activation, ", ".join(_ACTIVATIONS)))
    if rows.is_cuda:
        if rows.dtype is torch.float32:
            raise TypeError("expert_linear: float32 is taken on the CPU only; the tensor cores multiply float16 and bfloat16")
        if rows.shape[0] > _MAX_PLACES:
            raise ValueError("expert_linear: %d rows; up to 2^30 are taken" % rows.shape[0])
        out = _kernel("expert_linear", rows, weight, starts, act)
        return out if out is not NotImplemented else _refuse("expert_linear")
    n = rows.shape[0]
    out, at = rows.new_zeros(n, out_width), list(itertools.accumulate((min(max(s, 0), n) for s in starts.tolist()), max))
    for e, (start, end) in enumerate(zip(at, at[1:])):
        if end > start or e == 0:       # a product of no rows ties the result to its inputs
            v = rows[start:end].float() @ weight[e].float().t()
            out = out.index_copy(0, torch.arange(start, end, device=rows.device), (v if activation is None else _activate_on_cpu(v, activation)).to(rows.dtype))
    return out
