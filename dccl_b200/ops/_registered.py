"""Calls that something observes (a mode of torch's, a tracer, a subclass of Tensor): the same kernels as operators of torch's dispatcher.

The fast way into an operator, a function of the extension, is invisible to torch. Where its host side finds that somebody is looking, the call comes here.
"""
import threading

import torch

_operators, _registering = {}, threading.Lock()


def _register(name, schema, compute):
    """`name` as an operator of torch's dispatcher, dccl::name, and its gradient as another, so that modes see them and tracers record them. The
    gradient runs the forward pass again: what that keeps is not among the results that a tracer could hand over."""
    def forward(*args):
        with torch._C.DisableTorchFunction(), torch.no_grad():
            return compute(name, args)

    def backward(grads, *rest):
        *args, needed = rest
        with torch._C.DisableTorchFunction(), torch.enable_grad():
            args = [a.detach().contiguous().requires_grad_(n) if isinstance(a, torch.Tensor) else a for a, n in zip(args, needed)]
            outs = [(o, g) for o, g in zip(compute(name, args), grads) if g is not None]
            leaves = [a for a, n in zip(args, needed) if n]
            found, seen = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs], allow_unused=True), []
            for leaf, g in zip(leaves, found):      # results of an operator are tensors of their own
                seen.append(torch.zeros_like(leaf) if g is None else g.clone() if any(g is s for s in seen) else g)
            return seen

    run = torch.library.custom_op("dccl::" + name, forward, mutates_args=(), device_types="cuda", schema="(%s) -> Tensor[]" % schema)
    run_back = torch.library.custom_op("dccl::%s_backward" % name, backward, mutates_args=(), device_types="cuda",
                                       schema="(Tensor?[] grads, %s, bool[] needed) -> Tensor[]" % schema)

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


def call(name, schema, compute, args):
    """The call through torch's dispatcher, which tells whoever follows it. compute(name, args): the results as a list, where nothing observes it any more."""
    with _registering:
        if name not in _operators:
            _operators[name] = _register(name, schema, compute)
    out = _operators[name](*args)
    return out[0] if len(out) == 1 else tuple(out)
