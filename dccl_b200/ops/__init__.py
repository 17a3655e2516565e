"""Differentiable collectives (``dccl_b200.ops.functional``) and operators of models: of a decoder block (``dccl_b200.ops.decoder``), of a mixture of experts
(``dccl_b200.ops.experts``), and of the step between the backward pass and the optimizer (``dccl_b200.ops.gradients``)."""
from .decoder import gated_linear, residual_norm, rms_norm, rotary, rotary_frequencies  # noqa: F401
from .experts import ExpertPlan, combine, dispatch, expert_linear, expert_plan, route  # noqa: F401
from .functional import (all_gather, all_reduce, all_to_all, broadcast, copy_to_region, get_default_communicator,  # noqa: F401
                         recv, reduce_from_region, reduce_scatter, ring_shift, send, set_default_communicator)
from .gradients import clip_grad_norm, grad_norm  # noqa: F401
