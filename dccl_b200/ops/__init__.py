"""Differentiable collectives (``dccl_b200.ops.functional``) and the operators of a decoder block (``dccl_b200.ops.decoder``)."""
from .decoder import gated_linear, residual_norm, rms_norm, rotary, rotary_frequencies  # noqa: F401
from .functional import (all_gather, all_reduce, all_to_all, broadcast, copy_to_region, get_default_communicator,  # noqa: F401
                         recv, reduce_from_region, reduce_scatter, ring_shift, send, set_default_communicator)
