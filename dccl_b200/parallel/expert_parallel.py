"""Expert-parallel mixture-of-experts layer over the differentiable all-to-all.

The original has no all-to-all (reference include/dccl/dccl.hpp:143-420 ends at send / recv); this library
composes one from grouped send / recv (``dcclAllToAllv``), and this layer is its consumer: E experts are dealt
out E / world to a rank, every token goes to the rank that holds its top-1 expert (dispatch), runs through that
expert and comes back to where it started (combine), scaled by its gate. Backward runs the same two exchanges
with the counts swapped.

    moe = ExpertParallelMLP(d_model, d_hidden, num_experts, comm)
    y = moe(x)                         # x, y: [tokens on this rank, d_model]

With ``fused=True`` the layer computes with the operators of ``dccl_b200.ops.experts``: any number of experts for a token, chosen and weighted as ``ops.route``
takes it, tokens put in the experts' order and added up by kernels, and one product for all experts of a rank instead of two for each segment::

    moe = ExpertParallelMLP(d_model, d_hidden, num_experts, comm, dtype=torch.bfloat16, device="cuda", fused=True, top_k=8,
                            routing=dict(scores="sigmoid", renormalize=True, scale=2.5))

Its experts' weights are one parameter each for all experts of the rank (``w_in`` [experts, h, d], ``w_out`` [experts, d, h]); a state dict of either form loads
into the other. A bias among the keywords of ``routing`` goes with the layer to its device, where it stays fp32, and into its state dict. One rank alone never reads anything back to the host, and can be captured into a graph. (In float32 on the GPU, without autocast, the experts' products are
the plain layer's, and how many rows each has is read.)

The router is replicated; its gradient on a rank covers that rank's tokens only and is summed with the other
replicated parameters (``tensor_parallel.sync_replicated_grads``) when the ranks hold different tokens.
"""
import math

import torch

from ..ops import experts as ops
from ..ops import functional as F


def expert_weights(d_model, d_hidden, expert, seed, dtype=torch.float32, device="cpu"):
    """(w_in [h, d], w_out [d, h]) of one expert, the same for every world size."""
    g = torch.Generator(device="cpu").manual_seed(seed * 1000003 + expert)
    w_in = torch.empty(d_hidden, d_model).uniform_(-1 / math.sqrt(d_model), 1 / math.sqrt(d_model), generator=g)
    w_out = torch.empty(d_model, d_hidden).uniform_(-1 / math.sqrt(d_hidden), 1 / math.sqrt(d_hidden), generator=g)
    return w_in.to(device=device, dtype=dtype), w_out.to(device=device, dtype=dtype)


def router_weight(d_model, num_experts, seed, dtype=torch.float32, device="cpu"):
    g = torch.Generator(device="cpu").manual_seed(seed * 1000003 + 999983)
    return torch.empty(num_experts, d_model).uniform_(-1.0, 1.0, generator=g).to(device=device, dtype=dtype)


class ExpertParallelMLP(torch.nn.Module):
    def __init__(self, d_model, d_hidden, num_experts, comm, seed=0, dtype=torch.float32, device="cpu", fused=False, top_k=1, routing=None):
        """routing: keyword arguments of ``ops.route``; without it the weights are the softmax's, as they are without `fused`."""
        super().__init__()
        if num_experts % comm.world:
            raise ValueError("num_experts must split evenly over the ranks")
        if not fused and (top_k != 1 or routing is not None):
            raise ValueError("top_k and routing need fused=True")
        self.comm, self.num_experts, self.per = comm, num_experts, num_experts // comm.world
        self.fused, self.top_k, self.routing = fused, top_k, dict(renormalize=False) if routing is None else dict(routing)
        self.router = torch.nn.Parameter(router_weight(d_model, num_experts, seed, dtype, device))
        first = comm.rank * self.per
        ws = [expert_weights(d_model, d_hidden, first + j, seed, dtype, device) for j in range(self.per)]
        if fused:
            self.w_in, self.w_out = (torch.nn.Parameter(torch.stack(w)) for w in zip(*ws))
        else:
            self.w_in = torch.nn.ParameterList([torch.nn.Parameter(w[0]) for w in ws])
            self.w_out = torch.nn.ParameterList([torch.nn.Parameter(w[1]) for w in ws])
        self.register_load_state_dict_pre_hook(_take_either_form)

    @property
    def routing_bias(self):
        """The bias among the keywords of ``routing``, by the name that it has in a state dict."""
        return self.routing.get("bias")

    def _apply(self, fn, *args, **kw):
        super()._apply(fn, *args, **kw)
        bias = self.routing_bias
        if bias is not None:            # as a buffer would, but for its type, which is not the layer's
            moved = fn(bias)
            self.routing["bias"] = moved if moved.dtype is bias.dtype else bias.to(moved.device)
        return self

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        bias = self.routing_bias
        if bias is not None:
            destination[prefix + "routing_bias"] = bias if keep_vars else bias.detach()

    def forward(self, x):
        if self.fused:
            return self._forward_fused(x)
        comm, n, per, E = self.comm, self.comm.world, self.per, self.num_experts
        probs = torch.softmax(torch.nn.functional.linear(x, self.router), dim=-1)
        gate, top = probs.max(dim=-1)
        order = torch.argsort(top, stable=True)                 # tokens grouped by expert, hence by destination rank
        counts = torch.bincount(top, minlength=E)               # per expert, on this rank
        # every rank learns how many tokens each source sends to each of its experts
        incoming = torch.empty_like(counts)
        comm.all_to_all(counts.contiguous(), incoming)          # row p: what rank p sends to my experts
        send_counts = counts.view(n, per).sum(1).tolist()
        incoming = incoming.view(n, per)
        recv_counts = incoming.sum(1).tolist()
        got = F.all_to_all(x[order], send_counts, recv_counts, comm)        # dispatch: grouped by source, then by expert
        outs, row = [], 0
        for p in range(n):
            for j in range(per):
                c = int(incoming[p, j])
                seg = got[row:row + c]
                outs.append(torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(seg, self.w_in[j])), self.w_out[j]))
                row += c
        done = torch.cat(outs, 0) if outs else got
        back = F.all_to_all(done, recv_counts, send_counts, comm)           # combine: the way they came
        y = torch.zeros_like(x)
        return y.index_add(0, order, back * gate[order].unsqueeze(-1))

    def _forward_fused(self, x):
        comm, n, per = self.comm, self.comm.world, self.per
        weights, experts = ops.route(torch.nn.functional.linear(x, self.router), self.top_k, **self.routing)
        plan = ops.expert_plan(experts, self.num_experts)
        rows = ops.dispatch(x, plan)                            # in the order of the experts, hence of their ranks
        if n == 1:
            return ops.combine(self._experts(rows, plan).to(x.dtype), plan, weights)
        incoming = torch.empty_like(plan.counts)
        comm.all_to_all(plan.counts, incoming)                  # row p: what rank p sends to my experts
        send_counts, recv_counts = (c.view(n, per).sum(1).tolist() for c in (plan.counts, incoming))
        used = sum(send_counts)
        got = F.all_to_all(rows[:used], send_counts, recv_counts, comm)         # dispatch: grouped by source, then by expert
        of = torch.arange(per, device=x.device).repeat(n).repeat_interleave(incoming, output_size=sum(recv_counts))
        mine = ops.expert_plan(of.unsqueeze(-1), per)
        done = ops.combine(self._experts(ops.dispatch(got, mine), mine), mine)
        back = F.all_to_all(done, recv_counts, send_counts, comm).to(x.dtype)   # combine: the way they came
        return ops.combine(torch.nn.functional.pad(back, (0, 0, 0, rows.shape[0] - used)), plan, weights)

    def _experts(self, rows, plan):
        """Both products of every expert of this rank, for rows in their order; under autocast in its type, as a linear layer's."""
        w_in, w_out = self.w_in, self.w_out
        if torch.is_autocast_enabled(rows.device.type):
            rows, w_in, w_out = (t.to(torch.get_autocast_dtype(rows.device.type)) for t in (rows, w_in, w_out))
        if rows.is_cuda and rows.dtype is torch.float32:        # which the tensor cores do not multiply
            done = [torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(r, w_in[j])), w_out[j])
                    for j, r in enumerate(rows[:int(plan.starts[-1])].split(plan.counts.tolist()))]
            return torch.nn.functional.pad(torch.cat(done), (0, 0, 0, rows.shape[0] - sum(d.shape[0] for d in done)))
        return ops.expert_linear(ops.expert_linear(rows, w_in, plan, activation="gelu"), w_out, plan)


def _take_either_form(module, state, prefix, _metadata, _strict, _missing, _unexpected, errors):
    """Experts' weights in a list or in one tensor, as the module has them, and the bias of its routing."""
    bias, key = module.routing_bias, prefix + "routing_bias"
    if key in state and bias is not None:
        value = state.pop(key)
        if value.shape == bias.shape:
            with torch.no_grad():
                bias.copy_(value)
        else:
            errors.append("size mismatch for %s: %s, and the layer has %s" % (key, tuple(value.shape), tuple(bias.shape)))
    elif not module.fused:
        state.pop(key, None)
    for name in ("w_in", "w_out"):
        one, each = prefix + name, ["%s%s.%d" % (prefix, name, j) for j in range(module.per)]
        if module.fused and each[0] in state and all(k in state for k in each):
            state[one] = torch.stack([state.pop(k) for k in each])
        elif not module.fused and one in state and len(state[one]) == module.per:       # of other numbers it stays, and is not expected
            state.update(zip(each, state.pop(one)))
