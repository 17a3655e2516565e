"""One rank of the test of the fused expert-parallel layer: several experts for a token, against all experts applied in one process; and with one expert
against the layer that is not fused, from its state dict."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

from dccl_b200 import Communicator  # noqa: E402
from dccl_b200.parallel.expert_parallel import ExpertParallelMLP, expert_weights, router_weight  # noqa: E402
from dccl_b200.parallel.tensor_parallel import sync_replicated_grads  # noqa: E402


def main():
    comm = Communicator()
    n, r = comm.world, comm.rank
    d, h, E, T, K = 8, 12, 2 * n, 11, 2
    torch.manual_seed(4321)
    xs = [torch.randn(T + p, d) for p in range(n)]    # a different number of tokens per rank
    ts = [torch.randn(T + p, d) for p in range(n)]
    ok = True

    def check(cond, what):
        nonlocal ok
        if not cond:
            ok = False
            print("rank %d: %s" % (r, what))

    router = router_weight(d, E, 0).requires_grad_(True)
    experts = [[w.requires_grad_(True) for w in expert_weights(d, h, e, 0)] for e in range(E)]
    ref_x = [x.clone().requires_grad_(True) for x in xs]
    ref_out = []
    for x in ref_x:
        s = torch.sigmoid(x @ router.t())
        w, top = s.topk(K, -1)
        w = w / w.sum(-1, keepdim=True) * 1.5
        ref_out.append(torch.stack([sum(w[t, j] * torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(x[t], experts[e][0])), experts[e][1])
                                        for j, e in enumerate(top[t].tolist())) for t in range(x.shape[0])]))
    sum(((o - t) ** 2).sum() for o, t in zip(ref_out, ts)).backward()

    moe = ExpertParallelMLP(d, h, E, comm, seed=0, fused=True, top_k=K, routing=dict(scores="sigmoid", scale=1.5))
    x = xs[r].clone().requires_grad_(True)
    out = moe(x)
    check(torch.allclose(out, ref_out[r].detach(), rtol=1e-4, atol=1e-5), "forward differs")
    ((out - ts[r]) ** 2).sum().backward()
    check(torch.allclose(x.grad, ref_x[r].grad, rtol=1e-4, atol=1e-5), "input gradient differs")
    for j in range(moe.per):
        e = r * moe.per + j
        check(torch.allclose(moe.w_in.grad[j], experts[e][0].grad, rtol=1e-4, atol=1e-5), "expert %d w_in gradient differs" % e)
        check(torch.allclose(moe.w_out.grad[j], experts[e][1].grad, rtol=1e-4, atol=1e-5), "expert %d w_out gradient differs" % e)
    sync_replicated_grads([moe.router], comm)
    check(torch.allclose(moe.router.grad, router.grad, rtol=1e-4, atol=1e-5), "router gradient differs")

    # one expert for a token, weights as the softmax gives them: the layer that is not fused
    plain = ExpertParallelMLP(d, h, E, comm, seed=3)
    fused = ExpertParallelMLP(d, h, E, comm, seed=4, fused=True)
    fused.load_state_dict(plain.state_dict())
    a, b = plain(xs[r]), fused(xs[r])
    check(torch.allclose(a, b, rtol=1e-5, atol=1e-6), "one expert differs")
    again = ExpertParallelMLP(d, h, E, comm, seed=5)
    again.load_state_dict(fused.state_dict())
    check(torch.equal(again(xs[r]), a), "state dict of the fused form")

    # nobody goes anywhere but to the first rank, and one rank has no tokens
    fused.router.data.zero_()
    some = xs[r][:0 if r == n - 1 and n > 1 else 5].clone().requires_grad_(True)
    y = fused(some)
    y.sum().backward()
    check(some.grad.shape == some.shape and bool(torch.isfinite(y).all()), "ranks without rows")
    comm.finalize()
    if not ok:
        sys.exit(1)
    print("OK moe fused worker rank %d" % r)


if __name__ == "__main__":
    main()
