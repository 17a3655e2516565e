"""One rank of the test of norms over ranks: gradients of which every rank has its own, a sharded optimizer with max_norm, and a reducer's clip."""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

from dccl_b200 import Communicator, ops  # noqa: E402
from dccl_b200.parallel.ddp import GradientAllReducer  # noqa: E402
from dccl_b200.parallel.zero import ShardedOptimizer  # noqa: E402


def model_and_data(rank):
    torch.manual_seed(5)
    model = torch.nn.Sequential(torch.nn.Linear(7, 33), torch.nn.GELU(), torch.nn.Linear(33, 5))
    g = torch.Generator().manual_seed(100 + rank)
    return model, torch.randn(6, 7, generator=g), torch.randn(6, 5, generator=g)


def main():
    comm = Communicator()
    n, r = comm.world, comm.rank
    ok = True

    def check(cond, what):
        nonlocal ok
        if not cond:
            ok = False
            print("rank %d: %s" % (r, what))

    parts = [[torch.randn(5 + p, generator=torch.Generator().manual_seed(p)), torch.randn(3, 4, generator=torch.Generator().manual_seed(50 + p))] for p in range(n)]
    want = math.sqrt(sum(float(t.double().square().sum()) for p in parts for t in p))
    mine = [t.clone() for t in parts[r]]
    check(abs(ops.grad_norm(mine, comm=comm).item() - want) < 1e-6 * want, "norm over ranks")
    check(abs(ops.clip_grad_norm(mine, 0.5, comm=comm).item() - want) < 1e-6 * want, "norm of a clip over ranks")
    check(all(torch.allclose(a, b * (0.5 / want), rtol=1e-5) for a, b in zip(mine, parts[r])), "clip over ranks")
    check(abs(ops.grad_norm([torch.zeros(0)] if r else mine, comm=comm).item() - float(torch.cat([t.reshape(-1) for t in parts[0]]).norm()) * 0.5 / want) < 1e-6, "a rank that has none")

    # the same steps on the mean of all ranks' gradients in one process
    plain, _, _ = model_and_data(0)
    opt = torch.optim.AdamW(plain.parameters(), lr=0.01)
    norms = []
    for _ in range(3):
        opt.zero_grad()
        (sum(((plain(x) - y) ** 2).sum() for _, x, y in (model_and_data(p) for p in range(n))) / n).backward()
        norms.append(torch.nn.utils.clip_grad_norm_(plain.parameters(), 0.3).item())
        opt.step()

    model, x, y = model_and_data(r)
    sharded = ShardedOptimizer(model.parameters(), comm, lr=0.01, max_norm=0.3)
    reduced, _, _ = model_and_data(r)
    reducer = GradientAllReducer(reduced, comm, bucket_bytes=512)
    ropt = torch.optim.AdamW(reduced.parameters(), lr=0.01)
    for want in norms:
        sharded.zero_grad()
        ((model(x) - y) ** 2).sum().backward()
        sharded.step()
        check(abs(sharded.grad_norm.item() - want) < 1e-4 * want, "norm of a sharded step")
        reducer.zero_grad()
        ((reduced(x) - y) ** 2).sum().backward()
        reducer.finish()
        check(abs(reducer.clip(0.3).item() - want) < 1e-4 * want, "norm of reduced gradients")
        ropt.step()
    for other, what in ((model, "sharded"), (reduced, "reduced")):
        # three steps of AdamW, which divides by the size of a gradient of rounding errors of 1e-7
        check(all(torch.allclose(a, b, rtol=1e-3, atol=1e-4) for a, b in zip(plain.parameters(), other.parameters())), "parameters, " + what)
    reducer.close()
    sharded.close()
    comm.finalize()
    if not ok:
        sys.exit(1)
    print("OK clip worker rank %d" % r)


if __name__ == "__main__":
    main()
