"""One rank of the fused tensor-parallel decoder: its plain, in-place, vocabulary- and sequence-parallel forms against the unsplit decoder of
torch's own operations (loss, and a gradient of each kind)."""
import copy
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

from dccl_b200 import Communicator  # noqa: E402
from dccl_b200.models.llama import LlamaConfig, LlamaDecoder  # noqa: E402
from dccl_b200.models.llama_tp import shard  # noqa: E402


def main():
    comm = Communicator()
    n, r = comm.world, comm.rank
    torch.manual_seed(11)
    full = LlamaDecoder(LlamaConfig(vocab_size=128, hidden=64, layers=2, heads=4, kv_heads=2, ffn=96, max_seq=32))
    tokens = torch.randint(0, 128, (2, 17))
    want = full.loss(tokens)
    want.backward()
    ok = True
    for kw in ({}, {"in_place_reduce": True}, {"vocab_parallel": True}, {"sequence_parallel": True}):
        clean = copy.deepcopy(full)
        clean.zero_grad(set_to_none=True)
        clean.cfg.fused = True
        tp = shard(clean, comm, **kw)
        loss = tp.loss(tokens)
        loss.backward()
        tp.sync_replicated_grads()
        total = loss.detach().clone()
        if "sequence_parallel" in kw:
            comm.all_reduce(total, op="sum")
        got = {"loss": (total, want.detach()), "final norm": (tp.norm.weight.grad, full.norm.weight.grad)}
        for i, (tb, fb) in enumerate(zip(tp.blocks, full.blocks)):
            qw, per = tb.attn.h * tb.attn.hd, tb.gate.out_features
            got.update({"n1 %d" % i: (tb.n1.weight.grad, fb.n1.weight.grad), "n2 %d" % i: (tb.n2.weight.grad, fb.n2.weight.grad),
                        "k %d" % i: (tb.attn.k.weight.grad, fb.attn.k.weight.grad[r * qw // 2:(r + 1) * qw // 2]), "o %d" % i: (tb.attn.o.weight.grad, fb.attn.o.weight.grad[:, r * qw:(r + 1) * qw]),
                        "gate %d" % i: (tb.gate.weight.grad, fb.gate.weight.grad[r * per:(r + 1) * per]), "up %d" % i: (tb.up.weight.grad, fb.up.weight.grad[r * per:(r + 1) * per]),
                        "down %d" % i: (tb.down.weight.grad, fb.down.weight.grad[:, r * per:(r + 1) * per])})
        for what, (a, b) in got.items():
            if not torch.allclose(a, b, rtol=2e-4, atol=2e-5):
                ok = False
                print("rank %d, %s: %s differs by %g" % (r, kw, what, (a - b).abs().max().item()))
        tp.close()
    comm.finalize()
    if not ok:
        sys.exit(1)
    print("OK llama fused worker rank %d" % r)


if __name__ == "__main__":
    main()
