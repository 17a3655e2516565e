"""The norm of many tensors and clipping (dccl_b200.ops.gradients) against their formulas in 64 bits.

The norm is rounded to fp32 once; the squares of up to eight elements are added in fp32 before that (each off by 2^-24 of at most eight partial sums), which half of counts
in the root: 2^-21 in all, with some to spare. A result of type T is off by half a step of T, and by its factor: the norm's, and the factor's own rounding.
"""
import math
import os

import pytest

torch = pytest.importorskip("torch")
import torch.utils._python_dispatch  # noqa: E402

from dccl_b200 import ops  # noqa: E402
from dccl_b200.utils.launch import python_ranks  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
gpu = pytest.mark.gpu
EACH = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NORM = 2.0 ** -21


def reference(tensors, limit):
    norm = math.sqrt(math.fsum(float(t.detach().double().cpu().square().sum()) for t in tensors))
    return norm, min(1.0, limit / (norm + 1e-6))


def gradients(sizes, dtypes, device="cpu", seed=0, off=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = (torch.randn(n + off, generator=g) * 10.0 ** (-i % 4)).to(dtypes[i % len(dtypes)]).to(device)
        out.append(t[off:])
    return out


def clip_check(tensors, limit, out=None):
    want_norm, factor = reference(tensors, limit)
    before = [t.detach().clone() for t in tensors]
    assert abs(ops.grad_norm(tensors).item() - want_norm) <= NORM * want_norm
    norm = ops.clip_grad_norm(tensors, limit, out=out)
    assert norm.dtype is torch.float32 and norm.dim() == 0 and norm.device == tensors[0].device and abs(norm.item() - want_norm) <= NORM * want_norm
    for t, b, o in zip(tensors, before, out or tensors):
        if out is not None:
            assert torch.equal(t, b)
        want = b.double() * factor
        if factor == 1.0:
            assert torch.equal(o.double(), b.double())
        else:
            u = torch.finfo(o.dtype).eps / 2
            off = (o.double() - want).abs() - (want.abs() * (u + 2 * NORM) + torch.finfo(o.dtype).tiny * u)
            assert bool((off <= 0).all()), (o.dtype, off.max())


SIZES = [[1], [7, 0, 33], [4096], [4097, 1, 2048, 5], [100003, 64, 70000], [3] * 30, [17] * 513, [1000] * 1030]


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dof%d" % (len(s), s[0]))
def test_clipping(device, sizes):
    for dtypes in ([torch.float32], [torch.bfloat16], [torch.float16], DTYPES):
        clip_check(gradients(sizes, dtypes, device), 0.25)
        clip_check(gradients(sizes, dtypes, device), 1e5)
        t = gradients(sizes, dtypes, device)
        clip_check(t, 0.25, out=[torch.empty_like(v) for v in t])
        clip_check(t, 1e5, out=[torch.empty_like(v, dtype=torch.float32) for v in t])
        clip_check(t, 0.25, out=[torch.empty_like(v, dtype=torch.float32) for v in t])


@gpu
@pytest.mark.parametrize("off", range(1, 8))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_tensors_that_start_anywhere(off, dtype):
    sizes = [5, 8, 4096, 4099, 30001, 1, 200000]
    clip_check(gradients(sizes, [dtype], "cuda", off=off), 0.1)
    for other in {dtype, torch.float32}:
        for off2 in (0, 1, off):
            out = [t[off2:] for t in (torch.full((n + off2,), 7.0, device="cuda", dtype=other) for n in sizes)]
            clip_check(gradients(sizes, [dtype], "cuda", off=off), 0.1, out=out)


@gpu
def test_what_lies_beside_the_tensors_is_left():
    buffer = torch.full((50000,), 3.0, device="cuda").bfloat16()
    parts = [buffer[i * 5000 + 3:i * 5000 + 4000 + i] for i in range(10)]
    beside = torch.ones(50000, dtype=torch.bool, device="cuda")
    for i in range(10):
        beside[i * 5000 + 3:i * 5000 + 4000 + i] = False
    clip_check(parts, 1.0)
    assert bool((buffer[beside] == 3).all()) and bool((buffer[~beside] != 3).all())


@gpu
def test_large_tensors():
    """More pieces than CTAs, in both sizes of the table of tensors."""
    clip_check(gradients([30_000_001, 12345, 8_000_000], [torch.bfloat16], "cuda"), 1.0)
    clip_check(gradients([1_000_003] * 40, DTYPES, "cuda"), 1.0)


@pytest.mark.parametrize("device", EACH)
def test_layouts(device):
    """Tensors that are not contiguous: transposed, of channels last, with holes, negated; with outs that lie otherwise."""
    def make():
        g = torch.Generator().manual_seed(3)
        a = torch.randn(40, 60, generator=g).to(device)
        return [a.t(), torch.randn(2, 8, 5, 6, generator=g).to(device).to(memory_format=torch.channels_last), torch.randn(30, 80, generator=g).to(device)[:, 10:61],
                torch.randn((), generator=g).to(device), torch.randn(5, 1, 7, generator=g).to(device)]
    clip_check(make(), 0.5)
    t = make()
    clip_check(t, 0.5, out=[torch.empty(v.shape, device=device) for v in t])
    t = make()
    holes = torch.zeros(40, 200, device=device)
    clip_check(t[:1], 0.5, out=[holes[:, 3:63].t()])
    assert bool((holes[:, :3] == 0).all()) and bool((holes[:, 63:] == 0).all())
    v = torch._neg_view(torch.ones(10, device=device))
    assert abs(ops.grad_norm([v]).item() - math.sqrt(10)) < 1e-5


@pytest.mark.parametrize("device", EACH)
def test_values_that_are_not_finite(device):
    """As torch.nn.utils.clip_grad_norm_ leaves them."""
    for bad in (math.nan, math.inf, -math.inf):
        mine = gradients([40, 30000], [torch.float32], device)
        mine[1][77] = bad
        theirs = [torch.nn.Parameter(torch.zeros_like(t)) for t in mine]
        for p, t in zip(theirs, mine):
            p.grad = t.clone()
        want = torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        norm = ops.clip_grad_norm(mine, 1.0)
        assert norm.isnan().item() == want.isnan().item() and norm.isinf().item() == want.isinf().item()
        for t, p in zip(mine, theirs):
            assert torch.equal(t.isnan(), p.grad.isnan()) and bool((t[~t.isnan()] == 0).all())
    zeros = gradients([40], [torch.float32], device)
    ops.clip_grad_norm(zeros, 0.0)
    assert bool((zeros[0] == 0).all())
    t = [torch.zeros(100, device=device)]
    assert ops.clip_grad_norm(t, 1.0).item() == 0 and bool((t[0] == 0).all())
    t = gradients([100], [torch.float32], device)
    clip_check(t, math.inf)


# What the squares of some eight elements are where fp32 cannot hold them, or only with few bits.
EXTREMES = [6.0e18, 7.0e18, 9.3e18, 3.0e19, 1.0e25, 1.0e33, 1.0e-17, 1.0e-19, 3.0e-21, 1.0e-22, 1.0e-25, 1.0e-33]


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("size", EXTREMES)
def test_squares_beyond_fp32(device, dtype, size):
    """The same norm wherever the tensors start."""
    for off in range(0, 8 if device == "cuda" else 1):
        for sizes in ([5], [64, 1], [4099, 70, 8]):
            tensors = [(t / 10.0 ** (-i % 4) * size).clone() for i, t in enumerate(gradients(sizes, [torch.float32], device))]
            whole = [torch.zeros(t.numel() + off, device=device, dtype=dtype) for t in tensors]
            moved = [v[off:].copy_(t) for v, t in zip(whole, tensors)]
            clip_check(moved, 1.0e-3 if size > 1 else size * 1.0e-8)
    few = torch.zeros(3000, device=device, dtype=dtype)        # among zeros, and beside one element of another size
    few[7], few[2008] = size, -size
    clip_check([few], 1.0e-3 if size > 1 else size * 1.0e-8)
    few[9] = 1.0
    clip_check([few], 1.0e-3)
    assert ops.grad_norm([few * 0]).item() == 0.0


@pytest.mark.parametrize("device", EACH)
def test_gradients_of_a_model(device):
    """Parameters without a gradient are left out, and the answer is torch's."""
    torch.manual_seed(1)
    model = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.ReLU(), torch.nn.Linear(30, 4), torch.nn.Linear(4, 4)).to(device)
    model[:3](torch.randn(9, 20, device=device)).sum().backward()
    grads = [p.grad for p in model.parameters()]
    assert None in grads
    clones = [torch.nn.Parameter(p.detach().clone()) for p in model.parameters()]
    for c, p in zip(clones, model.parameters()):
        c.grad = None if p.grad is None else p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(clones, 0.1)
    versions = [g._version for g in grads if g is not None]
    norm = ops.clip_grad_norm(grads, 0.1)
    assert abs(norm - want) < 1e-5 * want
    for c, p in zip(clones, model.parameters()):
        assert c.grad is None and p.grad is None or torch.allclose(c.grad, p.grad, rtol=1e-5, atol=1e-9)
    assert all(g._version > v for g, v in zip((g for g in grads if g is not None), versions))
    assert ops.grad_norm([]).item() == 0 and ops.clip_grad_norm([None], 1.0).item() == 0
    leaf = torch.ones(5, device=device, requires_grad=True)
    assert not ops.clip_grad_norm([leaf], 1.0).requires_grad and abs(leaf.detach().norm().item() - 1) < 1e-5
    assert ops.grad_norm(leaf).dim() == 0 and not ops.grad_norm(leaf).requires_grad
    assert ops.grad_norm(iter([leaf, leaf])).item() > ops.grad_norm((leaf,)).item()


@pytest.mark.parametrize("device", EACH)
def test_refusals(device):
    t = torch.ones(10, device=device)
    for args, kw, error in ((([t.double()], 1.0), {}, TypeError), (([t.long()], 1.0), {}, TypeError), (([t], -1.0), {}, ValueError), (([t], math.nan), {}, ValueError),
                            ((["a"], 1.0), {}, TypeError), (([t], 1.0), {"out": []}, ValueError), (([t], 1.0), {"out": [t[:5]]}, ValueError),
                            (([t.half()], 1.0), {"out": [t.bfloat16()]}, ValueError), (([t], 1.0), {"out": [t.half()]}, ValueError), (([t, t], 1.0), {}, ValueError),
                            (([t[:1].expand(10)], 1.0), {}, ValueError), (([t.to_sparse()], 1.0), {}, TypeError)):
        with pytest.raises(error):
            ops.clip_grad_norm(*args, **kw)
    assert bool((t == 1).all())
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.clip_grad_norm([t, torch.ones(3)], 1.0)
        for other in ([t[:6], t[4:]], [t[:8], t[4:6]]):
            with pytest.raises(ValueError):
                ops.clip_grad_norm(other, 1.0)
        with pytest.raises(ValueError):
            ops.clip_grad_norm([t[:5]], 1.0, out=[t[3:8]])
        ops.clip_grad_norm([t[:5], t[5:]], 1.0, out=[t[:5], t[5:]])
        assert abs(t.norm().item() - 1) < 1e-5


@pytest.mark.parametrize("device", EACH)
def test_gradients_that_are_read_twice(device):
    """What is only read may be in the list more than once, and in part; what is written may not be what another one reads."""
    t = gradients([1000, 70], [torch.bfloat16], device)
    clip_check([t[0], t[0], t[0][:100], t[1], t[1]], 0.5, [torch.empty_like(v) for v in (t[0], t[0], t[0][:100], t[1], t[1])])
    if device == "cuda":
        for to in ([t[0], torch.empty_like(t[0])], [torch.empty_like(t[0]), t[0]]):
            with pytest.raises(ValueError):
                ops.clip_grad_norm([t[0], t[0]], 0.5, out=to)
        with pytest.raises(ValueError):
            ops.clip_grad_norm([t[0], t[0][:900], t[0][10:20]], 0.5, out=[torch.empty_like(t[0]), torch.empty_like(t[0][:900]), t[0][950:960]])


@gpu
def test_gradients_are_not_widened_in_place():
    """An element of fp32 lies where two of bf16 are read."""
    wide = torch.ones(1000, device="cuda")
    narrow = wide.view(torch.bfloat16)[:1000]
    with pytest.raises(ValueError):
        ops.clip_grad_norm([narrow], 0.5, out=[wide])
    assert bool((wide == 1).all())


@pytest.mark.parametrize("device", EACH)
def test_any_sequence_takes_what_is_clipped(device):
    t = gradients([100, 1], [torch.float32], device)
    want, factor = reference(t, 0.5)
    for tensors, out in ((t, lambda o: iter(o)), (t, tuple), (tuple(t), list), (iter(t), tuple)):
        to = [torch.zeros_like(v) for v in t]
        assert abs(ops.clip_grad_norm(tensors, 0.5, out=out(to)).item() - want) <= NORM * want
        assert all(bool(((o.double() - v.double() * factor).abs() <= v.double().abs() * (2.0 ** -24 + 2 * NORM)).all()) for o, v in zip(to, t))
    one, to = t[:1], torch.zeros_like(t[0])
    ops.clip_grad_norm(one, 0.5, out=to)
    assert abs(to.norm().item() - 0.5) < 1e-5


class SeesDispatch(torch.utils._python_dispatch.TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@gpu
def test_an_active_mode_sees_what_is_done():
    a, b = gradients([100, 3000], DTYPES, "cuda"), gradients([100, 3000], DTYPES, "cuda")
    with SeesDispatch() as m:
        norm = ops.clip_grad_norm(a, 0.5)
    assert any("copy_" in s for s in m.seen) and abs(norm - ops.clip_grad_norm(b, 0.5)) <= 2 * NORM * norm
    for x, y in zip(a, b):
        assert (x.double() - y.double()).abs().max() <= 2 * torch.finfo(x.dtype).eps * y.double().abs().max()


@gpu
def test_clipping_in_graphs():
    """Two captured graphs and eager calls between, on new gradients."""
    t = gradients([5000, 33, 70001], DTYPES, "cuda")
    outs = [torch.empty_like(v) for v in t]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.clip_grad_norm(t, 0.5, out=outs)
    torch.cuda.synchronize()
    graphs = []
    for limit in (0.5, 0.01):
        graph, mine = torch.cuda.CUDAGraph(), [torch.empty_like(v) for v in t]
        with torch.cuda.graph(graph, stream=stream):
            norm = ops.clip_grad_norm(t, limit, out=mine)
        graphs.append((limit, graph, mine, norm))
    for seed in range(3):
        for v, n in zip(t, gradients([5000, 33, 70001], DTYPES, "cuda", seed)):
            v.copy_(n)
        for limit, graph, mine, norm in graphs:
            graph.replay()
            want = ops.clip_grad_norm(t, limit, out=outs)
            torch.cuda.synchronize()
            assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(mine, outs))


@gpu
def test_clipping_on_two_streams():
    t = [gradients([300_000, 44, 100_001], DTYPES, "cuda", seed) for seed in range(2)]
    outs = [[torch.empty_like(v) for v in s] for s in t]
    want = [ops.clip_grad_norm(s, 0.5, out=[torch.empty_like(v) for v in s]) for s in t]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.clip_grad_norm(t[i], 0.5, out=outs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(n, want[i]) for i in range(2) for n in got[i])


@gpu
def test_clipping_on_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    clip_check(gradients([5000, 33], DTYPES, "cuda:1"), 0.5)
    assert torch.cuda.current_device() == 0


@gpu
def test_offsets_beyond_32_bits():
    t = torch.zeros(2 ** 32 + 1001, device="cuda", dtype=torch.bfloat16)
    t[-3:] = torch.tensor([3.0, 4.0, 12.0], device="cuda")
    out = torch.empty_like(t)
    assert ops.clip_grad_norm([t], 6.5, out=[out]).item() == 13.0
    assert out[-3:].tolist() == [1.5, 2.0, 6.0] and out.count_nonzero() == 3


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_steps_that_clip_on_the_gpu(dccl_lib, dtype):
    """The sharded optimizer (the general step and the one-kernel one after it) and the reducer, on one rank, against clipping by torch."""
    from dccl_b200 import Communicator
    from dccl_b200.parallel.ddp import GradientAllReducer
    from dccl_b200.parallel.zero import ShardedOptimizer
    comm = Communicator(rank=0, world=1, device=0)
    try:
        def make():
            torch.manual_seed(3)
            return torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.GELU(), torch.nn.Linear(65, 7)).cuda().to(dtype)
        x = torch.randn(40, 33, device="cuda").to(dtype)
        plain, sharded, reduced = make(), make(), make()
        masters = [torch.nn.Parameter(p.detach().float()) for p in plain.parameters()]
        opt, mine = torch.optim.AdamW(masters, lr=1e-2), ShardedOptimizer(sharded.parameters(), comm, lr=1e-2, max_norm=0.25)
        reducer = GradientAllReducer(reduced, comm)
        for step in range(4):
            for model in (plain, sharded, reduced):
                model.zero_grad(set_to_none=False) if model is plain else (mine.zero_grad() if model is sharded else reducer.zero_grad())
                (model(x).float() - step).pow(2).sum().backward()
            reducer.finish()
            want = torch.nn.utils.clip_grad_norm_(plain.parameters(), 0.25)
            if step == 0:               # later the models differ
                assert abs(reducer.clip(0.25) - want) <= 2.0 ** -6 * want
                assert all(torch.allclose(a.grad, b.grad, rtol=2.0 ** -6, atol=1e-6) for a, b in zip(plain.parameters(), reduced.parameters()))
            for m, p in zip(masters, plain.parameters()):
                m.grad = p.grad.float()
            opt.step()
            mine.step()
            with torch.no_grad():
                for m, p in zip(masters, plain.parameters()):
                    p.copy_(m)
            # clipped gradients rounded once to their type in both
            assert mine.grad_norm.dtype is torch.float32 and abs(mine.grad_norm - want) <= 2.0 ** -5 * want
            # a step moves a parameter by lr at most, and by how much hangs on its gradient's rounding
            for a, b in zip(plain.parameters(), sharded.parameters()):
                assert (a.float() - b.float()).abs().max() <= (step + 1) * 2e-2 * (0.25 if dtype is torch.bfloat16 else 0.05) + torch.finfo(dtype).eps
        reducer.close()
        mine.close()
    finally:
        comm.finalize()


def test_limits_of_the_sharded_optimizer(dccl_lib):
    from dccl_b200 import Communicator
    from dccl_b200.parallel.zero import ShardedOptimizer
    comm = Communicator(rank=0, world=1)
    try:
        for bad in (-1.0, math.nan):
            with pytest.raises(ValueError):
                ShardedOptimizer([torch.nn.Parameter(torch.ones(3))], comm, max_norm=bad)
    finally:
        comm.finalize()


def test_an_optimizer_keeps_a_max_norm_of_its_own(dccl_lib):
    """One that takes the keyword gets it, as it did before there was one of the sharded optimizer."""
    from dccl_b200 import Communicator
    from dccl_b200.parallel.zero import ShardedOptimizer
    seen = []

    class Clips(torch.optim.SGD):
        def __init__(self, params, lr=0.1, max_norm=7.0):
            super().__init__(params, lr=lr)
            seen.append(max_norm)

    comm = Communicator(rank=0, world=1)
    try:
        def step(*args, **kw):
            p = torch.nn.Parameter(torch.zeros(3))
            opt = ShardedOptimizer([p], comm, *args, **kw)
            p.grad.fill_(4.0)
            opt.step()
            return p.detach(), opt.grad_norm

        p, norm = step(Clips, max_norm=0.5)
        assert seen == [0.5] and norm is None and torch.allclose(p, torch.full((3,), -0.4))
        p, norm = step(Clips, lr=1.0)
        assert seen == [0.5, 7.0] and norm is None
        p, norm = step(torch.optim.SGD, lr=1.0, max_norm=0.5)
        assert abs(norm.item() - 48 ** 0.5) < 1e-5 and torch.allclose(p, torch.full((3,), -0.5 / 3 ** 0.5), atol=1e-5)
    finally:
        comm.finalize()


@pytest.mark.parametrize("world", [1, 3])
def test_norms_over_ranks(dccl_lib, world):
    """Gradients of which every rank has its own: grad_norm and clip_grad_norm with a communicator, the sharded optimizer's max_norm and the reducer's clip, against all of
    them in one process."""
    res = python_ranks(os.path.join(HERE, "workers", "clip_worker.py"), [], world, timeout=300)
    for r, p in enumerate(res):
        assert p.returncode == 0, "rank %d:\n%s\n%s" % (r, p.stdout[-3000:], p.stderr[-3000:])
        assert p.stdout.strip().splitlines()[-1].startswith("OK"), p.stdout
