"""The operators of a mixture of experts (dccl_b200.ops.experts) against their formulas in 64 bits.

Tolerances count roundings, as in tests/test_decoder_ops.py: a result of type T is off by half a step of T, and what is computed in fp32 before that by a few times
2^-24 of the terms that went into it. Which experts are chosen, and where rows go, has to be the same.
"""
import math
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
import torch.utils._python_dispatch  # noqa: E402

from dccl_b200 import ops  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EACH = ["cpu", pytest.param("cuda", marks=gpu)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bound = bound + torch.finfo(got.dtype).tiny * half_step(got.dtype)      # below the smallest normal number the steps get no smaller
    got, want, bound = got.detach().double().cpu(), want.detach().cpu(), bound.detach().cpu() if torch.is_tensor(bound) else bound
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), "%s: %.3g over its bound at %s (%.9g, not %.9g)" % (name, off.max(), off.argmax().item(), got.reshape(-1)[off.argmax()], want.reshape(-1)[off.argmax()])


def test_early_launched_kernels_promise_nothing_about_their_inputs():
    """They are launched before the one ahead of them has written, so every one waits, and none declares what it reads read-only for as long as it runs."""
    found = set()
    for folder in ("experts", "gradients"):
        folder = os.path.join(ROOT, "csrc", folder)
        for name in sorted(os.listdir(folder)):
            text = open(os.path.join(folder, name)).read()
            assert "__restrict__" not in text and "__ldg" not in text, name
            for part in text.split("__global__")[1:]:
                signature, body = part.split("{", 1)
                kernel = signature[:signature.rindex("(")].split("k_")[-1].split("(")[0]
                body = body.split("\n}", 1)[0]
                assert "wait_for_stream()" in body or "plan<" in body.split("\n", 1)[0] or body.strip().startswith("grouped<"), kernel
                found.add(kernel)
    assert found >= {"route", "route_grad", "plan", "plan_cluster", "dispatch", "combine", "combine_grad", "grouped", "grouped_pair", "join_parts", "pad_rows", "act_grad", "grad_squares", "grad_total", "grad_clip"}
    plan = open(os.path.join(ROOT, "csrc", "experts", "exchange.cu")).read().split("void plan(")[1]
    assert plan.index("wait_for_stream()") < plan.index("plan_expert(a")
    grouped = open(os.path.join(ROOT, "csrc", "experts", "grouped.cu")).read().split("void grouped(")[1].split("\n}", 1)[0]
    assert grouped.index("wait_for_stream()") < grouped.index("list_tiles(") < grouped.index("grouped_place(") < grouped.index(" load(")


def test_limits_are_those_of_the_entry_points():
    import re
    from dccl_b200.ops import experts
    text = open(os.path.join(ROOT, "csrc", "experts", "expert_ops.hpp")).read()
    limits = {k: eval(v) for k, v in re.findall(r"DCCL_EXPERTS_MAX(\w*) = ([0-9 <]+)", text)}
    assert limits == {"": experts._MAX_EXPERTS, "_CHOSEN": experts._MAX_CHOSEN, "_GROUPS": experts._MAX_GROUPS, "_WIDTH": experts._MAX_WIDTH, "_PLACES": experts._MAX_PLACES}


@pytest.fixture(scope="module")
def tiles_program(tmp_path_factory):
    """tests/sim/grouped_tiles.cpp: how products are cut, without a GPU."""
    exe = str(tmp_path_factory.mktemp("tiles") / "grouped_tiles")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "sim", "grouped_tiles.cpp"), "-o", exe], check=True)
    return exe


def test_tiles_cover_every_expert(tiles_program):
    """Which tiles a product has, and what one that gave up leaves."""
    res = subprocess.run([tiles_program], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout == "OK\n", res.stdout


def test_every_row_is_stored_once(tmp_path):
    """tests/sim/expert_rows.cpp: rows before the first start, and behind the last, as well as those of the experts."""
    exe = str(tmp_path / "expert_rows")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "sim", "expert_rows.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout == "OK\n", res.stdout


def test_kernels_that_give_up_wait_for_their_copies(tmp_path):
    """tests/sim/loads_in_flight.cpp: the barriers and parities of what is under way."""
    exe = str(tmp_path / "loads_in_flight")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "sim", "loads_in_flight.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout == "OK\n", res.stdout


def test_kernels_that_give_up_mark_their_results():
    text = open(os.path.join(ROOT, "csrc", "experts", "grouped.cu")).read()
    parts = text.split("if (failed) {")[1:]
    assert len(parts) == 1 and "grouped_mark(" in parts[0].split("*reinterpret_cast<volatile int*>(a.gave_up) = 1")[0]


# ---------------------------------------------------------------------------------------------- routing

def chosen_of(score, n):
    value, at = torch.sort(score, dim=-1, descending=True, stable=True)
    return torch.where(value[..., :n] > -math.inf, at[..., :n], -1)


def route_reference(z, k, scores, bias, groups, top_groups, group_score, renormalize, scale):
    """(weights, experts) in 64 bits, differentiable."""
    z = z.double()
    closed = (z == -math.inf) | z.isnan()
    p = torch.sigmoid(z) if scores == "sigmoid" else torch.softmax(z.masked_fill((z == -math.inf).all(-1, keepdim=True), 0.0), -1)
    c = (p + (0 if bias is None else bias.double())).detach()
    if bias is None and (groups == 1 or group_score == "max"):
        c = z.detach().clone()
    c = c.masked_fill(closed | c.isnan(), -math.inf)
    if groups > 1:
        g = c.unflatten(-1, (groups, -1))
        best = torch.sort(g, dim=-1, descending=True).values[..., :1 if group_score == "max" else 2]
        score = best.masked_fill(best == -math.inf, 0.0).sum(-1).masked_fill(best[..., 0] == -math.inf, -math.inf)
        stays = (chosen_of(score, top_groups).unsqueeze(-1) == torch.arange(groups, device=z.device)).any(-2)
        c = g.masked_fill(~stays.unsqueeze(-1), -math.inf).flatten(-2)
    experts = chosen_of(c, k)
    there = experts >= 0
    if renormalize:     # s_j / sum s, as the softmax of the logarithms: where all s are zeros to 64 bits their shares are not
        z = z.gather(-1, experts.clamp(min=0))
        z = (torch.nn.functional.logsigmoid(z) if scores == "sigmoid" else z).masked_fill(~there, -math.inf).masked_fill(~there.any(-1, keepdim=True), 0.0)
        p = torch.softmax(z, -1)
    else:
        p = p.gather(-1, experts.clamp(min=0))
    return torch.where(there, p, 0.0) * scale, experts


def route_check(z, k, scores="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0, seed=0):
    how = dict(scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score, renormalize=renormalize, scale=scale)
    weights, experts = ops.route(z, k, **how)
    z = z.detach().clone().requires_grad_(True)
    again, same = ops.route(z, k, **how)
    assert torch.equal(weights, again) and torch.equal(experts, same) and weights.dtype is torch.float32 and experts.dtype is torch.int32
    leaf = z.detach().double().requires_grad_(True)
    want, chosen = route_reference(leaf, k, scores, bias, groups, top_groups, group_score, renormalize, scale)
    assert torch.equal(experts.long(), chosen), (experts.long() != chosen).nonzero()[:5]
    # an exponential is off by 2^-23 and by the rounding of its argument, 2^-24 of up to 128; sums of up to 1024 by 2^-19; with a factor of two
    rel = 2.0 ** -16
    check("weights", again, want, rel * want.abs())
    dw = torch.randn(weights.shape, generator=torch.Generator().manual_seed(seed)).to(z.device)
    dz, = torch.autograd.grad(again, z, dw)
    want_dz, = torch.autograd.grad(want, leaf, dw.double())
    closed = z.detach() == -math.inf
    want_dz = want_dz.masked_fill(closed, 0.0)
    # dz_e = s_e (g_e - sum s_i g_i), or the same of the shares: each term to `rel`. The softmax's derivative of experts that were not chosen has the second term alone.
    size = scale * (dw.double() * (chosen >= 0)).abs()
    share = want.detach() / scale
    both = (share * (size + (share * size).sum(-1, keepdim=True)))
    terms = torch.zeros_like(want_dz).scatter_add(-1, chosen.clamp(min=0), both * (chosen >= 0))
    if scores == "softmax" and not renormalize:
        p = torch.softmax(leaf.detach().masked_fill(closed.all(-1, keepdim=True), 0.0), -1)
        terms = terms + p * (share * size).sum(-1, keepdim=True)
    check("dlogits", dz, want_dz, half_step(z.dtype) * want_dz.abs() + 2 * rel * terms)
    assert bool((dz[closed] == 0).all())


def logits_of(tokens, experts, dtype=torch.float32, device="cpu", seed=0, std=1.5):
    return (torch.randn(tokens, experts, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(device)


def bias_of(experts, device="cpu", std=0.1):
    return (torch.randn(experts, generator=torch.Generator().manual_seed(7)) * std).to(device)


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("form", ["plain", "bias", "groups", "top2", "all"])
def test_route_forms(device, scores, renormalize, form):
    kw = {"plain": {}, "bias": {"bias": bias_of(48, device)}, "groups": {"groups": 6, "top_groups": 2}, "top2": {"groups": 4, "top_groups": 3, "group_score": "top2"},
          "all": {"bias": bias_of(48, device), "groups": 8, "top_groups": 3, "group_score": "top2", "scale": 2.5}}[form]
    for dtype in DTYPES if device == "cuda" else DTYPES[2:]:
        route_check(logits_of(67, 48, dtype, device), 5, scores, renormalize=renormalize, **kw)


@gpu
@pytest.mark.parametrize("experts,k,groups", [(1, 1, 1), (2, 2, 1), (7, 3, 7), (31, 31, 1), (32, 32, 1), (33, 4, 3), (64, 6, 1), (65, 8, 5), (100, 12, 4), (128, 1, 16), (160, 6, 8), (255, 8, 17),
                                              (256, 8, 8), (257, 3, 1), (384, 8, 1), (512, 10, 32), (513, 2, 27), (1000, 32, 8), (1023, 5, 31), (1024, 32, 32)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_at_its_sizes(experts, k, groups, scores):
    for dtype, tokens in ((torch.float32, 301), (torch.bfloat16, 1), (torch.float16, 6)):
        top = min(groups, -(-k // (experts // groups)) + 1)
        route_check(logits_of(tokens, experts, dtype, "cuda"), k, scores)
        route_check(logits_of(tokens, experts, dtype, "cuda"), k, scores, bias_of(experts, "cuda"), groups, top, "top2", False, 1.5)
        route_check(logits_of(tokens, experts, dtype, "cuda"), k, scores, bias_of(experts, "cuda"), groups, top, "max", True, 1.0)


@pytest.mark.parametrize("device", EACH)
def test_route_ties_go_to_the_lower_number(device):
    """Equal logits, with and without a bias, and scores that only the biases make equal to fp32."""
    z = torch.zeros(3, 40, device=device)
    z[1, 20:] = 1.0
    z[2, ::2] = -1.0
    weights, experts = ops.route(z, 4)
    assert experts.tolist() == [[0, 1, 2, 3], [20, 21, 22, 23], [1, 3, 5, 7]] and bool((weights == 0.25).all())
    for bias in (torch.zeros(40, device=device), torch.full((40,), 0.3, device=device)):
        assert torch.equal(ops.route(z, 4, bias=bias, scores="sigmoid")[1], experts)
        assert torch.equal(ops.route(z, 4, bias=bias, groups=4, top_groups=3, group_score="top2")[1].cpu(), route_reference(z.cpu(), 4, "softmax", bias.cpu(), 4, 3, "top2", True, 1.0)[1])
    assert ops.route(z, 4, groups=5, top_groups=2)[1].tolist() == [[0, 1, 2, 3], [20, 21, 22, 23], [1, 3, 5, 7]]


@gpu
def test_route_decides_beyond_fp32():
    """Scores that differ by less than fp32 can tell: logits a step of fp32 apart where the sigmoid is flat, and biases that cancel what the scores differ by."""
    g = torch.Generator().manual_seed(3)
    z = 3 + torch.randint(0, 4, (500, 64), generator=g) * 2.0 ** -22
    z[:, 32:] -= 1.0
    bias = torch.zeros(64)
    bias[32:] = float(torch.sigmoid(torch.tensor(3.0, dtype=torch.float64)) - torch.sigmoid(torch.tensor(2.0, dtype=torch.float64)))
    for scores in ("sigmoid", "softmax"):
        for kw in ({}, {"groups": 8, "top_groups": 3}, {"groups": 8, "top_groups": 3, "group_score": "top2"}):
            _, experts = ops.route(z.cuda(), 6, scores, bias.cuda(), **kw)
            _, want = route_reference(z, 6, scores, bias, kw.get("groups", 1), kw.get("top_groups", 1), kw.get("group_score", "max"), True, 1.0)
            assert torch.equal(experts.cpu().long(), want), (scores, kw)


def choice_check(z, k, scores, bias, **kw):
    _, experts = ops.route(z, k, scores, bias, **kw)
    _, want = route_reference(z.cpu(), k, scores, None if bias is None else bias.cpu(), kw.get("groups", 1), kw.get("top_groups", 1), kw.get("group_score", "max"), True, 1.0)
    wrong = (experts.cpu().long() != want).any(-1).nonzero().squeeze(-1)
    assert not len(wrong), (len(wrong), wrong[0].item(), experts[wrong[0]].tolist(), want[wrong[0]].tolist())


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("experts", [33, 40, 64, 96, 128, 200, 256, 512, 1000, 1024])
def test_route_at_a_border_of_equal_scores(device, experts):
    """The last chosen and the first that is not are the same numbers, and one further back is a step above or below them, or so close that fp32 cannot tell."""
    def case(low, high, above=()):
        """Pairs of `low` and one of `high` at many places, the largest distance apart among them; before them experts that are above both."""
        rows = []
        for a, b, c in ((0, 1, 32), (0, 32, experts - 1), (1, experts - 2, experts - 1), (31, 32, 2), (experts - 3, experts - 1, 0), (5, 30, 32), (0, 2, 3)):
            if len({a, b, c}) < 3:
                continue
            row = torch.zeros(experts)
            row[[a, b]], row[c] = low, high
            for v in above:
                row[[e for e in range(7, experts) if row[e] == 0][0]] = v
            rows.append(row)
        return torch.stack(rows).to(device)

    step = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)).item()
    same = torch.full((experts,), 0.25, device=device)
    for above in ((), (2.0,), (2.0, 3.0, 2.0)):
        for more in (0, 1):
            k = len(above) + 1 + more
            for low, high in ((1.0, step), (step, 1.0), (-1.0, -step), (1.0, 1.0)):
                choice_check(case(low, high, above), k, "softmax", None)
                choice_check(case(low, high, above), k, "sigmoid", None)
            for low, high in ((20.0, 30.0), (30.0, 20.0), (18.0, 18.125), (25.0, 25.0)):
                for bias in (torch.zeros(experts, device=device), same):
                    choice_check(case(low, high, [v + 29 for v in above]), k, "sigmoid", bias)
            for low, high in ((-40.0, -30.0), (-30.0, -30.5), (-20.0, -20.0)):          # beside a softmax's first, which has all but nothing left
                z = case(low, high) - 50.0 * (case(low, high) == 0)
                z[:, 6] = 1.0
                choice_check(z, 1 + k, "softmax", torch.zeros(experts, device=device))
    if experts % 8 == 0:
        for kw in ({"groups": 4, "top_groups": 2}, {"groups": 8, "top_groups": 8}, {"groups": 4, "top_groups": 3, "group_score": "top2"}):
            for low, high in ((20.0, 30.0), (30.0, 20.0), (20.0, 20.0)):
                choice_check(case(low, high), 1, "sigmoid", torch.zeros(experts, device=device), **kw)
                choice_check(case(low, high), 2, "sigmoid", None, **kw)


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("experts,k", [(64, 1), (64, 6), (96, 2), (128, 1), (256, 8), (512, 3), (1024, 32)])
def test_route_of_scores_that_saturate(device, experts, k):
    """bf16 logits of a wide spread, many of them equal, and many sigmoids within a step of 1."""
    z = logits_of(700, experts, torch.bfloat16, device, std=8.0).clamp(-30, 30)
    for bias in (torch.zeros(experts, device=device), torch.full((experts,), 0.5, device=device), (torch.arange(experts, device=device) % 3).float() / 4):
        choice_check(z, k, "sigmoid", bias)
        choice_check(z, k, "softmax", bias)
    choice_check(z, k, "sigmoid", None)
    choice_check(z, k, "sigmoid", torch.zeros(experts, device=device), groups=8, top_groups=max(2, -(-8 * k // experts)), group_score="top2")


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_route_with_closed_experts(device, scores, renormalize, dtype):
    """Logits of minus infinity, some, but for two, and all of a row; rows of the type's lowest number; biases of minus infinity."""
    z = logits_of(9, 40, dtype)
    z[0, 5:] = -math.inf
    z[1] = -math.inf
    z[2] = -math.inf
    z[2, 33], z[2, 7] = 1.0, -2.0
    z[3] = torch.finfo(dtype).min
    z[4, ::2] = torch.finfo(dtype).min
    z[5, 20:] = -math.inf
    z = z.to(device)
    for kw in ({}, {"groups": 5, "top_groups": 2}, {"groups": 4, "top_groups": 4, "group_score": "top2"}):
        route_check(z, 6, scores, renormalize=renormalize, **kw)
        route_check(z, 6, scores, bias_of(40, device), renormalize=renormalize, **kw)
    weights, experts = ops.route(z, 6, scores, renormalize=renormalize)
    assert experts[1].tolist() == [-1] * 6 and experts[2].tolist() == [33, 7, -1, -1, -1, -1] and bool((weights[1] == 0).all()) and bool((weights[2, 2:] == 0).all())
    bias = torch.zeros(40, device=device)
    bias[3:37] = -math.inf
    _, experts = ops.route(logits_of(5, 40, dtype, device), 8, scores, bias, renormalize=renormalize)
    assert all(sorted(row) == [-1, -1, 0, 1, 2, 37, 38, 39] for row in experts.tolist())


@pytest.mark.parametrize("device", EACH)
def test_route_with_nan(device):
    z = logits_of(3, 20, device=device)
    z[1, 4] = math.nan
    for scores in ("softmax", "sigmoid"):
        for bias in (None, bias_of(20, device)):
            weights, experts = ops.route(z, 3, scores, bias)
            clean = ops.route(z[::2], 3, scores, bias)
            assert torch.equal(weights[::2], clean[0]) and torch.equal(experts[::2], clean[1])
            assert 4 not in experts[1].tolist()
            if scores == "softmax":
                assert bool((weights[1].isnan() | (experts[1] < 0)).all())
            else:
                assert bool((experts[1] >= 0).all()) and bool(weights[1].isfinite().all())


@pytest.mark.parametrize("device", EACH)
def test_route_with_infinities(device):
    z = logits_of(2, 20, device=device)
    z[1, 11] = math.inf
    weights, experts = ops.route(z, 3, "sigmoid")
    assert experts[1, 0] == 11 and bool(weights.isfinite().all()) and bool(((weights.sum(-1) - 1).abs() < 1e-6).all())
    weights, experts = ops.route(z, 3, "sigmoid", bias_of(20, device), renormalize=False)
    assert 11 in experts[1].tolist() and bool(weights.isfinite().all())
    weights, experts = ops.route(z, 3)
    assert experts[1, 0] == 11 and bool(weights[1].isnan().all()) and bool(weights[0].isfinite().all())
    bias = torch.zeros(20, device=device)
    bias[3], bias[5], bias[6] = math.inf, math.inf, math.nan
    _, experts = ops.route(z[:1], 18, "sigmoid", bias)
    assert experts[0, :2].tolist() == [3, 5] and 6 not in experts[0].tolist()


@pytest.mark.parametrize("device", EACH)
def test_route_zeros_of_either_sign_are_equal(device):
    z = torch.zeros(1, 12, device=device)
    z[0, ::2] = -0.0
    assert ops.route(z, 4)[1].tolist() == [[0, 1, 2, 3]] and ops.route(z, 4, bias=z[0] * 1.0)[1].tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("device", EACH)
def test_route_scores_that_underflow(device):
    """Shares of the chosen exist where the scores themselves are zero in fp32."""
    z = torch.tensor([[-120.0, -121.0, -500.0, -130.0], [90.0, 89.0, -90.0, 88.0], [-3.0e38, -3.1e38, -3.2e38, -3.3e38]], device=device)
    for scores in ("softmax", "sigmoid"):
        weights, experts = ops.route(z, 2, scores)
        assert experts.tolist() == [[0, 1], [0, 1], [0, 1]]
        e = math.e / (1 + math.e) if scores == "softmax" else None
        first = [e or math.e / (1 + math.e), e or 0.5, 1.0]
        assert all(abs(a - b) < 1e-6 for a, b in zip(weights[:, 0].tolist(), first)), weights
        assert bool(((weights.sum(-1) - 1).abs() < 1e-6).all())


@gpu
def test_route_of_views_and_shapes():
    z = logits_of(60, 48, device="cuda")
    want = ops.route(z, 5, bias=bias_of(48, "cuda"))
    wide = torch.full((60, 100), 9.0, device="cuda")
    wide[:, 1:97:2] = z
    for view in (wide[:, 1:97:2], z.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(ops.route(view, 5, bias=bias_of(48, "cuda")), want))
    a, b = ops.route(z.view(3, 4, 5, 48), 5, bias=bias_of(48, "cuda"))
    assert a.shape == b.shape == (3, 4, 5, 5) and torch.equal(a.view(60, 5), want[0])
    off = torch.zeros(60 * 48 + 1, device="cuda")[1:].view(60, 48).copy_(z)
    assert all(torch.equal(a, b) for a, b in zip(ops.route(off, 5, bias=bias_of(48, "cuda")), want))
    a, b = ops.route(z[:0], 5)
    assert a.shape == b.shape == (0, 5)
    empty = z[:0].requires_grad_(True)
    ops.route(empty, 5)[0].sum().backward()
    assert empty.grad.shape == (0, 48)


@pytest.mark.parametrize("device", EACH)
def test_route_gradient_against_differences(device):
    """Steps so small that no choice changes."""
    for scores in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            z = logits_of(6, 24, device=device).requires_grad_(True)
            dw = torch.randn(6, 4, generator=torch.Generator().manual_seed(5)).to(device)
            weights, experts = ops.route(z, 4, scores, renormalize=renormalize, scale=3.0)
            dz, = torch.autograd.grad(weights, z, dw)
            way, h = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).to(device), 2.0 ** -10
            with torch.no_grad():
                up, down = (ops.route(z + s * h * way, 4, scores, renormalize=renormalize, scale=3.0) for s in (1, -1))
            assert torch.equal(up[1], experts) and torch.equal(down[1], experts)
            want, got = ((up[0] - down[0]).double() * dw.double()).sum() / (2 * h), (dz * way).double().sum()
            # third derivatives are of the size of the first for h = 1; weights of up to 3 are off by 2^-22 each, over 2 h
            assert abs(want - got) <= 30 * h * h + 2.0 ** -22 * 24 * 3 / (2 * h), (scores, renormalize, want, got)


@pytest.mark.parametrize("device", EACH)
def test_route_refusals(device):
    z, b = torch.zeros(4, 12, device=device), torch.zeros(12, device=device)
    for kw, error in (({"k": 0}, ValueError), ({"k": 13}, ValueError), ({"k": 33}, ValueError), ({"k": 2.0}, TypeError), ({"k": True}, TypeError), ({"scores": "linear"}, ValueError),
                      ({"group_score": "mean"}, ValueError), ({"groups": 5}, ValueError), ({"groups": 0}, ValueError), ({"groups": 4, "top_groups": 5}, ValueError),
                      ({"groups": 4, "top_groups": 0}, ValueError), ({"groups": 4, "top_groups": 1, "k": 4}, ValueError), ({"bias": b[:5]}, ValueError), ({"bias": b.double()}, TypeError),
                      ({"bias": 1.0}, TypeError)):
        with pytest.raises(error):
            ops.route(z, **{"k": 2, **kw})
    for bad, error in ((z.double(), TypeError), (z.long(), TypeError), (z[0, 0], ValueError), ([1.0], TypeError), (torch.zeros(2, 1025, device=device), ValueError),
                       (torch.zeros(2, 0, device=device), ValueError)):
        with pytest.raises(error):
            ops.route(bad, 1)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.route(z, 2, bias=b.cpu())


# ---------------------------------------------------------------------------------------------- the order of the experts

def plan_check(experts, n):
    plan = ops.expert_plan(experts, n)
    flat = experts.reshape(-1).cpu().tolist()
    counts, rows = [0] * n, []
    for e in flat:
        if 0 <= e < n:
            counts[e] += 1
    starts = [sum(counts[:e]) for e in range(n + 1)]
    at = list(starts)
    for e in flat:
        if 0 <= e < n:
            rows.append(at[e])
            at[e] += 1
        else:
            rows.append(-1)
    assert plan.rows.dtype is plan.counts.dtype is plan.starts.dtype is torch.int32 and plan.num_experts == n
    assert plan.counts.tolist() == counts and plan.starts.tolist() == starts and plan.rows.shape == experts.shape
    assert plan.rows.reshape(-1).tolist() == rows
    return plan


def chosen_case(tokens, k, experts, seed=0, dropped=0.0, device="cpu", dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    # the first experts are liked better
    at = (torch.rand(tokens, k, generator=g) ** 2 * experts).long().clamp(max=experts - 1)
    at = torch.where(torch.rand(tokens, k, generator=g) < dropped, -1, at)
    return at.to(dtype).to(device)


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
def test_plan(device, dtype):
    for tokens, k, experts in ((0, 2, 3), (1, 1, 1), (5, 3, 4), (40, 2, 7), (33, 1, 2), (100, 4, 9)):
        plan_check(chosen_case(tokens, k, experts, dropped=0.2, device=device, dtype=dtype), experts)


@gpu
@pytest.mark.parametrize("tokens,k,experts", [(1, 32, 8), (32, 1, 1024), (33, 1, 64), (2047, 1, 5), (2048, 1, 256), (2049, 1, 256), (683, 3, 1000), (700, 3, 1024), (8192, 8, 256), (5001, 7, 33),
                                              (100000, 1, 3), (40001, 5, 61)])
def test_plan_at_its_sizes(tokens, k, experts):
    plan_check(chosen_case(tokens, k, experts, device="cuda"), experts)
    plan_check(chosen_case(tokens, k, experts, seed=1, dropped=0.4, device="cuda", dtype=torch.int64), experts)


@pytest.mark.parametrize("device", EACH)
def test_plan_of_numbers_of_no_expert(device):
    big = torch.iinfo(torch.int64)
    plan_check(torch.tensor([[3, -1], [big.min, 2], [big.max, 1 << 32], [(1 << 32) + 1, 0], [4, 5], [-2, 2]], device=device), 4)
    plan_check(torch.tensor([[-1, -1], [7, -5]], device=device, dtype=torch.int32), 3)
    plan_check(torch.full((100, 4), 2, device=device, dtype=torch.int32), 3)
    plan_check(chosen_case(30, 4, 5, device=device).t(), 5)


@pytest.mark.parametrize("device", EACH)
def test_plan_refusals(device):
    e = torch.zeros(4, 2, dtype=torch.int32, device=device)
    for bad, n, error in ((e.float(), 2, TypeError), (e.short(), 2, TypeError), (e, 0, ValueError), (e, 1025, ValueError), (e, 2.0, TypeError), ([1], 2, TypeError), (e[0, 0], 2, ValueError),
                          (torch.zeros(2, 33, dtype=torch.int32, device=device), 2, ValueError), (e[:, :0], 2, ValueError)):
        with pytest.raises(error):
            ops.expert_plan(bad, n)
    import numpy as np
    assert ops.expert_plan(e, np.int64(2)).counts.tolist() == [8, 0]


# ---------------------------------------------------------------------------------------------- dispatch and combine

def exchange_check(tokens, k, experts, width, dtype, device, dropped=0.2, weights32=True, weighted=True, x=None, rows=None):
    plan = plan_check(chosen_case(tokens, k, experts, dropped=dropped, device=device), experts)
    g = torch.Generator().manual_seed(width)
    x = torch.randn(tokens, width, generator=g).to(dtype).to(device) if x is None else x
    done = torch.randn(tokens * k, width, generator=g).to(dtype).to(device) if rows is None else rows
    w = torch.rand(tokens, k, generator=g).to(torch.float32 if weights32 else dtype).to(device) if weighted else None
    drows, dy = torch.randn(tokens * k, width, generator=g).to(dtype).to(device), torch.randn(tokens, width, generator=g).to(dtype).to(device)
    leaves = [t.detach().requires_grad_(True) for t in (x, done, w) if t is not None]
    out = ops.dispatch(leaves[0], plan)
    y = ops.combine(leaves[1], plan, leaves[2] if weighted else None)
    assert torch.equal(out, ops.dispatch(x, plan)) and torch.equal(y, ops.combine(done, plan, w))
    grads = torch.autograd.grad((out, y), leaves, (drows, dy))
    u, at = half_step(dtype), plan.rows.reshape(-1).long().cpu()
    there = at >= 0
    used, token = at[there], torch.arange(tokens * k)[there] // k
    x, done, drows, dy = (t.detach().double().cpu() for t in (x, done, drows, dy))
    w = w.double().cpu().reshape(-1) if weighted else torch.ones(tokens * k, dtype=torch.float64)
    want = torch.zeros(tokens * k, width, dtype=torch.float64)
    want[used] = x[token]
    assert torch.equal(out.detach().double().cpu(), want)

    def sums(r, of):
        v = torch.zeros(tokens * k, width, dtype=torch.float64)
        v[there] = r[used] * of[there].unsqueeze(-1)
        v = v.view(tokens, k, width)
        return v.sum(1), v.abs().sum(1)

    for name, got, (total, size) in (("y", y, sums(done, w)), ("dx", grads[0], sums(drows, torch.ones_like(w)))):
        check(name, got, total, u * total.abs() + (k + 1) * 2.0 ** -24 * size)
    want = torch.zeros(tokens * k, width, dtype=torch.float64)
    want[used] = dy[token] * w[there].unsqueeze(-1)
    check("ddone", grads[1], want, (u + 2.0 ** -24) * want.abs())
    if weighted:
        want, size = torch.zeros(tokens * k, dtype=torch.float64), torch.zeros(tokens * k, dtype=torch.float64)
        want[there], size[there] = (done[used] * dy[token]).sum(-1), (done[used] * dy[token]).abs().sum(-1)
        # sums of at most width terms: of a thread's, and sixteen more
        check("dweights", grads[2].reshape(-1), want, half_step(grads[2].dtype) * want.abs() + (width / 32 + 16) * 2.0 ** -24 * size)
        assert bool((grads[2].reshape(-1).cpu()[~there] == 0).all())


def test_exchange_on_cpu():
    exchange_check(13, 3, 5, 10, torch.float32, "cpu")
    exchange_check(1, 1, 1, 1, torch.float32, "cpu", dropped=0.0)
    exchange_check(6, 2, 4, 7, torch.bfloat16, "cpu", weights32=False)
    exchange_check(6, 2, 4, 7, torch.float32, "cpu", weighted=False)
    exchange_check(6, 2, 4, 7, torch.float32, "cpu", dropped=1.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1), (1, 4, 8, 8), (3, 2, 5, 33), (8, 6, 64, 2048), (257, 3, 11, 1451), (300, 8, 16, 250), (100, 1, 3, 1024), (40, 32, 60, 72), (17, 5, 9, 8192), (5, 2, 4, 8200),
                                   (3, 7, 9, 20001), (1000, 2, 8, 64), (700, 4, 256, 4), (64, 9, 33, 1030), (50, 17, 20, 515)], ids=str)
def test_exchange_at_its_sizes(dtype, sizes):
    exchange_check(*sizes, dtype, "cuda", weights32=sizes[0] % 2 == 0)
    exchange_check(*sizes, dtype, "cuda", dropped=0.0, weighted=sizes[1] % 2 == 0)


@gpu
@pytest.mark.parametrize("off", [1, 2, 4])
@pytest.mark.parametrize("width", [64, 66, 65, 1024, 1451])
def test_exchange_of_rows_that_start_anywhere(off, width):
    def moved(*shape):
        n = math.prod(shape)
        return torch.randn(n + 8, generator=torch.Generator().manual_seed(off)).bfloat16().cuda()[off:off + n].view(shape)
    exchange_check(31, 3, 7, width, torch.bfloat16, "cuda", x=moved(31, width), rows=moved(93, width))


@gpu
def test_exchange_of_views():
    plan = ops.expert_plan(chosen_case(6, 2, 4, device="cuda").view(2, 3, 2), 4)
    x = torch.randn(2, 3, 40, device="cuda").bfloat16()
    want = ops.dispatch(x, plan)
    assert torch.equal(ops.dispatch(x.transpose(0, 1).contiguous().transpose(0, 1), plan), want)
    assert torch.equal(ops.dispatch(x[:1, :1].expand(2, 3, 40), plan), ops.dispatch(x[:1, :1].repeat(2, 3, 1), plan))
    assert ops.combine(want, plan).shape == (2, 3, 40) and torch.equal(ops.combine(want.t().contiguous().t(), plan), ops.combine(want, plan))
    v = torch.randn(1, 40, device="cuda").requires_grad_(True)
    ops.dispatch(v.expand(6, 40).view(2, 3, 40), plan).sum().backward()
    assert bool((v.grad == 12).all())          # a token that six share, two rows each


@pytest.mark.parametrize("device", EACH)
def test_places_without_a_row_give_nothing(device):
    """Whatever their weights are, and rows that nobody has: NaN and infinities stay there."""
    plan = ops.expert_plan(torch.tensor([[1, -1], [-1, -1], [0, 1]], dtype=torch.int32, device=device), 2)
    done = torch.ones(6, 16, device=device)
    done[3:] = math.nan
    done.requires_grad_(True)
    w = torch.tensor([[2.0, math.nan], [math.inf, -math.inf], [0.5, 0.25]], device=device, requires_grad=True)
    y = ops.combine(done, plan, w)
    assert y[:, 0].tolist() == [2.0, 0.0, 0.75]
    y.sum().backward()
    assert done.grad[:, 0].tolist() == [0.5, 2.0, 0.25, 0, 0, 0] and w.grad.tolist() == [[16, 0], [0, 0], [16, 16]]
    x = torch.ones(3, 16, device=device, requires_grad=True)
    out = ops.dispatch(x, plan)
    assert out[:, 0].tolist() == [1, 1, 1, 0, 0, 0]
    g = torch.ones_like(out)
    g[3:] = math.nan
    out.backward(g)
    assert x.grad[:, 0].tolist() == [1, 0, 2]
    nothing = ops.expert_plan(torch.full((3, 2), -1, dtype=torch.int32, device=device), 2)
    assert bool((ops.dispatch(x, nothing) == 0).all()) and bool((ops.combine(done, nothing, w) == 0).all())


@gpu
def test_places_of_a_plan_that_is_none_are_not_followed():
    """Rows beyond all, as no plan has them."""
    rows = torch.tensor([[0, 1], [100, -7], [torch.iinfo(torch.int32).max, 2]], dtype=torch.int32, device="cuda")
    plan = ops.ExpertPlan(rows, torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 0, 3], dtype=torch.int32, device="cuda"))
    x = torch.arange(1.0, 4.0, device="cuda").unsqueeze(1).repeat(1, 24)
    out = ops.dispatch(x, plan)
    assert out[:, 5].tolist() == [1, 1, 3, 0, 0, 0]
    assert ops.combine(out, plan)[:, 3].tolist() == [2, 0, 3]


def partial_plans(plan, keep):
    """Plans of which some places have given up their rows, by each way that there is."""
    fewer = torch.where(keep, plan.rows, -1)
    assigned = ops.ExpertPlan(plan.rows, plan.counts, plan.starts)
    assigned.rows = fewer
    replaced = ops.expert_plan(torch.where(plan.rows >= 0, 0, -1).int(), 1)
    replaced.rows, replaced.counts, replaced.starts = fewer, plan.counts, plan.starts
    changed = ops.expert_plan(torch.where(plan.rows >= 0, 0, -1).int(), 1)
    changed.rows.copy_(fewer)
    changed.starts = plan.starts
    return {"made": ops.ExpertPlan(fewer, plan.counts, plan.starts), "assigned": assigned, "replaced": replaced, "changed": changed}


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("width", [64, 66, 1451])
def test_rows_that_no_place_of_a_plan_has(device, dtype, width):
    """Tokens over an expert's capacity are dropped from a plan, which leaves rows among the others' that nobody has: zeros, and so are their gradients."""
    g = torch.Generator().manual_seed(1)
    tokens, k = 37, 3
    plan = ops.expert_plan(chosen_case(tokens, k, 5, device=device), 5)
    keep = (torch.rand(tokens, k, generator=g) < 0.6).to(device)
    x, dy = (torch.randn(tokens, width, generator=g).to(dtype).to(device) for _ in range(2))
    rows = torch.randn(tokens * k, width, generator=g).to(dtype).to(device).requires_grad_(True)
    w = torch.rand(tokens, k, generator=g).to(device)
    for how, fewer in partial_plans(plan, keep).items():
        kept = fewer.rows[fewer.rows >= 0].long()
        nobody = torch.ones(tokens * k, dtype=torch.bool, device=device)
        nobody[kept] = False
        soil(rows)
        out = ops.dispatch(x, fewer)
        assert torch.equal(out[kept], x[(fewer.rows >= 0).nonzero()[:, 0]]) and bool((out[nobody] == 0).all()), how
        y = ops.combine(rows, fewer, w)
        soil(rows)
        grad, = torch.autograd.grad(y, rows, dy)
        want = (w[fewer.rows >= 0].unsqueeze(-1) * dy[(fewer.rows >= 0).nonzero()[:, 0]].float()).to(dtype)
        assert torch.equal(grad[kept], want) and bool((grad[nobody] == 0).all()), how


@pytest.mark.parametrize("device", EACH)
def test_plans_can_be_copied(device):
    """Pickled, copied, and as they were pickled when they had three tensors and nothing else."""
    import copy
    import pickle
    plan = ops.expert_plan(chosen_case(9, 2, 4, device=device), 4)
    old = ops.ExpertPlan.__new__(ops.ExpertPlan)
    old.__setstate__((None, {"rows": plan.rows, "counts": plan.counts, "starts": plan.starts}))
    x = torch.randn(9, 16, generator=torch.Generator().manual_seed(2)).to(device)
    want = ops.dispatch(x, plan)
    for other in (pickle.loads(pickle.dumps(plan)), copy.copy(plan), copy.deepcopy(plan), old):
        assert torch.equal(ops.dispatch(x, other), want) and torch.equal(ops.combine(want, other), ops.combine(want, plan)) and other.num_experts == 4
        other.rows = torch.where(other.rows == 0, -1, other.rows)
        assert bool((ops.dispatch(x, other)[0] == 0).all()) and torch.equal(ops.dispatch(x, other)[1:], want[1:])


@gpu
def test_rows_that_nobody_has_while_a_mode_looks_on():
    plan = ops.expert_plan(chosen_case(20, 2, 5, device="cuda"), 5)
    fewer = ops.ExpertPlan(torch.where(torch.arange(40, device="cuda").view(20, 2) % 3 == 0, -1, plan.rows), plan.counts, plan.starts)
    x = torch.randn(20, 64, device="cuda")
    rows = torch.randn(40, 64, device="cuda", requires_grad=True)
    nobody = torch.ones(40, dtype=torch.bool, device="cuda")
    nobody[fewer.rows[fewer.rows >= 0].long()] = False
    soil(rows)
    with SeesDispatch():
        out = ops.dispatch(x, fewer)
        soil(rows)
        ops.combine(rows, fewer).sum().backward()
    assert bool((out[nobody] == 0).all()) and bool((rows.grad[nobody] == 0).all()) and bool((rows.grad[~nobody] == 1).all())


@pytest.mark.parametrize("device", EACH)
def test_exchange_refusals(device):
    plan = ops.expert_plan(torch.zeros(4, 2, dtype=torch.int32, device=device), 3)
    x, rows, w = torch.zeros(4, 8, device=device), torch.zeros(8, 8, device=device), torch.zeros(4, 2, device=device)
    for call, error in ((lambda: ops.dispatch(x[:3], plan), ValueError), (lambda: ops.dispatch(x.long(), plan), TypeError), (lambda: ops.dispatch(x, plan.rows), TypeError),
                        (lambda: ops.dispatch(x[:, :0], plan), ValueError), (lambda: ops.dispatch(x.view(2, 2, 8), plan), ValueError), (lambda: ops.combine(rows[:7], plan, w), ValueError),
                        (lambda: ops.combine(rows.view(4, 2, 8), plan, w), ValueError), (lambda: ops.combine(rows, plan, w[:, :1]), ValueError), (lambda: ops.combine(rows, plan, w.double()), TypeError),
                        (lambda: ops.combine(rows, None, w), TypeError), (lambda: ops.combine(rows.half(), plan, w.bfloat16()), TypeError),
                        (lambda: ops.combine(rows, ops.ExpertPlan(plan.rows.long(), plan.counts, plan.starts), w), TypeError)):
        with pytest.raises(error):
            call()
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.dispatch(x, ops.expert_plan(torch.zeros(4, 2, dtype=torch.int32), 3))
        with pytest.raises(ValueError):
            ops.combine(rows, plan, w.cpu())


# ---------------------------------------------------------------------------------------------- the experts' products

ACTS = [None, "silu", "gelu", "gelu_tanh"]


def act_of(v, name):
    if name is None:
        return v * 1.0
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))


def linear_case(counts, width, out, dtype, device, behind=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    n, experts = sum(counts) + behind, len(counts)
    x, dh = torch.randn(n, width, generator=g), torch.randn(n, out, generator=g)
    w = torch.randn(experts, out, width, generator=g) / math.sqrt(width)
    starts = torch.tensor([sum(counts[:e]) for e in range(experts + 1)], dtype=torch.int32)
    return [t.to(dtype).to(device) for t in (x, w, dh)] + [starts.to(device)]


def linear_check(x, w, dh, starts, act, h, grads):
    """fp32 sums of k products are off by 2^-24 of every partial sum at most: k 2^-24 of the sum of sizes. The rounding of the product's gradient goes through
    the products that take it."""
    dtype, u, F32 = h.dtype, half_step(h.dtype), 2.0 ** -20
    x, w, dh, h = (t.detach().double().cpu() for t in (x, w, dh, h))
    at = starts.tolist()
    want = torch.zeros_like(h)
    bound = torch.zeros_like(h)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    b_dx, b_dw = torch.zeros_like(x), torch.zeros_like(w)
    for e, (i, j) in enumerate(zip(at, at[1:])):
        if i == j:
            continue
        z = (x[i:j] @ w[e].t()).requires_grad_(True)
        size = x.shape[1] * 2.0 ** -24 * (x[i:j].abs() @ w[e].abs().t())
        a = act_of(z, act)
        slope, = torch.autograd.grad(a.sum(), z)
        a, z = a.detach(), z.detach()
        # |act'| is at most 1.13, |act''| at most 0.8; sixteen fp32 operations on the activation
        e_a = size if act is None else 1.13 * size + F32 * (a.abs() + z.abs())
        want[i:j], bound[i:j] = a, u * a.abs() + e_a
        if grads is None:
            continue
        dz = dh[i:j] * slope
        e_dz = 0 * dz if act is None else u * dz.abs() + dh[i:j].abs() * (0.8 * size + F32 * (1 + z.abs())) + torch.finfo(dtype).tiny * u
        dx[i:j], b_dx[i:j] = dz @ w[e], e_dz @ w[e].abs() + w.shape[1] * 2.0 ** -24 * (dz.abs() @ w[e].abs())
        dw[e], b_dw[e] = dz.t() @ x[i:j], e_dz.t() @ x[i:j].abs() + (j - i) * 2.0 ** -24 * (dz.abs().t() @ x[i:j].abs())
    check("h", h.to(dtype), want, bound)
    assert bool((h[at[-1]:] == 0).all())
    if grads is not None:
        check("dx", grads[0], dx, u * dx.abs() + b_dx)
        check("dw", grads[1], dw, u * dw.abs() + b_dw)
        assert bool((grads[0][at[-1]:] == 0).all())


def linear_run(counts, width, out, dtype, act="gelu", device="cuda", behind=0):
    x, w, dh, starts = linear_case(counts, width, out, dtype, device, behind)
    h = ops.expert_linear(x, w, starts, activation=act)
    x.requires_grad_(True)
    w.requires_grad_(True)
    h2 = ops.expert_linear(x, w, starts, activation=act)
    assert torch.equal(h, h2), "with and without a graph"
    linear_check(x, w, dh, starts, act, h, torch.autograd.grad(h2, (x, w), dh))


@pytest.mark.parametrize("act", ACTS)
def test_expert_linear_on_cpu(act):
    linear_run([3, 0, 5, 1], 12, 20, torch.float32, act, "cpu", behind=2)
    linear_run([0, 0], 4, 4, torch.float32, act, "cpu", behind=3)


COUNTS = [([1], 8, 8), ([1, 0, 2], 64, 64), ([16] * 4, 64, 128), ([0, 0, 1], 1, 1), ([5, 3, 17, 0, 2], 5, 7), ([128, 128], 128, 256), ([129, 127, 1], 72, 136), ([200, 0, 57], 1000, 384),
          ([63, 64, 65, 66], 333, 191), ([777], 264, 130), ([300, 5, 0, 0, 400], 65, 1033), ([1] * 40, 96, 72), ([0] * 63 + [70], 128, 64), ([2] * 300, 40, 24), ([0, 1] * 512, 16, 8),
          ([1500, 30], 512, 520), ([17, 31, 47, 15, 16], 2048, 264)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("sizes", COUNTS, ids=lambda s: "%dof%d-%dx%d" % (sum(s[0]), len(s[0]), s[1], s[2]))
def test_expert_linear_at_its_sizes(dtype, sizes):
    linear_run(*sizes, dtype, ACTS[sum(sizes[0]) % 4], behind=len(sizes[0]) % 3 * 70)


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_expert_linear_activations(act):
    linear_run([70, 10, 0, 133], 136, 200, torch.bfloat16, act, behind=5)
    linear_run([70, 10, 0, 133], 131, 203, torch.float16, act)


# Sums that are cut into parts, in each of the products: few tiles with a long k.
CUT = [([128], 2048, 128), ([100, 28], 2001, 100), ([128], 136, 2048), ([70, 0, 50], 99, 2050), ([3000], 128, 136), ([1500, 1, 1400], 130, 121), ([2500], 200, 72)]


@gpu
@pytest.mark.parametrize("sizes", CUT, ids=str)
def test_expert_linear_of_parts(sizes):
    linear_run(*sizes, torch.bfloat16 if sizes[1] % 2 else torch.float16, ACTS[len(sizes[0]) % 4], behind=len(sizes[0]) % 2 * 40)


def test_sizes_reach_every_kind_of_plan(tiles_program):
    seen = set()
    for counts, width, out in COUNTS + CUT + MANY:
        rows = str(sum(counts) + len(counts) % 3 * 70)
        for form, m, n, k in ((0, 0, out, width), (1, 0, width, out), (2, out, width, 0)):
            tall, columns, splits = subprocess.run([tiles_program, "plan", "148", str(form), rows, str(len(counts)), str(m), str(n), str(k)], capture_output=True, text=True,
                                                   check=True).stdout.split()
            seen.add((form, tall, columns, int(splits) > 1))
    assert seen >= {(0, "32", "64", False)} | {(f, "128", c, cut) for f in range(3) for c, cut in (("128", False), ("128", True), ("256", False))}, sorted(seen)
    assert seen >= {(f, "256", "256", False) for f in range(3)}, sorted(seen)


# Rows of tiles enough for columns of 256, in all three products, and more tiles than CTAs.
# (The last ones: pairs of CTAs, with sums that end inside a block, experts without rows and of a single one, odd widths; and few rows of many experts, which one CTA each takes.)
MANY = [([2000, 1300, 0, 1011], 776, 1544), ([700] * 8, 520, 1032), ([3000], 1288, 808), ([9, 5000], 72, 1800), ([130, 1, 269], 4350, 3327),
        ([131, 269, 0], 3328, 4352), ([4330], 512, 4864), ([1900, 1, 0, 2100, 3059], 510, 3833), ([100] * 140, 136, 250)]


@gpu
@pytest.mark.parametrize("counts,width,out", MANY, ids=str)
def test_expert_linear_of_many_tiles(counts, width, out):
    linear_run(counts, width, out, torch.bfloat16, "silu", behind=130)


@gpu
@pytest.mark.parametrize("counts,width,out", [([130, 1, 269], 4350, 3327), ([131, 269, 0], 3328, 4352), ([4330], 512, 4864)], ids=str)
def test_pairs_in_graphs_and_on_two_streams(counts, width, out):
    """Products of pairs of CTAs (forward, for the rows' gradient, for the weights'), captured and replayed on new values, and two at once: the bits of calls alone."""
    n, experts = sum(counts), len(counts)
    starts = torch.tensor([sum(counts[:e]) for e in range(experts + 1)], dtype=torch.int32, device="cuda")

    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        return [torch.randn(*size, generator=g, device="cuda").mul(scale).bfloat16() for size, scale in (((n, width), 1.0), ((experts, out, width), width ** -0.5), ((n, out), 1.0))]

    def step(x, w, dh):
        x, w = (t.detach().requires_grad_(True) for t in (x, w))
        h = ops.expert_linear(x, w, starts, activation="gelu")
        return (h.detach(), *torch.autograd.grad(h, (x, w), dh))

    states = [inputs(seed) for seed in range(3)]
    want = [step(*s) for s in states]
    torch.cuda.synchronize()
    still, stream = [t.clone() for t in states[0]], torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        got = step(*still)
    for s, wanted in zip(states, want):
        for t, v in zip(still, s):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wanted))
    streams, both = [stream, torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i, side in enumerate(streams):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                both[i] = step(*states[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(both[i], want[i]))


@gpu
def test_expert_linear_keeps_experts_apart():
    """NaN and infinities in one expert's rows and weights, and behind all rows, stay there."""
    counts, width, out = [20, 70, 33, 5], 72, 136
    x, w, dh, starts = linear_case(counts, width, out, torch.bfloat16, "cuda", behind=90)
    for t in (x, w):
        t.requires_grad_(True)

    def run():
        h = ops.expert_linear(x, w, starts, activation="gelu")
        return [h] + list(torch.autograd.grad(h, (x, w), dh))

    clean = run()
    with torch.no_grad():
        x[20:90], w[1], x[128:] = math.nan, math.inf, math.nan
        dh[128:] = math.inf
    dirty = run()
    for a, b in zip(clean[:2], dirty[:2]):
        assert torch.equal(a[:20], b[:20]) and torch.equal(a[90:], b[90:])
    assert torch.equal(clean[2][[0, 2, 3]], dirty[2][[0, 2, 3]]) and bool(dirty[0][20:90].isnan().all())


@gpu
def test_expert_linear_of_starts_that_are_none():
    """Numbers outside of the rows, and an end before its start: no expert has more rows than there are."""
    x, w, _, _ = linear_case([40, 40, 40], 64, 72, torch.bfloat16, "cuda")
    starts = torch.tensor([-5, 30, 1000, 2000], dtype=torch.int32, device="cuda")
    h = ops.expert_linear(x, w, starts)
    want = ops.expert_linear(x, w, torch.tensor([0, 30, 120, 120], dtype=torch.int32, device="cuda"))
    assert torch.equal(h, want)
    h = ops.expert_linear(x, w, torch.tensor([0, 50, 20, 120], dtype=torch.int32, device="cuda"))
    assert torch.equal(h[:20], ops.expert_linear(x, w, torch.tensor([0, 50, 50, 50], dtype=torch.int32, device="cuda"))[:20])


def soil(*like):
    """NaN in the memory that the next tensors of these sizes will get."""
    held = [torch.full_like(t, math.nan) for t in like for _ in range(4)]
    if any(t.is_cuda for t in like):
        torch.cuda.synchronize()
    del held


# Rows before the first start, experts and their rows, width, out: of every kind of tile, of sums in parts, and of more experts than the list of tiles holds one by one.
SOME = [(3, [5, 0, 17], 64, 72), (40, [1], 8, 8), (1, [129, 127, 1], 72, 136), (300, [63, 64, 65], 333, 191), (513, [700] * 3, 520, 1032), (200, [131, 269, 0], 3328, 4352), (128, [128], 2048, 128),
        (77, [70, 0, 50], 99, 2050), (900, [1500], 130, 121), (9, [2] * 300, 40, 24), (130, [100] * 140, 136, 250), (50, [0, 0], 24, 40), (7, [0] * 200, 16, 8)]


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("before,counts,width,out", SOME, ids=lambda v: str(v) if isinstance(v, int) else "%dof%d" % (sum(v), len(v)))
def test_expert_linear_of_some_of_the_experts(device, before, counts, width, out):
    """The weights of some experts and where their rows start: rows before the first start are nobody's, as those behind the last end are."""
    if device == "cpu" and width * out > 1 << 18:
        pytest.skip("sizes of the kernels")
    dtype = torch.float32 if device == "cpu" else torch.bfloat16 if before % 2 else torch.float16
    x, w, dh, starts = linear_case([before] + counts, width, out, dtype, device, behind=len(counts) % 3 * 35)
    w, starts = w[1:].contiguous().requires_grad_(True), starts[1:]
    x.requires_grad_(True)
    for act in ("gelu", None):
        soil(dh)
        with torch.no_grad():
            h = ops.expert_linear(x, w, starts, activation=act)
        soil(dh, x, w)
        h2 = ops.expert_linear(x, w, starts, activation=act)
        assert torch.equal(h, h2)
        soil(dh, x, w)
        grads = torch.autograd.grad(h2, (x, w), dh)
        linear_check(x, w, dh, starts, act, h, grads)
        assert bool((h[:before] == 0).all()) and bool((grads[0][:before] == 0).all())


@pytest.mark.parametrize("device", EACH)
def test_expert_linear_by_a_part_of_a_plan(device):
    """Slices of weights and of a plan's starts: the rows that the whole product has there, and zeros."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    plan = ops.expert_plan(chosen_case(90, 2, 8, device=device), 8)
    x, w, dh, _ = linear_case([180] + [0] * 7, 64, 72, dtype, device)
    whole, starts = ops.expert_linear(x, w, plan, activation="silu"), plan.starts.tolist()
    for i, j in ((0, 8), (2, 5), (7, 8), (1, 2)):
        soil(dh)
        part = ops.expert_linear(x, w[i:j], plan.starts[i:j + 1], activation="silu")
        assert torch.equal(part[starts[i]:starts[j]], whole[starts[i]:starts[j]])
        assert bool((part[:starts[i]] == 0).all()) and bool((part[starts[j]:] == 0).all())


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("starts", [[0, 50, 20, 120], [40, 90, 10, 30], [-5, 70, 130, 60], [120, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 90], [0, 119, 118, 117]], ids=str)
@pytest.mark.parametrize("act", [None, "gelu"])
def test_expert_linear_of_starts_that_go_back(device, starts, act):
    """A start that lies before one ahead of it counts as that one: no row is of two experts, and every row is stored."""
    x, w, dh, _ = linear_case([40, 40, 40], 64, 72, torch.float32 if device == "cpu" else torch.bfloat16, device)
    go_back_check(x, w, dh, starts, act)


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("experts,tokens,width,out", [(11, 700, 72, 136), (119, 900, 24, 40), (120, 900, 24, 40), (300, 1500, 40, 24), (1024, 3000, 16, 8), (4, 6000, 520, 1032)])
def test_expert_linear_of_many_starts_that_go_back(device, experts, tokens, width, out):
    if device == "cpu" and tokens > 900:
        pytest.skip("sizes of the kernels")
    g = torch.Generator().manual_seed(experts)
    x, w, dh, _ = linear_case([tokens] + [0] * (experts - 1), width, out, torch.float32 if device == "cpu" else torch.float16, device)
    for table in range(2):
        starts = torch.randint(0, tokens + 1, (experts + 1,), generator=g).sort().values
        some = torch.rand(experts + 1, generator=g) < 0.1
        starts = torch.where(some, torch.randint(-tokens, starts[-1].item() if table else tokens + 1, (experts + 1,), generator=g), starts)
        go_back_check(x, w, dh, starts.tolist(), "silu")


def go_back_check(x, w, dh, starts, act):
    table, want, reached = torch.tensor(starts, dtype=torch.int32, device=x.device), [], 0
    for s in starts:
        reached = max(reached, min(max(s, 0), x.shape[0]))
        want.append(reached)
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    runs = []
    for _ in range(2):
        soil(dh, x, w)
        h = ops.expert_linear(*leaves, table, activation=act)
        soil(dh, x, w)
        runs.append((h.detach(), *torch.autograd.grad(h, leaves, dh)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    linear_check(x, w, dh, torch.tensor(want), act, runs[0][0], runs[0][1:])
    assert bool((runs[0][0][:want[0]] == 0).all()) and bool((runs[0][1][:want[0]] == 0).all())


@gpu
def test_expert_linear_of_views():
    x, w, dh, starts = linear_case([20, 0, 13], 128, 96, torch.bfloat16, "cuda")
    want = ops.expert_linear(x, w, starts)
    assert torch.equal(ops.expert_linear(x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), starts), want)
    wide = torch.zeros(33, 300, device="cuda").bfloat16()
    wide[:, 101:229] = x
    assert torch.equal(ops.expert_linear(wide[:, 101:229], w, starts), want)
    off = torch.zeros(33 * 128 + 3, device="cuda").bfloat16()[3:].view(33, 128).copy_(x)
    linear_check(off, w, dh, starts, None, ops.expert_linear(off, w, starts), None)
    shared = w[:1].clone().requires_grad_(True)
    each = shared.detach().repeat(3, 1, 1).requires_grad_(True)
    one, = torch.autograd.grad(ops.expert_linear(x, shared.expand(3, 96, 128), starts), shared, dh)
    three, = torch.autograd.grad(ops.expert_linear(x, each, starts), each, dh)
    assert torch.equal(one[0], three.sum(0))


@gpu
def test_expert_linear_gradients_of_some_inputs():
    x, w, dh, starts = linear_case([30, 7], 64, 72, torch.bfloat16, "cuda")
    both = [t.clone().requires_grad_(True) for t in (x, w)]
    want = torch.autograd.grad(ops.expert_linear(both[0], both[1], starts, activation="silu"), both, dh)
    assert torch.equal(torch.autograd.grad(ops.expert_linear(both[0], w, starts, activation="silu"), both[0], dh)[0], want[0])
    assert torch.equal(torch.autograd.grad(ops.expert_linear(x, both[1], starts, activation="silu"), both[1], dh)[0], want[1])


@gpu
def test_expert_linear_without_rows():
    x, w, _, starts = linear_case([0, 0], 64, 72, torch.bfloat16, "cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    h = ops.expert_linear(x, w, starts, activation="gelu")
    h.sum().backward()
    assert h.shape == (0, 72) and x.grad.shape == (0, 64) and bool((w.grad == 0).all())
    linear_run([0, 0, 0], 64, 72, torch.bfloat16, "gelu", behind=200)


@gpu
def test_expert_linear_gradient_against_differences():
    x, w, dh, starts = linear_case([9, 0, 14], 64, 48, torch.float16, "cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    grads = torch.autograd.grad(ops.expert_linear(x, w, starts, activation="gelu"), (x, w), dh)
    for i, (v, g) in enumerate(zip((x, w), grads)):
        way = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).cuda().half()
        h = 2.0 ** -5
        with torch.no_grad():
            up, down = (ops.expert_linear(*((v + s * h * way, w) if i == 0 else (x, v + s * h * way)), starts, activation="gelu") for s in (1, -1))
        want, got = ((up.double() - down.double()) * dh.double()).sum() / (2 * h), (g.double() * way.double()).sum()
        # 23 x 48 results of about 1, each rounded to 2^-11 of itself and so moved at random, over 2 h; inputs rounded to 2^-11 of h's way likewise. A product moves by m h,
        # m = |w . way| = 1 of unit rows of w, or |x . way| = sqrt(64) = 8, so that gelu's third derivative (below 1) leaves m^3 h^2 / 6 of each result, of either sign.
        m = (1, 8)[i]
        assert abs(want - got) <= 6 * math.sqrt(23 * 48) * (2.0 ** -11 / h + max(m ** 3 / 6, 1) * h * h), (i, want, got)


@pytest.mark.parametrize("device", EACH)
def test_expert_linear_refusals(device):
    half = torch.float16 if device == "cuda" else torch.float32
    x, w, s = torch.zeros(4, 8, device=device, dtype=half), torch.zeros(2, 6, 8, device=device, dtype=half), torch.tensor([0, 1, 4], dtype=torch.int32, device=device)
    for args, error in (((x[0], w, s), ValueError), ((x, w[0], s), TypeError), ((x, w, s[:2]), ValueError), ((x, w, s.long()), TypeError), ((x[:, :7], w, s), ValueError),
                        ((x, w.double(), s), TypeError), ((x, w, None), ValueError), ((x, w[:0], s[:1]), ValueError), ((x, w[:, :0], s), ValueError), ((x.long(), w, s), TypeError)):
        with pytest.raises(error):
            ops.expert_linear(*args)
    for act in ("relu", 3, ["silu"]):
        with pytest.raises(ValueError):
            ops.expert_linear(x, w, s, activation=act)
    if device == "cuda":
        with pytest.raises(TypeError):
            ops.expert_linear(x.float(), w.float(), s)
        with pytest.raises(ValueError):
            ops.expert_linear(x, w, s.cpu())


# ---------------------------------------------------------------------------------------------- together

def layer(x, router, w_in, w_out, k, bias=None):
    weights, experts = ops.route(x @ router.t(), k, "sigmoid", bias, groups=2, top_groups=1)
    plan = ops.expert_plan(experts, router.shape[0])
    h = ops.expert_linear(ops.dispatch(x, plan), w_in, plan, activation="gelu")
    return ops.combine(ops.expert_linear(h, w_out, plan), plan, weights)


def layer_case(tokens, width, hidden, experts, dtype, device):
    g = torch.Generator().manual_seed(11)
    make = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1]))  # noqa: E731
    return [t.to(dtype).to(device) for t in (torch.randn(tokens, width, generator=g), make(experts, width) * 2, make(experts, hidden, width), make(experts, width, hidden))]


@pytest.mark.parametrize("device", EACH)
def test_a_layer_of_all_operators(device):
    """Against every token's experts one by one, in 64 bits. bf16: h and the experts' results are rounded between the operators, and so are their gradients."""
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    x, router, w_in, w_out = (t.requires_grad_(True) for t in layer_case(60, 72, 40, 8, dtype, device))
    bias = bias_of(8, device, 0.02)
    y = layer(x, router, w_in, w_out, 3, bias)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dtype).to(device)
    grads = torch.autograd.grad(y, (x, router, w_in, w_out), dy)
    d = [t.detach().double().requires_grad_(True) for t in (x, router, w_in, w_out)]
    logits = (d[0] @ d[1].t()) + ((x @ router.t()).double() - d[0] @ d[1].t()).detach()       # the logits that the operators saw
    weights, experts = route_reference(logits, 3, "sigmoid", bias, 2, 1, "max", True, 1.0)
    want = torch.stack([sum(weights[t, j] * (act_of(d[0][t] @ d[2][e].t(), "gelu") @ d[3][e].t()) for j, e in enumerate(experts[t].tolist())) for t in range(60)])
    want_grads = torch.autograd.grad(want, d, dy.double())
    # five roundings in a row, or 2^-18 for the whole chain in fp32, of the largest value
    for a, b in zip([y] + list(grads), [want] + list(want_grads)):
        assert (a.double() - b).abs().max() <= (5 * half_step(dtype) + 2.0 ** -18) * b.abs().max()


def test_a_layer_on_cpu_while_another_device_is_the_default():
    case = [t.requires_grad_(True) for t in layer_case(9, 12, 8, 4, torch.float32, "cpu")]
    want = layer(*case, 2)
    grads = torch.autograd.grad(want.sum(), case)
    with torch.device("meta"):
        got = layer(*case, 2)
        again = torch.autograd.grad(got.sum(), case)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(again, grads))


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements of rows, results and saved products: the last rows are what they are alone."""
    tokens, width = 300_001, 1024
    experts = torch.full((tokens, 8), 1, dtype=torch.int32, device="cuda")
    experts[-3:] = torch.tensor([2, 1, 0, 2, 2, 1, 0, 0], dtype=torch.int32, device="cuda")
    plan = ops.expert_plan(experts, 3)
    x = torch.zeros(tokens, width, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, width, device="cuda").bfloat16()
    rows = ops.dispatch(x, plan)
    assert rows.numel() > 2 ** 31 and torch.equal(rows[-9:], x[-3:].repeat_interleave(3, 0)[:9])
    w = torch.rand(tokens, 8, device="cuda")
    y = ops.combine(rows, plan, w)
    want = (x[-3:].double() * w[-3:].double().sum(-1, keepdim=True))
    check("y", y[-3:], want, half_step(torch.bfloat16) * want.abs() + 9 * 2.0 ** -24 * want.abs())
    rows.requires_grad_(True)
    dy = torch.zeros_like(y)
    dy[-1] = 1.0
    drows, = torch.autograd.grad(ops.combine(rows, plan, w), rows, dy)
    got = drows[plan.rows[-1].long()]
    assert bool((got == w[-1].bfloat16().unsqueeze(-1)).all()) and drows[-9:].count_nonzero() == 3 * width       # of the last token's three rows of expert 2
    del rows, drows, dy, y, x, plan, experts
    n, out = 530_000, 4104
    x = torch.zeros(n, 64, device="cuda", dtype=torch.bfloat16)
    x[-200:] = torch.randn(200, 64, device="cuda").bfloat16()
    weight = torch.randn(2, out, 64, device="cuda").bfloat16() / 8
    starts = torch.tensor([0, n - 130, n - 5], dtype=torch.int32, device="cuda")
    few = torch.tensor([0, 70, 195], dtype=torch.int32, device="cuda")
    mine, alone = x.clone().requires_grad_(True), x[-200:].clone().requires_grad_(True)
    h, g = ops.expert_linear(mine, weight, starts, activation="silu"), ops.expert_linear(alone, weight, few, activation="silu")
    assert h.numel() > 2 ** 31
    # k is not cut in either, and one block of it: the same sums
    assert torch.equal(h[-200:], g)
    dh = torch.zeros_like(h)
    dh[-200:] = torch.randn(200, out, device="cuda").bfloat16()
    big, = torch.autograd.grad(h, mine, dh)
    small, = torch.autograd.grad(g, alone, dh[-200:])
    size = torch.zeros(200, 64, dtype=torch.float64, device="cuda")
    for i, j, e in ((0, 70, 0), (70, 195, 1)):
        size[i:j] = dh[-200:][i:j].double().abs() @ weight[e].double().abs() * 1.13
    check("dx", big[-200:], small.double(), 2 * half_step(torch.bfloat16) * small.double().abs() + out * 2.0 ** -23 * size)
    assert big[:-200].count_nonzero() == 0


@gpu
def test_compiled_functions_stay_right():
    """The compiler leaves the operators out of its graphs and calls them between."""
    case = [t.requires_grad_(True) for t in layer_case(33, 64, 72, 8, torch.bfloat16, "cuda")]
    want = layer(*case, 2)
    grads = torch.autograd.grad(want.sum(), case)
    compiled = torch.compile(layer, backend="eager")
    for _ in range(2):
        got = compiled(*case, 2)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got.sum(), case), grads))


@gpu
def test_a_layer_in_graphs():
    """Captured twice on one stream, replayed with other tokens; forward alone, and with its backward pass."""
    with torch.no_grad():
        x, router, w_in, w_out = layer_case(5, 64, 72, 8, torch.bfloat16, "cuda")
    train = [t.clone().requires_grad_(True) for t in (x, router, w_in, w_out)]
    dy = torch.randn(5, 64, device="cuda").bfloat16()

    def decode():
        with torch.no_grad():
            return [layer(x, router, w_in, w_out, 2)]

    def step():
        y = layer(*train, 2)
        return [y] + list(torch.autograd.grad(y, train, dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        decode(), step()
    torch.cuda.synchronize()
    for f in (decode, decode, step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = f()
        graphs.append((f, graph, [o.detach() for o in outs]))
        del outs
    for seed in range(3):
        new = torch.randn(5, 64, generator=torch.Generator().manual_seed(seed)).bfloat16()
        x.copy_(new)
        train[0].data.copy_(new)
        for f, graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, f()))


FIRST = """
import torch
from dccl_b200 import ops
x, r, a, b = (torch.randn(s, device="cuda").bfloat16() for s in ((200, 128), (16, 128), (16, 64, 128), (16, 128, 64)))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
logits = x @ r.t()
def step():
    w, e = ops.route(logits, 3)
    p = ops.expert_plan(e, 16)
    y = ops.combine(ops.expert_linear(ops.expert_linear(ops.dispatch(x, p), a, p, activation="silu"), b, p), p, w)
    return y, ops.grad_norm([y, x]), ops.clip_grad_norm([y], 1.0, out=[torch.empty_like(y)])
with torch.cuda.graph(graph):
    outs = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, step()))
print("OK")
"""


@gpu
@pytest.mark.parametrize("experts", [8, 200])
def test_dropped_places_and_some_of_the_experts_in_graphs(experts):
    """Places over a capacity dropped from the plan, the products of some experts, and a table that goes back: captured forward and backward, replayed on other tokens, and on
    two streams at once."""
    tokens, width, out, capacity = 300, 64, 72, 2 * 600 // experts
    g = torch.Generator().manual_seed(experts)
    w = (torch.randn(experts, out, width, generator=g) / 8).bfloat16().cuda().requires_grad_(True)
    dy, dh = (torch.randn(n, out, generator=g).bfloat16().cuda() for n in (tokens, 2 * tokens))
    back = torch.tensor([0, 400, 100] + [100 + 2 * e for e in range(experts - 2)], dtype=torch.int32, device="cuda")

    def step(x, chosen, weights):
        plan = ops.expert_plan(chosen, experts)
        place = plan.rows - plan.starts[chosen.long()]
        fewer = ops.ExpertPlan(torch.where(place < capacity, plan.rows, -1), plan.counts, plan.starts)
        leaf = x.detach().requires_grad_(True)
        rows = ops.dispatch(leaf, fewer)
        h = ops.expert_linear(rows, w, plan, activation="silu")
        y = ops.combine(h, fewer, weights)
        part = ops.expert_linear(rows, w[2:5], plan.starts[2:6])
        odd = ops.expert_linear(rows, w, back, activation="gelu")
        return [t.detach() for t in (rows, h, y, part, odd)] + list(torch.autograd.grad((y, part, odd), (leaf, w), (dy, dh, dh)))

    cases = [(torch.randn(tokens, width, generator=g).bfloat16().cuda(), torch.randint(0, experts, (tokens, 2), generator=g).int().cuda(), torch.rand(tokens, 2, generator=g).cuda())
             for _ in range(3)]
    wants = []
    for c in cases:
        soil(cases[0][0], dh, w)
        wants.append(step(*c))
    assert all(bool(t.isfinite().all()) for want in wants for t in want)
    still, stream, graph = [t.clone() for t in cases[0]], torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step(*still)
    for c, want in zip(cases, wants):
        for t, v in zip(still, c):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams, both = [stream, torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i, side in enumerate(streams):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                both[i] = step(*cases[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(both[i], wants[i]))


@gpu
def test_the_first_call_of_a_process_can_be_captured():
    res = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout + res.stderr[-2000:]


THREADS = """
import threading, torch
from dccl_b200 import ops
x, w, starts = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(2, 72, 64, device="cuda").bfloat16(), torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")
w.requires_grad_(True)
y, room = ops.expert_linear(x, w, starts), [torch.empty(1 << 20, device="cuda") for _ in range(4)]
del room
torch.cuda.synchronize()
g, = torch.autograd.grad(y, w, torch.ones_like(y))          # the autograd engine's thread
got = []
def call():
    got.append(ops.expert_linear(x, w, starts))
    got.append(ops.gated_linear(x, w[0], w[1]))
thread = threading.Thread(target=call)
thread.start()
thread.join()
assert torch.equal(got[0], y) and torch.equal(got[1], ops.gated_linear(x, w[0], w[1])) and bool((g != 0).any())
print("OK")
"""


@gpu
def test_the_first_call_of_a_thread():
    """Threads that have not called CUDA before: the one that runs backward passes, and one of the user's."""
    res = subprocess.run([sys.executable, "-c", THREADS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout + res.stderr[-2000:]


@gpu
def test_operators_of_two_streams_at_once():
    x, router, w_in, w_out = layer_case(700, 256, 328, 16, torch.bfloat16, "cuda")
    want = layer(x, router, w_in, w_out, 4)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(15):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(layer(x, router, w_in, w_out, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for o in outs for v in o)


@gpu
def test_operators_on_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    case = [t.requires_grad_(True) for t in layer_case(70, 64, 72, 8, torch.bfloat16, "cuda:1")]
    y = layer(*case, 2)
    grads = torch.autograd.grad(y.sum(), case)
    with torch.cuda.device(1):
        again = layer(*case, 2)
        assert torch.equal(y, again) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again.sum(), case)))
    assert torch.cuda.current_device() == 0


@gpu
def test_the_same_bits_twice():
    case = [t.requires_grad_(True) for t in layer_case(900, 200, 264, 12, torch.bfloat16, "cuda")]
    runs = []
    for _ in range(3):
        y = layer(*case, 3)
        runs.append([y] + list(torch.autograd.grad(y.sum(), case)))
    assert all(torch.equal(a, b) for other in runs[1:] for a, b in zip(runs[0], other))


def calls(device="cuda"):
    """Each differentiable operator as a function of one tensor, and that tensor."""
    g = torch.Generator().manual_seed(4)
    plan = ops.expert_plan(chosen_case(9, 2, 4, dropped=0.1, device=device), 4)
    w = torch.rand(9, 2, generator=g).to(device)
    weight = torch.randn(4, 40, 64, generator=g).to(device).bfloat16()
    x = torch.randn(9, 64, generator=g).to(device).bfloat16()
    rows = torch.randn(18, 64, generator=g).to(device).bfloat16()
    return [(lambda v: ops.route(v, 3, bias=torch.zeros(64, device=device))[0], x), (lambda v: ops.dispatch(v, plan), x), (lambda v: ops.combine(v, plan, w), rows),
            (lambda v: ops.expert_linear(v, weight, plan, activation="silu"), rows)]


@gpu
def test_autograd_of_the_operators():
    """retain_graph, a second pass over a freed graph, inputs changed in place, gradients of gradients, forward mode, inference mode."""
    for make, x in calls():
        x = x.clone().requires_grad_(True)
        y = make(x)
        first, = torch.autograd.grad(y.sum(), x, retain_graph=True)
        again, = torch.autograd.grad(y.sum(), x)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.sum(), x)
        g, = torch.autograd.grad(make(x).float().pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises((NotImplementedError, RuntimeError)):
                make(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))
        with torch.inference_mode():
            assert torch.equal(make(x), make(x.detach()))
        assert torch.equal(make(torch._neg_view(x.detach())), make(-x.detach()))
    for make, x in calls()[::3]:        # those that keep their input
        z = x.clone().requires_grad_(True) * 1
        y = make(z)
        z.add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


@gpu
def test_checkpointed_operators():
    from torch.utils.checkpoint import checkpoint
    case = [t.requires_grad_(True) for t in layer_case(40, 65, 72, 8, torch.bfloat16, "cuda")]
    want = torch.autograd.grad(layer(*case, 2).sum(), case)
    got = torch.autograd.grad(checkpoint(layer, *case, 2, use_reentrant=False).sum(), case)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # what is saved may come back from elsewhere in memory
    def unpack(t):
        return torch.cat([t.new_zeros(1).expand(1), t.reshape(-1)])[1:].view(t.shape) if t.numel() else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        y = layer(*case, 2)
    for a, b in zip(torch.autograd.grad(y.sum(), case), want):
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -7 * b.double().abs().max()


@gpu
def test_operators_refuse_tensors_without_memory():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        with pytest.raises(TypeError):
            ops.route(torch.empty(4, 64, device="cuda"), 2)
        with pytest.raises(TypeError):
            ops.expert_plan(torch.empty(4, 2, device="cuda", dtype=torch.int32), 2)
    del mode
    with pytest.raises((TypeError, RuntimeError)):
        torch.func.vmap(lambda v: ops.route(v, 2)[0])(torch.zeros(3, 4, 8, device="cuda"))


class SeesDispatch(torch.utils._python_dispatch.TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


class SeesFunctions(torch.overrides.TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@gpu
@pytest.mark.parametrize("mode", [SeesDispatch, SeesFunctions])
def test_an_active_mode_sees_the_operators(mode):
    case = [t.requires_grad_(True) for t in layer_case(33, 64, 72, 8, torch.bfloat16, "cuda")]

    def step():
        y = layer(*case, 2, bias_of(8, "cuda"))
        return [y] + list(torch.autograd.grad(y.sum(), case))

    want = step()
    with mode() as m:
        got = step()
    seen = " ".join(m.seen)
    for name in ("route", "expert_plan", "dispatch", "expert_linear", "combine"):
        assert "dccl." + name in seen and (mode is SeesFunctions or name == "expert_plan" or "dccl.%s_backward" % name in seen), (name, m.seen)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("tracer", ["trace", "make_fx"])
def test_tracers_record_the_operators(tracer):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, router, w_in, w_out = layer_case(33, 64, 72, 8, torch.bfloat16, "cuda")
    f, other = lambda v: layer(v, router, w_in, w_out, 2), torch.randn(33, 64, device="cuda").bfloat16()  # noqa: E731
    with torch.no_grad():
        recorded = torch.jit.trace(f, (x,)) if tracer == "trace" else make_fx(f)(x)
        assert torch.equal(recorded(other), f(other))


@gpu
def test_subclasses_of_tensor_see_the_operators():
    class Sees(torch.Tensor):
        seen = []

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.seen.append(str(func))
            return super().__torch_function__(func, types, args, kwargs or {})

    for make, x in calls():
        want = make(x)
        got = make(x.as_subclass(Sees))
        assert type(got) is Sees and torch.equal(got.as_subclass(torch.Tensor), want)
    assert all(any("dccl.%s" % name in s for s in Sees.seen) for name in ("route", "dispatch", "combine", "expert_linear"))


# ---------------------------------------------------------------------------------------------- the expert-parallel layer

@pytest.mark.parametrize("world", [1, 4])
def test_the_fused_expert_parallel_layer(dccl_lib, world):
    from dccl_b200.utils.launch import python_ranks
    res = python_ranks(os.path.join(ROOT, "tests", "workers", "moe_fused_worker.py"), [], world, timeout=300)
    for r, p in enumerate(res):
        assert p.returncode == 0, "rank %d:\n%s\n%s" % (r, p.stdout[-3000:], p.stderr[-3000:])
        assert p.stdout.strip().splitlines()[-1].startswith("OK"), p.stdout


def test_the_plain_layer_takes_no_options_of_the_fused_one(dccl_lib):
    from dccl_b200 import Communicator
    from dccl_b200.parallel.expert_parallel import ExpertParallelMLP
    comm = Communicator(rank=0, world=1)
    try:
        for kw in ({"top_k": 2}, {"routing": {}}):
            with pytest.raises(ValueError):
                ExpertParallelMLP(8, 8, 4, comm, **kw)
    finally:
        comm.finalize()


@pytest.mark.parametrize("device", EACH)
def test_the_routing_bias_goes_with_the_layer(dccl_lib, device):
    """To other devices, where it stays fp32, and into state dicts: it holds how the load has been balanced."""
    import copy
    from dccl_b200 import Communicator
    from dccl_b200.parallel.expert_parallel import ExpertParallelMLP
    comm = Communicator(rank=0, world=1, **({"device": 0} if device == "cuda" else {}))
    try:
        def layer(bias, **kw):
            return ExpertParallelMLP(16, 24, 4, comm, fused=True, top_k=2, routing=dict(scores="sigmoid", **({} if bias is None else {"bias": bias})), **kw)

        bias = torch.tensor([0.5, -0.25, 3.0, 0.0])
        a, b = layer(bias.clone()), layer(torch.zeros(4))
        mine = a.routing["bias"]
        assert a.to("cpu").routing["bias"] is mine and a.double().float().routing["bias"] is mine       # whoever balances the load may keep it
        type_ = torch.bfloat16 if device == "cuda" else torch.float32
        a, b = a.to(device).to(type_), b.to(device).to(type_)
        assert a.routing["bias"].dtype is torch.float32 and a.routing["bias"].device.type == device and torch.equal(a.routing["bias"].cpu(), bias)
        state = copy.deepcopy(a.state_dict())
        assert torch.equal(state["routing_bias"].cpu(), bias)
        held = b.routing["bias"]
        assert all(hasattr(b, name) for name in state)
        b.load_state_dict(state)
        assert b.routing["bias"] is held and torch.equal(held.cpu(), bias)
        x = torch.randn(9, 16, generator=torch.Generator().manual_seed(0)).to(device).to(type_)
        assert torch.equal(a(x), b(x))
        held.add_(1.0)
        del state["routing_bias"]           # of a layer that had none
        b.load_state_dict(state)
        assert torch.equal(held.cpu(), bias + 1.0)
        ExpertParallelMLP(16, 24, 4, comm).load_state_dict(a.state_dict())          # the plain layer has no use for it
        with pytest.raises(RuntimeError):
            layer(None).load_state_dict(a.state_dict())
        state = a.state_dict()
        state["routing_bias"] = torch.zeros(5)
        with pytest.raises(RuntimeError, match="routing_bias"):
            b.load_state_dict(state)
    finally:
        comm.finalize()


def test_a_layer_loads_no_part_of_other_experts(dccl_lib):
    """The weights of more experts than the layer has, or fewer, in one tensor or in a list, are refused in either form."""
    from dccl_b200 import Communicator
    from dccl_b200.parallel.expert_parallel import ExpertParallelMLP
    comm = Communicator(rank=0, world=1)
    try:
        for other in (2, 6):
            for had in (True, False):
                state = ExpertParallelMLP(8, 12, other, comm, seed=1, fused=had).state_dict()
                for fused in (True, False):
                    layer = ExpertParallelMLP(8, 12, 4, comm, fused=fused)
                    state["router"] = layer.router.detach().clone()
                    with pytest.raises(RuntimeError):
                        layer.load_state_dict(state)
    finally:
        comm.finalize()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_the_fused_layer_on_the_gpu(dccl_lib, dtype):
    """One rank: against the layer that is not fused. Both round h, the experts' results and their weighted ones to bf16, the plain one its gates as well: four half
    steps, and as many for the gradients again; fp32 is off by sums in other orders."""
    from dccl_b200 import Communicator
    from dccl_b200.parallel.expert_parallel import ExpertParallelMLP
    comm = Communicator(rank=0, world=1, device=0)
    try:
        plain = ExpertParallelMLP(64, 72, 8, comm, dtype=dtype, device="cuda")
        fused = ExpertParallelMLP(64, 72, 8, comm, dtype=dtype, device="cuda", fused=True)
        fused.load_state_dict(plain.state_dict())
        x = torch.randn(50, 64, device="cuda").to(dtype)
        a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
        ya, yb = plain(a), fused(b)
        dy = torch.randn_like(ya)
        ya.backward(dy)
        yb.backward(dy)
        u = half_step(dtype) if dtype is torch.bfloat16 else 2.0 ** -18
        pairs = [(ya, yb), (a.grad, b.grad), (plain.router.grad, fused.router.grad)]
        pairs += [(p[j].grad, f.grad[j]) for p, f in ((plain.w_in, fused.w_in), (plain.w_out, fused.w_out)) for j in range(8) if p[j].grad is not None]
        for p, f in pairs:
            assert (p.double() - f.double()).abs().max() <= 16 * u * p.double().abs().max()
        if dtype is torch.bfloat16:
            graph, still = torch.cuda.CUDAGraph(), x.clone()
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.no_grad(), torch.cuda.graph(graph, stream=stream):
                out = fused(still)
            still.copy_(torch.randn_like(still))
            graph.replay()
            torch.cuda.synchronize()
            with torch.no_grad():
                assert torch.equal(out, fused(still))
    finally:
        comm.finalize()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_the_fused_layer_under_autocast(dccl_lib, dtype):
    """fp32 parameters, multiplied in 16 bits: what comes out has the types of the plain layer. Both round the tokens, the weights, h and the experts' results; the plain one
    what the activation takes as well, and the gradients of all of those: as in the test above."""
    from dccl_b200 import Communicator
    from dccl_b200.parallel.expert_parallel import ExpertParallelMLP
    comm = Communicator(rank=0, world=1, device=0)
    try:
        plain = ExpertParallelMLP(64, 72, 8, comm, device="cuda")
        fused = ExpertParallelMLP(64, 72, 8, comm, device="cuda", fused=True)
        fused.load_state_dict(plain.state_dict())
        x = torch.randn(50, 64, generator=torch.Generator().manual_seed(3)).cuda()
        a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=dtype):
            ya, yb = plain(a), fused(b)
        assert yb.dtype is ya.dtype
        dy = torch.randn_like(ya)
        ya.backward(dy)
        yb.backward(dy)
        pairs = [(ya, yb), (a.grad, b.grad), (plain.router.grad, fused.router.grad)]
        pairs += [(p[j].grad, f.grad[j]) for p, f in ((plain.w_in, fused.w_in), (plain.w_out, fused.w_out)) for j in range(8) if p[j].grad is not None]
        for p, f in pairs:
            assert p.dtype is f.dtype and (p.double() - f.double()).abs().max() <= 16 * half_step(dtype) * p.double().abs().max()
    finally:
        comm.finalize()
