"""The operators of a decoder block (dccl_b200.ops.decoder) against their formulas in 64 bits.

Tolerances count roundings. A result of type T is off by half a step of T, u = eps / 2 of its size; what is computed in fp32 before
that is off by a few times 2^-24 of the terms that went into it. Where a value is rounded to T on the way, its u goes through
the formula as well: each bound below says how.
"""
import math

import pytest

torch = pytest.importorskip("torch")
import torch.utils._python_dispatch  # noqa: E402

from dccl_b200 import ops  # noqa: E402

EPS = 1e-5
F32 = 2.0 ** -20      # of the sum of a result's terms: up to sixteen fp32 operations on each
SUMS = 2.0 ** -17     # of the sum of a column's terms: up to a hundred more additions in a row
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(name, got, want, bound):
    assert got.shape == want.shape, name
    # below the smallest normal number (6e-5 of float16) the steps get no smaller: half of one is tiny * eps / 2, 2^-25 of float16
    bound = bound + torch.finfo(got.dtype).tiny * half_step(got.dtype)
    got = got.detach().double().cpu()
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), "%s: %.3g over its bound %.3g at %s (%.6g, not %.6g)" % (
        name, off.max(), bound.reshape(-1)[off.argmax()], off.argmax().item(), got.reshape(-1)[off.argmax()], want.reshape(-1)[off.argmax()])


def test_early_launched_kernels_promise_nothing_about_their_inputs():
    """As tests/test_local_calls.py asks of the kernels that it knows: they are launched before the one ahead of them has written, so every one
    waits, and none declares what it reads read-only for as long as it runs."""
    import os
    folder, found = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "decoder"), set()
    for name in sorted(os.listdir(folder)):
        text = open(os.path.join(folder, name)).read()
        assert "__restrict__" not in text and "__ldg" not in text, name
        for part in text.split("__global__")[1:]:
            signature, body = part.split("{", 1)
            kernel = signature[:signature.rindex("(")].split("k_")[-1]
            assert "wait_for_stream()" in body.split("\n}", 1)[0] or "gemm<" in body.split("\n", 1)[0], kernel
            found.add(kernel.split("(")[0])
    assert found == {"residual_norm", "residual_norm_grad", "norm_columns", "rotary", "gemm", "gemm_pair", "gated_few", "join", "pad", "gate_grad"}
    gemm = open(os.path.join(folder, "gated_linear.cu")).read()
    assert gemm.index("wait_for_stream()") < gemm.index("load(to_a")


def test_limits_are_those_of_the_entry_points():
    import os
    import re
    from dccl_b200.ops import decoder
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "decoder", "decoder_ops.hpp")).read()
    limits = {k: eval(v) for k, v in re.findall(r"DCCL_(\w+_MAX_\w+) = ([0-9 <]+)", text)}
    assert limits == {"NORM_MAX_WIDTH": decoder._MAX_WIDTH, "ROTARY_MAX_PAIRS": decoder._MAX_PAIRS, "ROTARY_MAX_TOKEN": decoder._MAX_TOKEN, "GATED_MAX_DIMENSION": decoder._MAX_DIMENSION}


# ---------------------------------------------------------------------------------------------- norms

def norm_case(shape, dtype, post, gate, wide, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    w = shape[-1]
    vec = torch.float32 if wide else dtype
    t = {"x": torch.randn(shape, generator=g) * 3, "branch": torch.randn(shape, generator=g), "weight": 1 + 0.2 * torch.randn(w, generator=g)}
    if post:
        t["post"] = 1 + 0.2 * torch.randn(w, generator=g)
    if gate:
        t["gate"] = torch.randn(gate, generator=g)
    t = {k: v.to(dtype if k in ("x", "branch") else vec).to(device).requires_grad_(True) for k, v in t.items()}
    dy, dn = (torch.randn(shape, generator=g).to(dtype).to(device) for _ in range(2))
    return t, dy, dn


def norm_call(t, scale):
    return ops.residual_norm(t["x"], t["branch"], t["weight"], eps=EPS, post_weight=t.get("post"), gate=t.get("gate"), scale=scale)


def norm_check(t, dy, dn, scale, y, n, grads, dtype):
    """Everything against the formulas, with the bounds that follow from them."""
    u = half_step(dtype)
    d = {k: v.detach().double().cpu() for k, v in t.items()}
    dy, dn = (0 if v is None else v.double().cpu() for v in (dy, dn))
    width = d["x"].shape[-1]
    post, gate = d.get("post", torch.ones(width, dtype=torch.float64)), d.get("gate", torch.ones(width, dtype=torch.float64))
    b = d["branch"]
    rb = (b.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() if "post" in d else torch.ones_like(b[..., :1])
    p = b * rb * post
    want_y = d["x"] + scale * gate * p
    ry = (want_y.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    yh = want_y * ry
    terms = d["x"].abs() + (scale * gate * p).abs()
    check("y", y, want_y, u * want_y.abs() + F32 * terms)
    check("n", n, yh * d["weight"], u * (yh * d["weight"]).abs() + F32 * d["weight"].abs() * (terms * ry + yh.abs()))
    if grads is None:
        return
    # backward: y is made again in fp32 from x and the branch
    e_yh = F32 * (terms * ry + yh.abs())
    tt = dn * d["weight"]
    c = (tt * yh).mean(-1, keepdim=True) if torch.is_tensor(tt) else torch.zeros_like(ry)
    c_abs, e_c = (tt * yh).abs().mean(-1, keepdim=True) if torch.is_tensor(tt) else c, (tt * e_yh).abs().mean(-1, keepdim=True) if torch.is_tensor(tt) else c
    D = dy + ry * (tt - yh * c)
    e_D = ry * (e_yh * c.abs() + yh.abs() * e_c) + F32 * (abs(dy) + ry * (abs(tt) + yh.abs() * c_abs))
    check("dx", grads["x"], D, u * D.abs() + e_D)
    rows = tuple(range(D.dim() - 1))
    if torch.is_tensor(dn):
        dw = (dn * yh).sum(rows)
        check("dweight", grads["weight"], dw, half_step(t["weight"].dtype) * dw.abs() + (dn.abs() * e_yh).sum(rows) + SUMS * (dn * yh).abs().sum(rows))
    dp, e_dp = scale * D, abs(scale) * e_D
    if "gate" in d:
        terms_g = dp * p
        over = [i for i in range(D.dim()) if i < D.dim() - gate.dim() or gate.shape[i - (D.dim() - gate.dim())] != D.shape[i]]
        dims = tuple(over) or ()
        fold = (lambda v: v.sum(dims).reshape(gate.shape)) if dims else (lambda v: v)
        check("dgate", grads["gate"], fold(terms_g), half_step(t["gate"].dtype) * fold(terms_g).abs() + fold((e_dp * p).abs()) + SUMS * fold(terms_g.abs()))
        dp, e_dp = dp * gate, e_dp * gate.abs()
    if "post" in d:
        bh = b * rb
        check("dpost", grads["post"], (dp * bh).sum(rows), half_step(t["post"].dtype) * (dp * bh).sum(rows).abs() + (e_dp * bh.abs()).sum(rows) + SUMS * (dp * bh).abs().sum(rows))
        v, e_v = dp * post, e_dp * post.abs()
        cb, cb_abs, e_cb = ((f).mean(-1, keepdim=True) for f in (v * bh, (v * bh).abs(), e_v * bh.abs()))
        dp, e_dp = rb * (v - bh * cb), rb * (e_v + bh.abs() * e_cb) + F32 * rb * (v.abs() + bh.abs() * cb_abs)
    check("dbranch", grads["branch"], dp, u * dp.abs() + e_dp + F32 * dp.abs())


def norm_run(shape, dtype, post=False, gate=None, scale=1.0, wide=False, use_y=True, use_n=True, device="cuda"):
    t, dy, dn = norm_case(shape, dtype, post, gate, wide, device=device)
    with torch.no_grad():
        y0, n0 = norm_call(t, scale)
    y, n = norm_call(t, scale)
    assert torch.equal(y0, y) and torch.equal(n0, n), "with and without a graph"
    outs = [(y, dy)] * use_y + [(n, dn)] * use_n
    names = [k for k in t if k != "weight" or use_n]
    grads = dict(zip(names, torch.autograd.grad([o for o, _ in outs], [t[k] for k in names], [g for _, g in outs])))
    norm_check(t, dy if use_y else None, dn if use_n else None, scale, y, n, grads, dtype)


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("post,gate", [(False, None), (True, None), (True, "row"), (False, "seq")])
def test_norm_on_cpu(post, gate):
    norm_run((2, 5, 24), torch.float32, post, {"row": (24,), "seq": (2, 1, 24)}.get(gate), 0.5, device="cpu")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (3, 2, 33), (5, 96), (2, 3, 257), (7, 250), (300, 1451), (2, 300, 2048), (9, 2049), (40, 4096), (3, 5000), (700, 6152), (5, 8192),
                                   (4, 8193), (3, 16384), (2, 32768)], ids=str)
@pytest.mark.parametrize("form", ["sum", "all"])
def test_norm_at_its_widths(dtype, shape, form):
    if form == "sum":
        norm_run(shape, dtype)
    else:
        norm_run(shape, dtype, post=True, gate=shape[-1:], scale=0.37, wide=shape[-1] % 2 == 0)


@gpu
@pytest.mark.parametrize("gate", [None, (96,), (1, 1, 1, 96), (3, 1, 1, 96), (3, 4, 1, 96), (3, 4, 5, 96)], ids=str)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("use", [(True, True), (True, False), (False, True)])
def test_norm_forms(gate, post, use):
    norm_run((3, 4, 5, 96), torch.bfloat16, post, gate, 1.0, use_y=use[0], use_n=use[1])
    norm_run((3, 4, 5, 96), torch.float32, post, gate, -2.0, use_y=use[0], use_n=use[1])


@gpu
def test_norm_with_more_gates_than_ctas():
    norm_run((1500, 2, 64), torch.float16, True, (1500, 1, 64), 0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("width", [258, 2046, 2050, 6002, 8190, 8194, 16386])
def test_norm_of_pairs(dtype, width):
    """Widths of which accesses hold two 16-bit elements: several warps, and 8, 16 and 32 elements per thread."""
    norm_run((11, width), dtype)
    norm_run((2, 3, width), dtype, post=True, gate=(2, 1, width), scale=0.37, wide=True)


@gpu
@pytest.mark.parametrize("shape", [(3000, 1451), (3000, 1450), (700, 6001), (700, 6002), (500, 8194), (500, 8193), (1400, 2048), (350, 8192)], ids=str)
@pytest.mark.parametrize("form", ["sum", "all"])
def test_norm_with_many_rows_for_a_cta(shape, form):
    """More rows than CTAs can be resident (148 x 3 of up to 2048 elements, 148 of more), so that each CTA takes several, whatever its accesses."""
    if form == "sum":
        norm_run(shape, torch.bfloat16)
    else:
        norm_run(shape, torch.float16, post=True, gate=shape[-1:], scale=0.37)


@gpu
@pytest.mark.parametrize("dtype,gates,width", [(torch.float16, 5200, 64), (torch.float16, 5200, 65), (torch.float16, 5200, 66), (torch.float32, 5200, 64), (torch.bfloat16, 1000, 2048),
                                               (torch.bfloat16, 1000, 1999), (torch.bfloat16, 1000, 1998), (torch.bfloat16, 400, 4096), (torch.bfloat16, 400, 4001)], ids=str)
def test_norm_with_more_units_than_ctas(dtype, gates, width):
    """At most 148 x 23 CTAs of one warp, 148 x 3 of up to 2048 elements and 148 of more are resident, and every gate is a unit of its own: each CTA starts several.
    5200 units are added by 32 threads a column, 163 each to a sum that grows from nothing and counts half, and their 32 sums: within the 128 of SUMS."""
    norm_run((gates, 2, width), dtype, True, (gates, 1, width), 0.5)


@gpu
def test_norm_of_views():
    """Rows that start between two accesses, and tensors that are not dense: transposed, expanded."""
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(6 * 512 + 3, device="cuda", generator=g).bfloat16()
    x = base[3:].view(6, 512)
    branch = torch.randn(512, 6, device="cuda", generator=g).bfloat16().t()
    weight = torch.randn(512 + 1, device="cuda", generator=g)[1:]
    t = {"x": x, "branch": branch, "weight": weight}
    y, n = norm_call(t, 1.0)
    norm_check(t, None, None, 1.0, y, n, None, torch.bfloat16)
    t["branch"] = base[:512].expand(6, 512)
    y, n = norm_call(t, 1.0)
    norm_check(t, None, None, 1.0, y, n, None, torch.bfloat16)


@gpu
@pytest.mark.parametrize("off", range(0, 8, 3))
@pytest.mark.parametrize("width", [41, 2047, 2052, 6001])
def test_norm_gradients_of_rows_that_start_anywhere(off, width):
    """x, branch and the gradients at different distances from a 16-byte boundary, in the middle of larger buffers."""
    dtype, rows = torch.bfloat16, 37
    t, dy, dn = norm_case((rows, width), dtype, True, (width,), False, device="cuda")
    def moved(v, o):
        buf = torch.full((v.numel() + 16,), float("nan"), dtype=dtype, device="cuda")
        buf[o:o + v.numel()] = v.detach().reshape(-1)
        return buf[o:o + v.numel()].view(v.shape)
    t["x"], t["branch"] = moved(t["x"], off).requires_grad_(True), moved(t["branch"], (off + 1) % 8).requires_grad_(True)
    dy, dn = moved(dy, (off + 2) % 8), moved(dn, (off + 5) % 8)
    y, n = norm_call(t, 0.5)
    grads = dict(zip(t, torch.autograd.grad((y, n), list(t.values()), (dy, dn))))
    norm_check(t, dy, dn, 0.5, y, n, grads, dtype)


@gpu
def test_norm_gate_that_was_broadcast_gets_the_sum():
    t, dy, dn = norm_case((4, 3, 64), torch.float32, False, (1, 1, 64), False, device="cuda")
    one = t["gate"]
    t["gate"] = one.expand(4, 1, 64)
    y, n = norm_call(t, 1.0)
    got = torch.autograd.grad((y, n), one, (dy, dn))[0]
    t["gate"] = one
    y, n = norm_call(t, 1.0)
    want = torch.autograd.grad((y, n), one, (dy, dn))[0]
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)      # fp32 sums of twelve terms of about 1, in two orders


@gpu
def test_norm_rows_do_not_touch_each_other():
    t, _, _ = norm_case((4, 200), torch.float32, True, (200,), False, device="cuda")
    with torch.no_grad():
        y, n = norm_call(t, 1.0)
        for bad, row in ((float("nan"), 0), (float("inf"), 2)):
            t["branch"][row, 7] = bad
        y2, n2 = norm_call(t, 1.0)
    for row in (1, 3):
        assert torch.equal(y[row], y2[row]) and torch.equal(n[row], n2[row])
    assert bool(n2[0].isnan().all()) and bool(n2[2, 7].isnan())


@gpu
def test_norm_without_rows():
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, n = ops.residual_norm(x, x, w)
    (y.sum() + n.sum()).backward()
    assert y.shape == n.shape == x.grad.shape and bool((w.grad == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rms_norm(dtype):
    t, _, dn = norm_case((5, 7, 1024), dtype, False, None, False, device="cuda")
    n = ops.rms_norm(t["x"], t["weight"], eps=EPS)
    grads = dict(zip(("x", "weight"), torch.autograd.grad(n, (t["x"], t["weight"]), dn)))
    assert torch.equal(n, ops.rms_norm(t["x"].detach(), t["weight"].detach(), eps=EPS))
    # a branch of zeros makes residual_norm the same function
    t["branch"] = torch.zeros_like(t["x"])
    grads["branch"] = grads["x"]
    norm_check(t, None, dn, 1.0, t["x"], n, grads, dtype)


@gpu
def test_norm_gradient_against_differences():
    t, dy, dn = norm_case((2, 3, 32), torch.float32, True, (2, 1, 32), False, device="cuda")
    def loss(vals):
        y, n = norm_call(vals, 0.7)
        return ((y * dy).sum(-1).double() + (n * dn).sum(-1).double()).sum()
    grads = torch.autograd.grad(loss(t), list(t.values()))
    for (k, v), g in zip(t.items(), grads):
        way = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).cuda()
        h = 2.0 ** -8
        with torch.no_grad():
            up, down = (loss({**t, k: v + s * h * way}) for s in (1, -1))
        # the third derivative is of the size of the first for h = 1: h^2 of it, and fp32 roundings of the loss over 2 h
        want, got = (up - down) / (2 * h), (g * way).sum()
        assert abs(want - got) <= 40 * h * h * g.norm() * way.norm() / math.sqrt(g.numel()) + 2e-3, (k, want, got)


@gpu
def test_gradients_have_the_same_bits_twice():
    t, dy, dn = norm_case((64, 9, 1000), torch.bfloat16, True, (64, 1, 1000), False, device="cuda")
    runs = []
    for _ in range(2):
        y, n = norm_call(t, 0.5)
        runs.append(torch.autograd.grad((y, n), list(t.values()), (dy, dn)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
@pytest.mark.parametrize("width", [64, 250, 257, 4096, 16384])
def test_norm_entry_point_writes_each_gradient_that_it_gets_room_for(width):
    """Of a plain sum the branch's gradient is x's: the entry point writes it all the same where a caller has a buffer for it."""
    from dccl_b200._lib import lib
    L, rows = lib(), 5
    g = torch.Generator(device="cuda").manual_seed(width)
    x, branch, dy, dn = (torch.randn(rows, width, device="cuda", generator=g) for _ in range(4))
    weight, rstd = torch.randn(width, device="cuda", generator=g), torch.empty(rows, device="cuda")
    y, n = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.dccl_residual_norm(0, 7, rows, width, x.data_ptr(), branch.data_ptr(), weight.data_ptr(), None, None, 0, 0, EPS, 1.0, y.data_ptr(), n.data_ptr(), rstd.data_ptr(),
                                None, stream) == 0
    size = L.dccl_residual_norm_workspace(0, 7, rows, width, 0, 0, 1)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    grads = []
    for room in (True, False):
        dx, dbranch, dweight = torch.full_like(x, math.nan), torch.full_like(x, math.nan), torch.full_like(weight, math.nan)
        assert L.dccl_residual_norm_backward(0, 7, rows, width, dy.data_ptr(), dn.data_ptr(), x.data_ptr(), branch.data_ptr(), weight.data_ptr(), None, None, 0, 0, 1.0,
                                             rstd.data_ptr(), None, dx.data_ptr(), dbranch.data_ptr() if room else None, dweight.data_ptr(), None, None, work.data_ptr(), size,
                                             stream) == 0
        grads.append((dx, dweight))
        if room:
            assert torch.equal(dbranch, dx)
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("missing", ["x", "weight", "y", "n"])
def test_norm_entry_points_refuse_missing_buffers(missing, dccl_lib, capfd):
    from dccl_b200._lib import lib
    L = lib()
    if not hasattr(L, "dccl_residual_norm"):
        pytest.skip("built without CUDA")
    at = {k: None if k == missing else 4096 for k in ("x", "weight", "y", "n")}      # never read: no call gets as far as a device
    assert L.dccl_residual_norm(0, 7, 1, 8, at["x"], 4096, at["weight"], None, None, 0, 0, EPS, 1.0, at["y"], at["n"], None, None, None) == -1
    assert L.dccl_residual_norm_backward(0, 7, 1, 8, 4096, 4096, at["x"], 4096, at["weight"], None, None, 0, 0, 1.0, 4096, None, at["y"], None, None, None, None,
                                         at["n"], 1 << 30, None) == -1
    assert capfd.readouterr().err.count("invalid argument") == 2


def norm_refusals(device):
    x, w = torch.zeros(2, 3, 8, device=device), torch.ones(8, device=device)
    with pytest.raises(TypeError):
        ops.rms_norm(x.double(), w)
    with pytest.raises(TypeError):
        ops.rms_norm([1.0], w)
    with pytest.raises(TypeError):
        ops.rms_norm(x.bfloat16(), w.half())
    with pytest.raises(ValueError):
        ops.rms_norm(x, w[:4])
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(2, 0, device=device), w[:0])
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(1, 32769, device=device), torch.zeros(32769, device=device))
    with pytest.raises(TypeError):
        ops.residual_norm(x, None, w)
    with pytest.raises(TypeError):
        ops.residual_norm(x, x.half(), w)
    with pytest.raises(ValueError):
        ops.residual_norm(x, x[0], w)
    for shape in ((2, 8), (1, 3, 8), (2, 3, 4), (2, 2, 8), (3,)):
        with pytest.raises(ValueError):
            ops.residual_norm(x, x, w, gate=torch.ones(shape, device=device))
    with pytest.raises(ValueError):
        ops.residual_norm(x, x, w, post_weight=torch.ones(7, device=device))


def test_norm_refusals():
    norm_refusals("cpu")


@gpu
def test_norm_refusals_on_the_gpu():
    norm_refusals("cuda")
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(2, 8, device="cuda"), torch.ones(8))


# ---------------------------------------------------------------------------------------------- rotary positions

def turn(x, freqs, positions, interleaved, scale):
    """In 64 bits, as complex numbers; positions [batch, seq] or [seq]."""
    p = freqs.shape[0]
    x = x.detach().double().cpu()
    angle = positions.double().cpu().unsqueeze(-1) * freqs.cpu()
    spin = torch.polar(torch.full_like(angle, scale), angle)
    v = x[..., :2 * p]
    z = torch.complex(v[..., 0::2], v[..., 1::2]) if interleaved else torch.complex(v[..., :p], v[..., p:])
    z = z * spin.unsqueeze(-2)
    out = torch.stack((z.real, z.imag), -1).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    a = z.abs()
    size = torch.stack((a, a), -1).flatten(-2) if interleaved else torch.cat((a, a), -1)
    rest = x[..., 2 * p:]
    return torch.cat((out, rest), -1), torch.cat((size, torch.zeros_like(rest)), -1)


def check_turned(name, got, x, freqs, positions, interleaved, scale=1.0):
    """The part of a turn is off by 2^-25 of one in fp32, which is 2^-22 radians, and the sine and cosine and the products by as much
    again; the whole turns are three products in 64 bits, the reference's own among them, each off by 2^-53 of the angle."""
    want, size = turn(x, freqs, positions, interleaved, scale)
    angle = positions.double().cpu().abs().unsqueeze(-1).unsqueeze(-1)
    check(name, got, want, half_step(got.dtype) * want.abs() + (2.0 ** -20 + angle * 2.0 ** -51) * size)


def rotary_run(batch, seq, heads, kv, dim, pairs, dtype, interleaved=False, scale=1.0, furthest=4000, per_sequence=True, int32=False, device="cuda", front=False):
    g = torch.Generator().manual_seed(seq * dim + pairs)
    q, k, dq, dk = (torch.randn(batch, seq, h, dim, generator=g).to(dtype).to(device) for h in (heads, kv, heads, kv))
    if front:       # the heads in front in memory
        q, k, dq, dk = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, dq, dk))
    q.requires_grad_(True), k.requires_grad_(True)
    freqs = ops.rotary_frequencies(2 * pairs, device=device)
    pos = torch.randint(0, furthest, (batch, seq) if per_sequence else (seq,), generator=g)
    at = pos.to(torch.int32 if int32 else torch.int64).to(device)
    with torch.no_grad():
        q0, k0 = ops.rotary(q, k, freqs, at, interleaved, scale)
    q1, k1 = ops.rotary(q, k, freqs, at, interleaved, scale)
    assert torch.equal(q0, q1) and torch.equal(k0, k1) and q0.stride() == q.stride()
    gq, gk = torch.autograd.grad((q1, k1), (q, k), (dq, dk))
    check_turned("q", q1, q, freqs, pos, interleaved, scale)
    check_turned("k", k1, k, freqs, pos, interleaved, scale)
    check_turned("dq", gq, dq, -freqs, pos, interleaved, scale)
    check_turned("dk", gk, dk, -freqs, pos, interleaved, scale)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_on_cpu(interleaved):
    rotary_run(2, 5, 4, 2, 12, 4, torch.float32, interleaved, 0.9, device="cpu")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 2, 1), (2, 3, 4, 2, 64, 32), (1, 300, 32, 4, 64, 32), (3, 7, 5, 1, 80, 17), (2, 9, 3, 3, 128, 64), (1, 5, 2, 2, 96, 24), (2, 4, 2, 1, 13, 3),
                                   (1, 3, 1, 1, 2048, 1024), (16, 1, 32, 4, 64, 32), (2, 50, 8, 8, 256, 32), (1, 6, 3, 1, 20, 4), (1, 6, 3, 1, 36, 16)], ids=str)
def test_rotary_at_its_sizes(dtype, interleaved, sizes):
    rotary_run(*sizes, dtype, interleaved)


@gpu
@pytest.mark.parametrize("per_sequence,int32,front", [(True, True, False), (False, False, True), (False, True, False), (True, False, True)])
def test_rotary_positions_and_layouts(per_sequence, int32, front):
    rotary_run(3, 11, 4, 2, 64, 32, torch.bfloat16, False, 1.25, per_sequence=per_sequence, int32=int32, front=front)


@gpu
def test_rotary_cosines_and_sines_are_exact_to_their_size():
    """Pairs (1, 0) become (cos, sin) with no further rounding. Each is off by one step of sincospif, the correction's rounding and that of what it adds:
    three steps of 2^-23 of the value itself, also next to zero (355 is 113 pi to 3e-5); and of the angle by what 64 bits lose."""
    freqs = ops.rotary_frequencies(64, device="cuda")
    pos = torch.cat((torch.tensor([0, 3, 22, 333, 355, 710, 103993, 104348, 312689, 833719]), torch.randint(0, 1 << 20, (2000,), generator=torch.Generator().manual_seed(4))))
    x = torch.zeros(1, pos.numel(), 1, 64, device="cuda")
    x[..., :32] = 1
    got = ops.rotary(x, None, freqs, pos.cuda())[0, :, 0].double().cpu()
    angle = pos.double().unsqueeze(-1) * freqs.cpu()
    for name, v, want in (("cos", got[:, :32], angle.cos()), ("sin", got[:, 32:], angle.sin())):
        off = (v - want).abs() - (3 * 2.0 ** -23 * want.abs() + angle * 2.0 ** -51)
        assert off.max() <= 0, (name, off.max().item())


@gpu
def test_rotary_far_positions():
    rotary_run(2, 40, 4, 2, 64, 32, torch.float32, furthest=(1 << 31) - 1)
    q = torch.randn(1, 3, 2, 64, device="cuda")
    freqs = ops.rotary_frequencies(64, device="cuda")
    far = (1 << 33) + 5         # a double holds the turns to 2^-23
    check_turned("q", ops.rotary(q, None, freqs, far), q, freqs, torch.arange(far, far + 3), False)
    check_turned("q", ops.rotary(q, None, freqs, -7), q, freqs, torch.arange(-7, -4), False)


@gpu
def test_rotary_of_views():
    """q and k as parts of one product, at an odd offset, one of them expanded, three dimensions, a transposed gradient."""
    g = torch.Generator(device="cuda").manual_seed(1)
    freqs = ops.rotary_frequencies(64, device="cuda")
    both = torch.randn(2, 9, 6 * 64 + 1, device="cuda", generator=g).half()
    pos = torch.arange(9)
    for off in (0, 1):
        q, k = both[..., off:off + 4 * 64].unflatten(-1, (4, 64)), both[..., off + 4 * 64:off + 6 * 64 - off].unflatten(-1, (-1, 64)) if off == 0 else both[..., 5 * 64 + 1:].unflatten(-1, (1, 64))
        qo, ko = ops.rotary(q, k, freqs)
        check_turned("q", qo, q, freqs, pos, False)
        check_turned("k", ko, k, freqs, pos, False)
    wide = both[..., :64].unsqueeze(2).expand(2, 9, 3, 64)
    check_turned("expanded", ops.rotary(wide, None, freqs), wide, freqs, pos, False)
    last = torch.randn(9, 64, 2, device="cuda", generator=g).transpose(1, 2)        # the head dim is not the dense one
    check_turned("three", ops.rotary(last, None, freqs, torch.arange(0, 18, 2, device="cuda")), last, freqs, torch.arange(0, 18, 2), False)
    x = torch.randn(2, 9, 4, 64, device="cuda", generator=g, requires_grad=True)
    out = ops.rotary(x, None, freqs)
    grad = torch.randn(64, 4, 9, 2, device="cuda", generator=g).permute(3, 2, 1, 0)
    check_turned("gradient", torch.autograd.grad(out, x, grad)[0], grad, -freqs, pos, False)
    pos = torch.randint(0, 99, (9, 4), device="cuda", generator=g)
    check_turned("strided positions", ops.rotary(x, None, freqs, pos[:, 1:3].t()), x, freqs, pos[:, 1:3].t(), False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_leaves_what_does_not_turn(dtype, interleaved):
    """The elements behind the pairs are copied, next to whatever stands beside them."""
    freqs = ops.rotary_frequencies(10, device="cuda")
    q = torch.randn(2, 3, 2, 32, device="cuda").to(dtype)
    q[..., 10::3], q[..., 11::3] = float("inf"), float("nan")
    out = ops.rotary(q, None, freqs, 9)
    assert torch.equal(out[..., 10:].nan_to_num(7.0), q[..., 10:].nan_to_num(7.0)) and bool(out[..., :10].isfinite().all())


@gpu
def test_rotary_one_of_two_outputs_used():
    freqs = ops.rotary_frequencies(16, device="cuda")
    q, k = torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True), torch.randn(1, 3, 1, 16, device="cuda", requires_grad=True)
    ops.rotary(q, k, freqs)[1].sum().backward()
    assert q.grad is None and k.grad is not None
    assert ops.rotary(q[:, :0], k[:, :0], freqs)[0].shape == (1, 0, 2, 16)


def test_frequencies():
    f = ops.rotary_frequencies(64, theta=500000.0)
    assert f.dtype is torch.float64 and torch.allclose(f, torch.tensor([500000.0 ** (-j / 32) for j in range(32)], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(ops.rotary_frequencies(64, 500000.0, "linear", 4.0), f / 4, rtol=1e-14)
    t = ops.rotary_frequencies(64, 500000.0, "theta", 8.0)
    assert t[0] == 1 and math.isclose(t[-1], f[-1] / 8, rel_tol=1e-12) and bool((t <= f * (1 + 1e-12)).all())
    for kind, slow, fast in (("turns", 1, 4), ("yarn", 1, 32)):
        s = ops.rotary_frequencies(64, 500000.0, kind, 8.0, original_length=8192)
        turns = f * 8192 / (2 * math.pi)
        assert torch.allclose(s[turns > fast * 1.6], f[turns > fast * 1.6], rtol=1e-12)      # 1.6 is more than one pair further
        assert torch.allclose(s[turns < slow / 1.6], f[turns < slow / 1.6] / 8, rtol=1e-12)
        assert bool((s.diff() < 0).all())
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, theta=1.0), dict(rotary_dim=2, scaling="theta", factor=2.0),
                dict(rotary_dim=64, scaling="yarn", factor=2.0), dict(rotary_dim=64, scaling="other", factor=2.0), dict(rotary_dim=64, scaling="turns", original_length=8, slow=5.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


def rotary_refusals(device):
    q, f = torch.zeros(2, 3, 4, 8, device=device), ops.rotary_frequencies(8, device=device)
    for bad in (f.float(), f.to(torch.int64)):
        with pytest.raises(TypeError):
            ops.rotary(q, None, bad)
    for bad in (f[:0], torch.ones(5, dtype=torch.float64, device=device), f.view(2, 2)):
        with pytest.raises(ValueError):
            ops.rotary(q, None, bad)
    with pytest.raises(TypeError):
        ops.rotary(q.double(), None, f)
    with pytest.raises(TypeError):
        ops.rotary(q, q.half(), f)
    for k in (q[:1], q[:, :2], q[..., :6], q[0]):
        with pytest.raises(ValueError):
            ops.rotary(q, k, f)
    with pytest.raises(ValueError):
        ops.rotary(q[0, 0], None, f)
    for pos in (torch.zeros(4, dtype=torch.int64, device=device), torch.zeros(3, 3, dtype=torch.int64, device=device), torch.zeros(1, 3, dtype=torch.int64, device=device), 2 ** 63):
        with pytest.raises(ValueError):
            ops.rotary(q, None, f, pos)
    for pos in (torch.zeros(3, device=device), 1.5, True):
        with pytest.raises(TypeError):
            ops.rotary(q, None, f, pos)
    with pytest.raises(ValueError):
        ops.rotary(torch.zeros(1, 1, 1, 4096, device=device), None, torch.ones(1025, dtype=torch.float64, device=device))


def test_rotary_refusals():
    rotary_refusals("cpu")


@gpu
def test_rotary_refusals_on_the_gpu():
    rotary_refusals("cuda")
    with pytest.raises(ValueError):
        ops.rotary(torch.zeros(1, 2, 1, 8, device="cuda"), None, ops.rotary_frequencies(8))


# ---------------------------------------------------------------------------------------------- gated linear

ACTS = ["silu", "gelu", "gelu_tanh"]


def act_of(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def gated_case(tokens, width, ffn, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, width, generator=g)
    wg, wu = (torch.randn(ffn, width, generator=g) / math.sqrt(width) for _ in range(2))
    dh = torch.randn(tokens, ffn, generator=g)
    return [t.to(dtype).to(device) for t in (x, wg, wu, dh)]


def gated_check(x, wg, wu, dh, act, h, grads, dtype):
    """fp32 sums of k products are off by 2^-24 of every partial sum at most: k 2^-24 of the sum of sizes. The rounding of dg and du to
    `dtype` goes through the products that take them."""
    u = half_step(dtype)
    x, wg, wu = (t.detach().double().cpu().requires_grad_(True) for t in (x, wg, wu))
    with torch.no_grad():
        g, up = x @ wg.t(), x @ wu.t()
        size = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    k = x.shape[1] * 2.0 ** -24
    g.requires_grad_(True)
    a = act_of(g, act)
    slope = torch.autograd.grad(a.sum(), g)[0]
    g, a = g.detach(), a.detach()
    # |act'| is at most 1.13; sixteen fp32 operations on the activation
    e_a, e_u = 1.13 * k * size[0] + F32 * (a.abs() + g.abs()), k * size[1]
    want = a * up
    check("h", h, want, u * want.abs() + e_a * up.abs() + a.abs() * e_u + e_a * e_u)
    if grads is None:
        return
    dh = dh.double().cpu()
    # |act''| is at most 0.8
    e_slope = 0.8 * k * size[0] + F32 * (1 + g.abs())
    dg, du = dh * up * slope, dh * a
    e_g = u * dg.abs() + dh.abs() * (e_u * slope.abs() + up.abs() * e_slope + e_u * e_slope)
    e_d = u * du.abs() + dh.abs() * e_a
    tiny = torch.finfo(dtype).tiny * u      # of dg and du, where they are below the normal numbers
    e_g, e_d = e_g + tiny, e_d + tiny
    x, wg, wu = x.detach(), wg.detach(), wu.detach()
    for name, got, want, bound, n in (
            ("dx", grads[0], dg @ wg + du @ wu, e_g @ wg.abs() + e_d @ wu.abs(), 2 * dg.shape[1]),
            ("dw_gate", grads[1], dg.t() @ x, e_g.t() @ x.abs(), x.shape[0]),
            ("dw_up", grads[2], du.t() @ x, e_d.t() @ x.abs(), x.shape[0])):
        terms = {"dx": dg.abs() @ wg.abs() + du.abs() @ wu.abs(), "dw_gate": dg.abs().t() @ x.abs(), "dw_up": du.abs().t() @ x.abs()}[name]
        check(name, got, want, u * want.abs() + bound + n * 2.0 ** -24 * terms)


def gated_run(tokens, width, ffn, dtype, act="silu", device="cuda", backward=True):
    x, wg, wu, dh = gated_case(tokens, width, ffn, dtype, device)
    h = ops.gated_linear(x, wg, wu, act)
    grads = None
    if backward:
        for t in (x, wg, wu):
            t.requires_grad_(True)
        h2 = ops.gated_linear(x, wg, wu, act)
        assert torch.equal(h, h2), "with and without a graph"
        grads = torch.autograd.grad(h2, (x, wg, wu), dh)
    gated_check(x, wg, wu, dh, act, h, grads, dtype)


@pytest.mark.parametrize("act", ACTS)
def test_gated_on_cpu(act):
    gated_run(5, 24, 36, torch.float32, act, device="cpu")


SIZES = [(1, 64, 64), (1, 8, 8), (2, 1, 1), (3, 5, 7), (40, 256, 512), (128, 64, 128), (129, 72, 136), (200, 1000, 384), (257, 333, 191), (64, 2048, 200), (1, 2048, 5632), (300, 65, 1033),
         (1000, 40, 48), (520, 512, 1024), (17, 96, 2050), (16, 4104, 96), (33, 4104, 2400), (65, 200, 31), (100, 136, 1000), (128, 129, 65)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_gated_at_its_sizes(dtype, sizes):
    gated_run(*sizes, dtype)


# Reach with SIZES every kind of plan that the rule gives on 148 SMs: tiles of one CTA or a pair, 128 or 256 columns, whole or cut along k, and up to three
# tiles for a CTA, with more blocks of k than it has stages and remainders in all dimensions.
LARGE = [(461, 8, 200), (1, 8, 10992), (545, 520, 816), (9484, 544, 8), (1547, 1288, 824), (2411, 792, 1080), (3589, 3408, 522), (4336, 1128, 1956), (667, 6200, 682), (513, 272, 14291),
         (17, 8200, 570)]


@gpu
@pytest.mark.parametrize("sizes", LARGE, ids=str)
def test_gated_in_every_kind_of_plan(sizes):
    gated_run(*sizes, torch.float16 if sizes[1] % 16 else torch.bfloat16)


def test_sizes_reach_every_kind_of_plan(tiles_program):
    import subprocess

    def kind(form, m, n, k):
        pair, columns, splits, rounds = (int(v) for v in subprocess.run([tiles_program, "plan", "148"] + [str(v) for v in (form, m, n, k)], capture_output=True, text=True, check=True).stdout.split())
        return "gated dx dw".split()[form], "pair" if pair else "one", columns, "cut" if splits > 1 else min(rounds, 3)

    found = set()
    for tokens, width, ffn in SIZES + LARGE:
        if tokens > 128 or (width > 4096 and ffn <= 73 * 8):         # few_tokens
            found.add(kind(0, tokens, ffn, width))
        found |= {kind(1, tokens, width, ffn), kind(2, ffn, width, tokens)}
    wanted = {(form, "pair", columns, how) for form in ("gated", "dx", "dw") for columns in (128, 256) for how in ("cut", 1, 2, 3)}
    wanted -= {("gated", "pair", 128, 3), ("dx", "pair", 128, 3)}             # the rule does not give these
    wanted |= {("gated", "one", 128, "cut"), ("gated", "one", 256, "cut")}    # 128 tokens at most, and a layer too wide for k_gated_few
    wanted |= {(form, "one", 128, how) for form in ("dx", "dw") for how in ("cut", 1)} | {("dx", "one", 256, "cut"), ("dw", "one", 256, "cut")}
    assert wanted <= found, wanted - found


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gated_activations(act):
    gated_run(150, 264, 320, torch.bfloat16, act)
    gated_run(9, 33, 65, torch.float16, act)


@gpu
def test_gated_of_views():
    """Operands that start between two accesses, a transposed weight, leading dimensions, a gradient that was expanded."""
    base = torch.randn(70 * 256 + 3, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    _, wg, wu, _ = gated_case(1, 256, 96, torch.bfloat16, "cuda")
    x = base[3:].view(70, 256)
    gated_check(x, wg, wu, None, "silu", ops.gated_linear(x, wg, wu), None, torch.bfloat16)
    wt = wg.t().contiguous().t()
    x3 = x.view(7, 10, 256).transpose(0, 1)
    h = ops.gated_linear(x3, wt, wu)
    gated_check(x3.reshape(70, 256), wg, wu, None, "silu", h.reshape(70, 96), None, torch.bfloat16)
    x = x.clone().requires_grad_(True)
    h = ops.gated_linear(x, wg, wu)
    one = torch.ones(1, 1, device="cuda").bfloat16().expand(70, 96)
    dx, = torch.autograd.grad(h, x, one, retain_graph=True)
    assert torch.equal(dx, torch.autograd.grad(h, x, torch.ones_like(h))[0])


@gpu
def test_gated_gradients_of_some_inputs():
    x, wg, wu, dh = gated_case(33, 64, 72, torch.bfloat16, "cuda")
    all_in = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    want = torch.autograd.grad(ops.gated_linear(*all_in), all_in, dh)
    for i in range(3):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, wg, wu))]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*some), some[i], dh)[0], want[i])


@gpu
@pytest.mark.parametrize("tokens", [20, 100, 140, 300])
def test_gated_infinities_stay_in_their_rows(tokens):
    x, wg, wu, _ = gated_case(tokens, 64, 72, torch.bfloat16, "cuda")
    h = ops.gated_linear(x, wg, wu)
    last = tokens - 10
    x[3, 5], x[last, 0] = float("nan"), float("inf")
    bad = ops.gated_linear(x, wg, wu)
    rows = [r for r in range(tokens) if r not in (3, last)]
    assert torch.equal(bad[rows], h[rows]) and bool(bad[3].isnan().all()) and not bool(bad[last].isfinite().any())


@gpu
def test_gated_without_tokens():
    x, wg, wu, _ = (t.requires_grad_(True) for t in gated_case(0, 64, 72, torch.bfloat16, "cuda"))
    ops.gated_linear(x, wg, wu).sum().backward()
    assert x.grad.shape == x.shape and bool((wg.grad == 0).all()) and bool((wu.grad == 0).all())


def gated_refusals(device, dtype):
    x, w = torch.zeros(2, 8, device=device, dtype=dtype), torch.zeros(6, 8, device=device, dtype=dtype)
    for bad in ((x.double(), w, w), (x.int(), w, w), (x, w.double(), w), (x, w, w.double()), (x, [1], w), (x, w, None), (x, w[0], w)):
        with pytest.raises(TypeError):
            ops.gated_linear(*bad)
    for bad in ((x, w[:, :4], w), (x, w, w[:3]), (x[:, :4], w, w), (x, w[:0], w[:0]), (x[:, :0], w[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            ops.gated_linear(*bad)
    for act in ("relu", None, "SILU"):
        with pytest.raises(ValueError):
            ops.gated_linear(x, w, w, act)


def test_gated_refusals():
    gated_refusals("cpu", torch.float32)


@gpu
def test_gated_refusals_on_the_gpu():
    gated_refusals("cuda", torch.bfloat16)
    with pytest.raises(TypeError):
        ops.gated_linear(torch.zeros(2, 8, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(6, 8, device="cuda"))
    with pytest.raises(ValueError):
        ops.gated_linear(torch.zeros(2, 8, device="cuda").half(), torch.zeros(6, 8).half(), torch.zeros(6, 8, device="cuda").half())


@pytest.fixture(scope="module")
def tiles_program(tmp_path_factory):
    """tests/sim/gated_tiles.cpp: how products are cut, without a GPU."""
    import os
    import subprocess
    exe = str(tmp_path_factory.mktemp("tiles") / "gated_tiles")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(os.path.dirname(os.path.abspath(__file__)), "sim", "gated_tiles.cpp"), "-o", exe],
                   check=True)
    return exe


def test_products_that_gave_up_leave_nan(tiles_program):
    """A wait that runs out must not be made to happen on a GPU: the stores that follow one run here, for every CTA and thread."""
    import subprocess
    res = subprocess.run([tiles_program, "mark"], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def test_kernels_that_give_up_mark_their_results():
    import os
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "decoder", "gated_linear.cu")).read()
    parts = text.split("if (failed) {")[1:]
    assert len(parts) == 2 and all("mark_incomplete(" in p.split("*reinterpret_cast<volatile int*>(a.gave_up) = 1")[0] for p in parts)


# ---------------------------------------------------------------------------------------------- together

def decoders(device, dtype, **kw):
    """The same decoder as a chain of torch's operations and fused, and tokens for it."""
    import copy
    from dccl_b200.models.llama import LlamaConfig, LlamaDecoder
    torch.manual_seed(5)
    plain = LlamaDecoder(LlamaConfig(vocab_size=192, hidden=128, layers=2, heads=4, kv_heads=2, ffn=200, max_seq=64, **kw)).to(dtype)
    fused = copy.deepcopy(plain)
    fused.cfg.fused = True
    plain.cfg = copy.copy(plain.cfg)
    plain.cfg.fused = False
    tokens = torch.randint(0, 192, (3, 33), generator=torch.Generator().manual_seed(6))
    return plain.to(device), fused.to(device), tokens.to(device)


def test_the_fused_decoder_is_the_same_model():
    """In fp32 on the CPU, where both are sums of the same terms in other orders: about fifty operations deep, each off by a few times 2^-24
    (1e-5 of the largest gradient), and angles of the tables are off by 2^-24 of up to 33 radians."""
    plain, fused, tokens = decoders("cpu", torch.float32)
    assert list(plain.state_dict()) == list(fused.state_dict())
    a, b = plain.loss(tokens), fused.loss(tokens)
    a.backward()
    b.backward()
    assert abs(a - b) < 1e-5 * abs(a)
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert (p.grad - q.grad).abs().max() <= 3e-5 * p.grad.abs().max() + 1e-7, name


class Doubled(torch.nn.Module):
    """Stands in a module's place and does more."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *args):
        return 2 * self.inner(*args)


def double(module, args, out):
    return 2 * out


def touch(model, how):
    """Changes what modules of a decoder do. The same change to its plain and its fused form has to have the same effect."""
    block, other = model.blocks[0], model.blocks[1]
    linears = {"%s of %d" % (name, i): (b, name) for i, b in enumerate(model.blocks) for name in ("gate", "up")}
    if how == "hooks on all":
        calls = []
        for name, m in model.named_modules():
            m.register_forward_hook(lambda m, a, o, name=name: calls.append(name))
        return calls
    if how == "hooks that change":
        for m in (block.n1, block.gate, other.n2, other.attn, other.up, model.norm):
            m.register_forward_hook(double)
    elif how == "hooks before":
        for m in (block.n2, block.up, other.n1, model.norm):
            m.register_forward_pre_hook(lambda m, args: (2 * args[0],))
    elif how == "a block's hook":
        block.register_forward_hook(double)
    elif how == "the last block's hook":
        other.register_forward_hook(double)
    elif how == "other modules":
        block.gate, block.n2, other.attn, other.n1, model.norm = (Doubled(m) for m in (block.gate, block.n2, other.attn, other.n1, model.norm))
    elif how == "other blocks":
        model.blocks[0], model.blocks[1] = Doubled(block), Doubled(other)
    elif how == "other classes":
        block.n2, other.n1 = (torch.nn.LayerNorm(model.cfg.hidden) for _ in range(2))
    elif how == "biases":
        for b, name in linears.values():
            getattr(b, name).bias = torch.nn.Parameter(torch.linspace(-1, 1, getattr(b, name).out_features, dtype=getattr(b, name).weight.dtype))
    elif how == "another forward":
        for m in (block.up, other.n2, block.attn, other):
            m.forward = lambda *args, f=m.forward: 2 * f(*args)
    elif how == "parametrized":
        torch.nn.utils.parametrizations.weight_norm(block.gate)
        torch.nn.utils.parametrize.register_parametrization(other.n2, "weight", Doubled(torch.nn.Identity()))
    elif how == "hooks backward":
        for m in (block.n1, block.gate, other.attn, other, model.norm):
            m.register_full_backward_hook(lambda m, gi, go: tuple(None if g is None else 2 * g for g in gi))
    else:
        raise ValueError(how)


TOUCHES = ["hooks on all", "hooks that change", "hooks before", "a block's hook", "the last block's hook", "other modules", "other blocks", "other classes", "biases", "another forward",
           "parametrized", "hooks backward"]


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("how", TOUCHES)
def test_what_is_done_to_a_modules_call_is_done_to_the_fused_decoder(how, split):
    """Bounds of test_the_fused_decoder_is_the_same_model, eight times as wide for what is doubled up to three times on the way."""
    from dccl_b200 import Communicator
    from dccl_b200.models.llama_tp import shard
    models = decoders("cpu", torch.float32)
    tokens = models[2]
    comm = Communicator(rank=0, world=1) if split else None
    try:
        seen = []
        pair = [shard(m, comm) if split else m for m in models[:2]]
        for m in pair:
            seen.append(touch(m, how))
        losses = [m.loss(tokens) for m in pair]
        for v in losses:
            v.backward()
        if how == "hooks on all":
            assert sorted(seen[0]) == sorted(seen[1])
        assert abs(losses[0] - losses[1]) < 8e-5 * abs(losses[0])
        for (name, p), q in zip(pair[0].named_parameters(), pair[1].named_parameters()):
            assert q[0] == name and (p.grad - q[1].grad).abs().max() <= 24e-5 * p.grad.abs().max() + 1e-6, name
    finally:
        if comm is not None:
            comm.finalize()


def test_a_hook_on_every_module_runs_in_the_fused_decoder():
    plain, fused, tokens = decoders("cpu", torch.float32)
    calls = []
    with torch.no_grad():
        want = fused(tokens)
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, o: calls.append(type(m).__name__))
    try:
        with torch.no_grad():
            got = fused(tokens)
        there, calls[:] = sorted(calls), []
        with torch.no_grad():
            plain(tokens)
    finally:
        handle.remove()
    assert there == sorted(calls) and torch.allclose(got, want, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        assert torch.equal(fused(tokens), want)


@pytest.mark.parametrize("world", [1, 2])
def test_the_fused_decoder_split_over_ranks(dccl_lib, world):
    import os
    from dccl_b200.utils.launch import python_ranks
    res = python_ranks(os.path.join(os.path.dirname(os.path.abspath(__file__)), "workers", "llama_fused_worker.py"), [], world, timeout=300)
    for r, p in enumerate(res):
        assert p.returncode == 0, "rank %d:\n%s\n%s" % (r, p.stdout[-3000:], p.stderr[-3000:])
        assert p.stdout.strip().splitlines()[-1].startswith("OK"), p.stdout


def fused_against_plain(device, dtype, autocast, loss_bound, grad_bound, norm):
    plain, fused, tokens = decoders(device, dtype)
    losses = []
    for m in (plain, fused):
        with torch.autocast(device, torch.bfloat16, enabled=autocast):
            losses.append(m.loss(tokens))
        losses[-1].backward()
    assert abs(losses[0] - losses[1]) <= loss_bound * abs(losses[0])
    for (name, p), q in zip(plain.named_parameters(), fused.named_parameters()):
        off, size = p.grad.double() - q[1].grad.double(), p.grad.double()
        assert q[1].grad.dtype == p.grad.dtype and (off.norm() <= grad_bound * size.norm() if norm else off.abs().max() <= grad_bound * size.abs().max() + 1e-7), name


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype,autocast", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, True), (torch.float64, False)], ids=str)
def test_the_fused_decoder_takes_the_types_of_the_plain_one(device, dtype, autocast):
    """fp32 as in test_the_fused_decoder_is_the_same_model, and of fp64 only what the norms and the turned heads round to fp32. Where bf16 comes in, about
    thirty results on the way and as many back, each off by 2^-9 in the root mean square in both: twice 8 x 2^-9 of a gradient's norm."""
    low = autocast or dtype is torch.bfloat16
    fused_against_plain(device, dtype, autocast, 2.0 ** -7 if low else 1e-5, 0.032 if low else 3e-5, low)


@pytest.mark.parametrize("norms,model", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)], ids=str)
def test_norms_of_another_type_in_the_fused_decoder(norms, model):
    plain, fused, tokens = decoders("cpu", model)
    for m in (plain, fused):
        for block in m.blocks:
            block.n1.to(norms), block.n2.to(norms)
    a, b = plain.loss(tokens), fused.loss(tokens)
    assert abs(a - b) <= 2.0 ** -7 * abs(a)


@pytest.mark.parametrize("device", ["cpu", "meta", pytest.param("cuda", marks=gpu)])
def test_the_fused_decoder_of_tensors_without_values(device):
    from torch._subclasses.fake_tensor import FakeTensorMode
    plain, fused, tokens = decoders("cpu", torch.bfloat16)
    if device == "meta":
        logits = [m.to("meta")(tokens.to("meta")) for m in (plain, fused)]
    else:
        from dccl_b200.models.llama import LlamaDecoder
        torch.set_default_dtype(torch.bfloat16)
        try:
            with FakeTensorMode(), torch.device(device):
                logits = [LlamaDecoder(m.cfg)(torch.zeros(3, 33, dtype=torch.int64)) for m in (plain, fused)]
        finally:
            torch.set_default_dtype(torch.float32)
    assert logits[0].shape == logits[1].shape and logits[1].device.type == device


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_the_fused_decoder_under_transforms(device):
    """torch.func.grad, and functions of parameters: bounds of test_the_fused_decoder_is_the_same_model."""
    plain, fused, tokens = decoders(device, torch.float32)
    grads = []
    for m in (plain, fused):
        params = {k: v.detach() for k, v in m.named_parameters()}
        grads.append(torch.func.grad(lambda p: torch.nn.functional.cross_entropy(torch.func.functional_call(m, p, (tokens[:, :-1],)).flatten(0, 1), tokens[:, 1:].flatten()))(params))
    for k, g in grads[0].items():
        assert (g - grads[1][k]).abs().max() <= 3e-5 * g.abs().max() + 1e-7, k


@gpu
def test_the_fused_decoder_compiled():
    _, fused, tokens = decoders("cuda", torch.bfloat16)
    want = fused.loss(tokens)
    want.backward()
    grads = {k: p.grad.clone() for k, p in fused.named_parameters()}
    fused.zero_grad(set_to_none=True)
    loss = torch.compile(fused.loss, backend="eager")(tokens)
    loss.backward()
    assert torch.equal(loss, want)
    for k, p in fused.named_parameters():        # the gradient of attention may add in another order from call to call: two steps of bf16
        assert (p.grad.double() - grads[k].double()).norm() <= 2.0 ** -6 * grads[k].double().norm(), k


@gpu
def test_the_fused_decoder_on_the_gpu():
    """bf16 on the GPU against the same operators on the CPU: about thirty bf16 results on the way to the loss and as many back, each off by
    2^-9 in the root mean square at most, at random: 8 x 2^-9 = 1.6 % of the norm of a gradient, twice that allowed."""
    import copy
    _, fused, tokens = decoders("cpu", torch.bfloat16)
    there = copy.deepcopy(fused).cuda()
    a, b = fused.loss(tokens), there.loss(tokens.cuda())
    a.backward()
    b.backward()
    assert abs(a.item() - b.item()) < 2.0 ** -7 * abs(a.item())
    for (name, p), q in zip(fused.named_parameters(), there.parameters()):
        off = (p.grad.double() - q.grad.double().cpu()).norm() / p.grad.double().norm()
        assert off < 0.032, (name, off)


@gpu
def test_the_fused_decoder_in_its_forms_on_one_gpu(dccl_lib):
    """A world of one rank runs the same code: with the block exits in pool buffers, which come round again before the backward pass, and with
    the sequence cut."""
    import copy
    from dccl_b200 import Communicator
    from dccl_b200.models.llama_tp import shard
    _, fused, tokens = decoders("cuda", torch.bfloat16)
    fused.loss(tokens).backward()
    want = {k: p.grad.clone() for k, p in fused.named_parameters()}
    fused.zero_grad(set_to_none=True)
    comm = Communicator(rank=0, world=1, device=0)
    try:
        for kw in ({}, {"in_place_reduce": True}, {"sequence_parallel": True}):
            tp = shard(copy.deepcopy(fused), comm, **kw)
            tp.loss(tokens).backward()
            for k, p in tp.named_parameters():
                # the loss's gradient differs by its scale's rounding at most: two steps of bf16
                assert (p.grad.double() - want[k].double()).norm() <= 2.0 ** -6 * want[k].double().norm(), (kw, k)
            torch.cuda.synchronize()
            tp.close()
    finally:
        comm.finalize()


@gpu
def test_a_decoding_step_in_a_graph():
    """One token of each sequence through norm, rotary and the gated layer, captured once and replayed with other inputs and positions; on a stream
    of its own, next to a second graph with workspaces of its own."""
    w = {k: torch.randn(s, device="cuda").bfloat16() * 0.05 for k, s in (("n", 256), ("g", (512, 256)), ("u", (512, 256)))}
    freqs = ops.rotary_frequencies(64, device="cuda")
    x, branch, q = (torch.randn(4, 1, 256, device="cuda").bfloat16() for _ in range(3))
    at = torch.tensor([[5], [0], [70000], [12]], device="cuda")

    def step():
        with torch.no_grad():
            y, n = ops.residual_norm(x, branch, w["n"])
            return y, ops.gated_linear(n, w["g"], w["u"]), ops.rotary(q.view(4, 1, 4, 64), None, freqs, at)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        step()
        for _ in range(2):
            graphs.append((torch.cuda.CUDAGraph(),))
            with torch.cuda.graph(graphs[-1][0], stream=stream):
                graphs[-1] += step(),
    torch.cuda.synchronize()
    for turn_ in range(3):
        for t in (x, branch, q):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(turn_)).bfloat16())
        at.add_(turn_ * 1000)
        want = step()
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
@pytest.mark.parametrize("rows,width,ffn", [(70, 96, 80), (300, 264, 320), (130, 65, 131)])
def test_a_training_step_in_a_graph(rows, width, ffn):
    """Forward and backward captured, replayed on new inputs."""
    x, branch, weight = (t.cuda().bfloat16().requires_grad_(True) for t in (torch.randn(rows, width), torch.randn(rows, width), torch.ones(width)))
    wg, wu = (torch.randn(ffn, width).mul(0.1).cuda().bfloat16().requires_grad_(True) for _ in range(2))
    dh = torch.randn(rows, ffn).cuda().bfloat16()

    def step():
        y, n = ops.residual_norm(x, branch, weight, post_weight=weight, scale=0.5)
        return torch.autograd.grad((ops.gated_linear(n, wg, wu), y), (x, branch, weight, wg, wu), (dh, torch.ones_like(y)))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step()
    for seed in range(2):
        with torch.no_grad():
            x.copy_(torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


FIRST = """
import torch
from dccl_b200 import ops
x, w, wg, wu = (torch.randn(s, device="cuda").bfloat16() for s in ((200, 128), (128,), (256, 128), (256, 128)))
freqs = ops.rotary_frequencies(32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
step = lambda: (ops.gated_linear(ops.rms_norm(x, w), wg, wu), ops.gated_linear(x[:1], wg, wu), ops.rotary(x.view(1, 200, 4, 32), None, freqs))
with torch.cuda.graph(graph):
    outs = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, step()))
print("OK")
"""


@gpu
def test_the_first_call_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys
    res = subprocess.run([sys.executable, "-c", FIRST], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout + res.stderr[-2000:]


@gpu
def test_operators_on_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x, wg, wu, dh = gated_case(140, 64, 144, torch.bfloat16, "cuda:1")
    for t in (x, wg, wu):
        t.requires_grad_(True)
    w = torch.ones(64, device="cuda:1").bfloat16()
    h = ops.gated_linear(ops.rms_norm(x, w), wg, wu)
    grads = torch.autograd.grad(h, (x, wg, wu), dh)
    with torch.cuda.device(1):
        again = ops.gated_linear(ops.rms_norm(x, w), wg, wu)
        assert torch.equal(h, again) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again, (x, wg, wu), dh)))
    assert torch.cuda.current_device() == 0


@gpu
def test_operators_of_two_streams_at_once():
    x, wg, wu, _ = gated_case(300, 512, 640, torch.bfloat16, "cuda")
    w = torch.ones(512, device="cuda").bfloat16()
    want = ops.gated_linear(ops.rms_norm(x, w), wg, wu)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(ops.gated_linear(ops.rms_norm(x, w), wg, wu))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for o in outs for v in o)


@gpu
def test_autograd_of_the_operators():
    """retain_graph, a second pass over a freed graph, inputs changed in place, gradients of gradients, forward mode."""
    x, wg, wu, dh = gated_case(9, 64, 72, torch.bfloat16, "cuda")
    w = torch.ones(64, device="cuda").bfloat16().requires_grad_(True)
    freqs = ops.rotary_frequencies(16, device="cuda")
    x.requires_grad_(True)
    for make in (lambda v: ops.gated_linear(v, wg, wu), lambda v: ops.rms_norm(v, w), lambda v: ops.residual_norm(v, v, w)[1], lambda v: ops.rotary(v.view(1, 9, 4, 16), None, freqs)):
        y = make(x)
        first, = torch.autograd.grad(y.sum(), x, retain_graph=True)
        again, = torch.autograd.grad(y.sum(), x)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.sum(), x)
        g, = torch.autograd.grad(make(x).float().pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)
    v = x.detach().clone().requires_grad_(True)
    z = v * 1
    y = ops.gated_linear(z, wg, wu)
    z.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            ops.rms_norm(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()), w.detach())
    with torch.inference_mode():
        assert torch.equal(ops.rms_norm(x, w), ops.rms_norm(x.detach(), w.detach()))


@gpu
def test_operators_refuse_tensors_without_memory():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        x, w = torch.empty(4, 64, device="cuda"), torch.ones(64, device="cuda")
        with pytest.raises(TypeError):
            ops.rms_norm(x, w)
    del mode


@gpu
def test_negated_views():
    x, w = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    assert torch.equal(ops.rms_norm(torch._neg_view(x), w), ops.rms_norm(-x, w))


@gpu
def test_checkpointed_operators():
    """What a backward pass needs is dropped and made again, also what no input or output is."""
    from torch.utils.checkpoint import checkpoint
    x, wg, wu, dh = gated_case(40, 65, 72, torch.bfloat16, "cuda")
    w = torch.ones(65, device="cuda").bfloat16().requires_grad_(True)
    for t in (x, wg, wu):
        t.requires_grad_(True)

    def part(v):
        return ops.gated_linear(ops.residual_norm(v, v, w, post_weight=w)[1], wg, wu)

    want = torch.autograd.grad(part(x), (x, w, wg, wu), dh)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(tuple(t.shape)) or t, lambda t: t):
        part(x)
    assert kept.count((40, 72)) == 2 and (40,) in kept          # the products and the rows' statistics
    got = torch.autograd.grad(checkpoint(part, x, use_reentrant=False), (x, w, wg, wu), dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------------------- what follows torch's operations

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


def chain(device="cuda"):
    """A function through every operator, each with what it may be given, and two inputs for it."""
    g = torch.Generator().manual_seed(9)
    t = [torch.randn(s, generator=g).to(device).bfloat16().requires_grad_(True) for s in ((2, 6, 64), (2, 6, 64), (64,), (64,), (2, 1, 64), (96, 64), (96, 64))]
    _, branch, w, post, gate, wg, wu = t
    freqs, at = ops.rotary_frequencies(16, device=device), torch.randint(0, 1000, (2, 6), generator=g).to(device)

    def f(x):
        y, n = ops.residual_norm(x, branch, w, post_weight=post, gate=gate, scale=0.5)
        q, k = ops.rotary(n.view(2, 6, 4, 16), y[..., :32].view(2, 6, 2, 16), freqs, at, interleaved=True)
        return ops.gated_linear(ops.rms_norm(q.flatten(2), w), wg, wu), ops.rotary(k, None, freqs, 7), y

    return f, t, torch.randn(2, 6, 64, generator=g).to(device).bfloat16()


def all_of(f, t, x):
    """The outputs of f and the gradients of everything that goes into it."""
    x = x.detach().requires_grad_(True)
    outs = f(x)
    return list(outs) + list(torch.autograd.grad(outs, [x] + t[1:], [torch.ones_like(o) for o in outs]))


@gpu
@pytest.mark.parametrize("mode", [SeesDispatch, SeesFunctions])
def test_an_active_mode_sees_the_operators(mode):
    f, t, x = chain()
    want = all_of(f, t, x)
    with mode() as m:
        got = all_of(f, t, x)
    seen = " ".join(m.seen)
    for name in ("residual_norm", "rotary", "gated_linear"):
        assert "dccl." + name in seen and (mode is SeesFunctions or "dccl.%s_backward" % name in seen), (name, m.seen)
    # x gets a sum of two gradients, which the kernels of one call and of two add in one order
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_a_mode_that_places_new_tensors_changes_nothing(monkeypatch):
    from dccl_b200.ops import decoder
    f, t, x = chain()
    want = all_of(f, t, x)
    monkeypatch.setattr(decoder, "_observed", None)
    with torch.device("cuda"):
        assert all(torch.equal(a, b) for a, b in zip(all_of(f, t, x), want))


@gpu
@pytest.mark.parametrize("tracer", ["trace", "make_fx"])
def test_tracers_record_the_operators(tracer):
    """A recorded call computes from its inputs, and not what the inputs were when it was recorded."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, t, other = chain()
    for v in t:
        v.requires_grad_(tracer == "make_fx")       # torch.jit.trace takes no constants that do
    with torch.no_grad():
        recorded = torch.jit.trace(f, (t[0],)) if tracer == "trace" else make_fx(f)(t[0])
        assert all(torch.equal(a, b) for a, b in zip(recorded(other), f(other)))
    if tracer == "make_fx":
        step = make_fx(lambda x: all_of(f, t, x))(t[0])
        assert all(torch.equal(a, b) for a, b in zip(step(other), all_of(f, t, other)))


@gpu
def test_a_traced_decoder_reads_its_tokens():
    _, fused, tokens = decoders("cuda", torch.bfloat16)
    fused.requires_grad_(False)
    traced = torch.jit.trace(fused, (tokens,))
    other = tokens.flip(0, 1)
    assert torch.equal(traced(other), fused(other)) and not torch.equal(fused(other), fused(tokens))


@gpu
def test_the_first_observed_calls_of_a_process_may_come_from_two_threads():
    import os
    import subprocess
    import sys
    code = """
import threading, torch
from dccl_b200 import ops
from torch.utils.flop_counter import FlopCounterMode
x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
want, got, start = ops.rms_norm(x, w), [], threading.Barrier(4)
def call():
    start.wait()
    with FlopCounterMode(display=False):
        got.append(ops.rms_norm(x, w))
threads = [threading.Thread(target=call) for _ in range(4)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(got) == 4 and all(torch.equal(g, want) for g in got)
print("OK")
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout + res.stderr[-2000:]


@gpu
def test_subclasses_of_tensor_see_the_operators():
    class Plain(torch.Tensor):
        pass

    class Sees(torch.Tensor):
        seen = []

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.seen.append(str(func))
            return super().__torch_function__(func, types, args, kwargs or {})

    f, t, x = chain()
    want = all_of(f, t, x)
    for cls in (Plain, Sees):
        with torch.no_grad():
            outs = f(x.as_subclass(cls))
        assert all(type(o) is cls for o in outs) and all(torch.equal(a.as_subclass(torch.Tensor), b) for a, b in zip(outs, want))
        y = x.detach().as_subclass(cls).requires_grad_(True)
        g, = torch.autograd.grad(f(y)[0].sum(), y)
        assert torch.equal(g.as_subclass(torch.Tensor), torch.autograd.grad(f(x.requires_grad_(True))[0].sum(), x)[0])
    assert any("dccl.gated_linear" in s for s in Sees.seen)


@gpu
def test_selective_checkpointing_of_the_operators():
    """It follows a region by a mode, and takes what that sees again from its cache or makes it again."""
    from functools import partial
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    f, t, x = chain()
    want = all_of(f, t, x)
    for keep in (True, False):
        def policy(ctx, op, *args, **kwargs):
            return CheckpointPolicy.MUST_SAVE if keep and "dccl" in str(op) else CheckpointPolicy.PREFER_RECOMPUTE
        got = all_of(lambda v: checkpoint(f, v, use_reentrant=False, context_fn=partial(create_selective_checkpoint_contexts, policy)), t, x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_compiled_functions_stay_right():
    """The compiler leaves the operators out of its graphs and calls them between."""
    f, t, x = chain()
    want = all_of(f, t, x)
    compiled = torch.compile(f, backend="eager")
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(all_of(compiled, t, x), want))


def elsewhere(t, how):
    """A copy of t whose values lie otherwise in memory."""
    if how == "transposed":
        return t.t().contiguous().t() if t.dim() == 2 else t.clone()
    step = max(1, 2 // t.element_size())
    buf = torch.empty(t.numel() + step, dtype=t.dtype, device=t.device)
    buf[step:] = t.reshape(-1)
    return buf[step:].view(t.shape)


@gpu
@pytest.mark.parametrize("how", ["transposed", "between two accesses"])
def test_saved_tensors_may_come_back_from_elsewhere(how):
    """Hooks on what a backward pass needs may keep it anywhere and hand back a copy."""
    x, wg, wu, dh = gated_case(40, 64, 72, torch.bfloat16, "cuda")
    t, dy, dn = norm_case((40, 64), torch.float32, True, (64,), False, device="cuda")
    freqs, at = ops.rotary_frequencies(16, device="cuda"), torch.arange(40, device="cuda")
    padded = gated_case(40, 65, 72, torch.bfloat16, "cuda")
    inputs = [v.requires_grad_(True) for v in [x, wg, wu] + padded[:3] + list(t.values())]

    def grads():
        outs = ops.gated_linear(x, wg, wu), ops.gated_linear(*padded[:3]), *norm_call(t, 0.5), ops.rotary(x.view(40, 4, 16), None, freqs, at)
        return torch.autograd.grad(outs, inputs, (dh, padded[3], dy, dn, torch.ones(40, 4, 16, device="cuda").bfloat16()))

    plain = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: elsewhere(v, how)):
        got = grads()
    # the norms' sums of a row of 64 fp32 terms have another order where a row starts elsewhere: a few steps of 2^-24 of terms of up to about ten
    for a, b in zip(plain, got):
        assert torch.equal(a, b) if a.dtype is torch.bfloat16 else torch.allclose(a, b, rtol=1e-4, atol=1e-4)


def test_rotary_on_cpu_while_another_device_is_the_default():
    q, freqs = torch.randn(1, 3, 2, 8), ops.rotary_frequencies(8)
    want = ops.rotary(q, None, freqs, 5)
    with torch.device("meta"):
        assert torch.equal(ops.rotary(q, None, freqs, 5), want)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rotary_takes_integers_of_other_classes(device):
    import enum
    first = enum.IntEnum("first", {"five": 5}).five
    q, freqs = torch.randn(1, 3, 2, 8, device=device), ops.rotary_frequencies(8, device=device)
    assert torch.equal(ops.rotary(q, None, freqs, first), ops.rotary(q, None, freqs, 5))
