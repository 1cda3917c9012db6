"""Every tile of the dense products, in every form it is compiled in (plain, rows of single values, gated, transposed operands, FP8), at the ragged shapes of
test_dense_tiles_host.py that select it.  Two kinds of values: integers, whose sums fp32 holds exactly in any order, so that a product lost, counted twice or
put elsewhere is seen for certain; and normal ones against the formula in 64 bits, with the kept pre-activations counted as the fp32 they are."""
import importlib
import math

import pytest
import torch

import test_dense_tiles_host as shapes
from test_gpu_dense import ACT_EVAL, CURVE, SLOPE, act64, dact64, gamma, gated_ref, linear_bounds, quantise_block, randn, tiny_of, u_of, value8, within

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
both = pytest.mark.parametrize("dt", ["bf16", "fp16"])


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


@pytest.fixture(autouse=True)
def no_device_error(mods, dev):
    yield
    assert mods.cukern.device_error(dev) == 0


def test_tables_on_this_device(mods, dev):
    """The tables are those of the GPU at hand (the kernels are still checked below where its SM count makes other choices)."""
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    if sms != shapes.SMS:
        pytest.skip(f"{sms} SMs")
    assert all(want == got for _, want, got in shapes.picks(mods.lib.lib(), sms))


def integers(shape, seed, dev, t):
    """-1, 0 or 1."""
    return torch.randint(-1, 2, shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(t)


def same(got, exact, what):
    """The result is the rounding of the exact sum (every step up to it is exact)."""
    ref = exact.to(got.dtype)
    bad = (got != ref).nonzero()
    assert bad.numel() == 0, f"{what}: {len(bad)} of {got.numel()} values differ, the first at {bad[0].tolist()}: {got[tuple(bad[0])].item()} for {ref[tuple(bad[0])].item()}"


# ------------------------------------------------------------------ forward
@both
@pytest.mark.parametrize("m,n,k", [*shapes.LINEAR, *shapes.LINEAR_ODD])
def test_linear(D, dev, dt, m, n, k):
    t = TYPES[dt]
    x, w, b, r = integers((m, k), 1, dev, t), integers((n, k), 2, dev, t), integers((n,), 3, dev, t), integers((m, n), 4, dev, t)
    same(D.linear_act(x, w, b, None, r), x.double() @ w.double().t() + b.double() + r.double(), "integers")
    x, w, b, r = randn((m, k), 1, dev, t), randn((n, k), 2, dev, t, 1 / math.sqrt(k)), randn((n,), 3, dev, t), randn((m, n), 4, dev, t)
    for act in ("silu", "gelu"):
        y = D.linear_act(x, w, b, act, r)
        ref, bound, _, _ = linear_bounds(x, w, b, act, r, t)
        within(y, ref, bound, act)
        assert torch.equal(y, D.linear_act(x, w, b, act, r))


@both
@pytest.mark.parametrize("m,inter,k", [*shapes.GATED, *shapes.GATED_ODD])
def test_gated(D, dev, dt, m, inter, k):
    t = TYPES[dt]
    x, w = integers((m, k), 1, dev, t), integers((2 * inter, k), 2, dev, t)
    gu = x.double() @ w.double().t()
    same(D.gated_linear(x, w, None), (gu[:, :inter] * gu[:, inter:]), "integers")  # each product below 2^24 too
    same(D.gated_linear(x, w, None, 5.0), gu[:, :inter].clamp(max=5) * gu[:, inter:].clamp(-5, 5), "integers with clamps")
    x, w = randn((m, k), 1, dev, t), randn((2 * inter, k), 2, dev, t, 2 / math.sqrt(k))
    h = D.gated_linear(x, w, "silu", 1.5)
    ref, bound, _ = gated_ref(x, w, "silu", 1.5, t)
    within(h, ref, bound, "silu")
    assert torch.equal(h, D.gated_linear(x, w, "silu", 1.5))


@pytest.mark.parametrize("m,n,k", list(shapes.FP8))
def test_fp8(D, dev, m, n, k):
    t = torch.bfloat16
    # codes of -1, 0 and 1 with scales of 2^-2 .. 2^2: multiples of 2^-4 below 2^4 each, exact sums
    x8, w8 = (integers(s, i, dev, torch.float32).to(torch.float8_e4m3fn).view(torch.uint8) for i, s in ((1, (m, k)), (2, (n, k))))
    g = torch.Generator(device=dev).manual_seed(3)
    xsf = torch.randint(125, 130, (m, k // 32), generator=g, device=dev).to(torch.uint8)
    s8 = torch.randint(125, 130, ((n + 31) // 32, k // 32), generator=g, device=dev).to(torch.uint8)
    b, r = integers((n,), 4, dev, t), integers((m, n), 5, dev, t)
    exact = value8(x8, xsf, 1) @ value8(w8, s8, 32).t()
    same(D.linear_act_q8(x8, xsf, w8, s8, b, None, r), exact + b.double() + r.double(), "integers")
    x8, xsf = quantise_block(randn((m, k), 1, dev, torch.float32) * torch.exp2(torch.arange(m, device=dev) % 7 - 3.0)[:, None], 1)
    w8, s8 = quantise_block(randn((n, k), 2, dev, torch.float32, 1 / math.sqrt(k)), 32)
    b, r = randn((n,), 3, dev, t), randn((m, n), 4, dev, t)
    y = D.linear_act_q8(x8, xsf, w8, s8, b, "silu", r)
    ref, bound, _, _ = linear_bounds(value8(x8, xsf, 1), value8(w8, s8, 32), b, "silu", r, t)
    within(y, ref, bound, "silu")
    assert torch.equal(y, D.linear_act_q8(x8, xsf, w8, s8, b, "silu", r))


def test_fp8_rows_of_single_values(D, dev):
    """An odd number of columns: residual and result rows start anywhere, in the 128- and the 192-column tiles."""
    t = torch.bfloat16
    for m, n, k in ((90, 931, 1920), (1665, 4015, 256)):
        x8, w8 = (integers(s, i, dev, torch.float32).to(torch.float8_e4m3fn).view(torch.uint8) for i, s in ((1, (m, k)), (2, (n, k))))
        one = lambda *s: torch.full(s, 127, device=dev, dtype=torch.uint8)  # noqa: E731
        r = integers((m, n), 5, dev, t)
        exact = x8.view(torch.float8_e4m3fn).double() @ w8.view(torch.float8_e4m3fn).double().t() + r.double()
        same(D.linear_act_q8(x8, one(m, k // 32), w8, one((n + 31) // 32, k // 32), None, None, r), exact, (m, n, k))


# ------------------------------------------------------------------ backward
def rounded(ref, e, u, t):
    return e + u * (ref.abs() + e) + tiny_of(t)


def linear_backward(D, dev, t, m, n, k, acts):
    """z is kept in fp32: it is off by its accumulation (and the bias' addition) alone.  The slope's error is CURVE times that and its evaluation; gy times the
    slope is one fp32 product; dz is rounded to t where an activation makes it, and is gy itself otherwise."""
    u = u_of(t)
    for act in acts:
        x, w = randn((m, k), 1, dev, t).requires_grad_(True), randn((n, k), 2, dev, t, 1 / math.sqrt(k)).requires_grad_(True)
        b, gy = randn((n,), 3, dev, t).requires_grad_(True), randn((m, n), 5, dev, t)
        dx, dw, db = torch.autograd.grad(D.linear_act(x, w, b, act), (x, w, b), gy)
        x64, w64, g = x.detach().double(), w.detach().double(), gy.double()
        _, _, z, ez = linear_bounds(x.detach(), w.detach(), b.detach(), act, None, t)
        dz = g * dact64(act, z)
        if act in (None, "relu"):
            edz = g.abs() * (z.abs() <= ez).double() if act else torch.zeros_like(dz)  # relu: z of either sign
            edz_r = edz
        else:
            edz = g.abs() * (CURVE * ez + ACT_EVAL * (1 + z.abs())) + 2.0 ** -23 * dz.abs()
            edz_r = rounded(dz, edz, u, t)
        ref = dz @ w64
        within(dx, ref, rounded(ref, edz_r @ w64.abs() + gamma(n) * ((dz.abs() + edz_r) @ w64.abs()), u, t), f"dx {act}")
        ref = dz.t() @ x64
        within(dw, ref, rounded(ref, edz_r.t() @ x64.abs() + gamma(m) * ((dz.abs() + edz_r).t() @ x64.abs()), u, t), f"dw {act}")
        ref = dz.sum(0)
        within(db, ref, rounded(ref, edz.sum(0) + gamma(m) * (dz.abs() + edz).sum(0), u, t), f"db {act}")


@both
@pytest.mark.parametrize("m,n,k", [*shapes.BACKWARD, *shapes.BACKWARD_ODD])
def test_linear_backward(D, dev, dt, m, n, k):
    t = TYPES[dt]
    x, w, gy = integers((m, k), 1, dev, t).requires_grad_(True), integers((n, k), 2, dev, t).requires_grad_(True), integers((m, n), 3, dev, t)
    b = integers((n,), 4, dev, t).requires_grad_(True)
    dx, dw, db = torch.autograd.grad(D.linear_act(x, w, b), (x, w, b), gy)
    x64, w64, g = x.detach().double(), w.detach().double(), gy.double()
    same(dx, g @ w64, "dx of integers")
    same(dw, g.t() @ x64, "dw of integers")
    same(db, g.sum(0), "db of integers")
    dx, dw = torch.autograd.grad(D.linear_act(x, w, b, "relu"), (x, w), gy)
    on = (x64 @ w64.t() + b.detach().double() > 0).double()
    same(dx, (g * on) @ w64, "dx of integers, relu")
    same(dw, (g * on).t() @ x64, "dw of integers, relu")
    linear_backward(D, dev, t, m, n, k, ["gelu"])


@both
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (4, 64, 128), (7, 33, 50), (130, 200, 136), (257, 136, 330)])
def test_linear_backward_small(D, dev, dt, m, n, k):
    linear_backward(D, dev, TYPES[dt], m, n, k, [None, "relu", "silu", "gelu", "gelu_tanh"])


def gated_backward(D, dev, t, m, inter, k, cases):
    """g and u are kept in fp32: off by their accumulation alone.  dg = gy u act'(g) and du = gy act(g) take two and one fp32 products more, then a rounding to t."""
    u_ = u_of(t)
    for act, limit in cases:
        x, w = randn((m, k), 1, dev, t).requires_grad_(True), randn((2 * inter, k), 2, dev, t, 2 / math.sqrt(k)).requires_grad_(True)
        gy = randn((m, inter), 3, dev, t)
        dx, dw = torch.autograd.grad(D.gated_linear(x, w, act, limit), (x, w), gy)
        _, _, (g, u, gc, uc, a, eg, eu, ea) = gated_ref(x.detach(), w.detach(), act, limit, t)
        gy64, da = gy.double(), dact64(act, gc)
        pg, pu = ((g <= limit).double(), (u.abs() <= limit).double()) if limit > 0 else (1.0, 1.0)
        dg, du = gy64 * uc * da * pg, gy64 * a * pu
        slope = 0.0 * g if act is None else (ACT_EVAL * (1 + gc.abs()) + (CURVE * eg if act != "relu" else (g.abs() <= eg).double()))
        near_g = ((g - limit).abs() <= eg).double() if limit > 0 else 0.0  # either side of the clamp
        near_u = ((u.abs() - limit).abs() <= eu).double() if limit > 0 else 0.0
        edg = gy64.abs() * (eu * (da.abs() + slope) + uc.abs() * slope) + 2.0 ** -22 * dg.abs() + near_g * gy64.abs() * (da.abs() + slope) * (uc.abs() + eu)
        edu = gy64.abs() * ea + 2.0 ** -23 * du.abs() + near_u * gy64.abs() * (a.abs() + ea)
        d, e = torch.cat([dg, du], 1), torch.cat([edg, edu], 1)
        e = rounded(d, e, u_, t)
        x64, w64 = x.detach().double(), w.detach().double()
        ref = d @ w64
        within(dx, ref, rounded(ref, e @ w64.abs() + gamma(2 * inter) * ((d.abs() + e) @ w64.abs()), u_, t), f"dx {act} {limit}")
        ref = d.t() @ x64
        within(dw, ref, rounded(ref, e.t() @ x64.abs() + gamma(m) * ((d.abs() + e).t() @ x64.abs()), u_, t), f"dw {act} {limit}")


@both
@pytest.mark.parametrize("m,inter,k", [(1, 8, 16), (3, 5, 7), (64, 129, 72), (130, 264, 256), (2001, 1160, 776)])
def test_gated_backward(D, dev, dt, m, inter, k):
    gated_backward(D, dev, TYPES[dt], m, inter, k, [("silu", 0.0), ("silu", 1.5), ("gelu_tanh", 2.0), ("relu", 1.0), (None, 0.0)] if m < 1000 else [("silu", 1.5)])


@both
@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (16, 129, 200), (90, 930, 1472), (130, 131, 330), (1500, 2056, 776)])
def test_kept_preactivations(D, dev, dt, m, n, k):
    """What a backward pass gets of z, g and u is off by their accumulation alone: fp32, not a rounding to 16 bits, which is 2^14 times that of fp32."""
    t = TYPES[dt]
    x, w, b = randn((m, k), 1, dev, t).requires_grad_(True), randn((2 * n, k), 2, dev, t, 1 / math.sqrt(k)).requires_grad_(True), randn((2 * n,), 3, dev, t)
    for f, bias in ((lambda: D.linear_act(x, w, b, "silu"), b), (lambda: D.gated_linear(x, w, limit=0.5), None)):
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v) or v, lambda v: v):
            f()
        z = [v for v in kept if v.dtype == torch.float32]
        assert len(z) == 1 and z[0].shape[0] == m
        _, _, z64, ez = linear_bounds(x.detach(), w.detach(), bias, None, None, t)
        within(z[0][:, :2 * n], z64, ez, "kept values")


# ------------------------------------------------------------------ one row
@both
def test_one_dimensional_input(D, dev, dt):
    """x [K] is one row, whose kernel is another than that of ten."""
    t = TYPES[dt]
    x, w, b, r = randn((264,), 1, dev, t), randn((40, 264), 2, dev, t, 1 / 16), randn((40,), 3, dev, t), randn((40,), 4, dev, t)
    y = D.linear_act(x, w, b, "silu", r)
    ref, bound, _, _ = linear_bounds(x[None], w, b, "silu", r[None], t)
    assert y.shape == (40,)
    within(y[None], ref, bound, "x [K]")
    h = D.gated_linear(x, w, "silu", 1.5)
    ref, bound, _ = gated_ref(x[None], w, "silu", 1.5, t)
    assert h.shape == (20,)
    within(h[None], ref, bound, "gated, x [K]")


def test_sums_fit_fp32():
    """What the integer tests rest on: |sum| <= the length of the contraction < 2^24, gated products of two sums of up to 5600 below 2^24 where random signs leave
    them (9 standard deviations of 0.67 sqrt(5600) each, squared), FP8 terms of at most 2^4 in steps of 2^-4."""
    longest = max(k for t in (shapes.LINEAR, shapes.LINEAR_ODD, shapes.GATED, shapes.GATED_ODD) for _, _, k in t)
    assert longest < 2 ** 24 and max(max(s) for t in (shapes.BACKWARD, shapes.BACKWARD_ODD) for s in t) < 2 ** 24
    assert (9 * 0.67 * math.sqrt(5600)) ** 2 < 2 ** 24
    assert max(k for _, _, k in shapes.FP8) * 2 ** 4 * 2 ** 4 < 2 ** 24


@both
@pytest.mark.parametrize("m", [8, 400])
def test_gelu_tail(D, dev, dt, m):
    """gelu of -12 .. 4 through an identity weight: Phi is off by 0.75e-7 at most and by 5 % at most below -8, and z Phi(z) is rounded once."""
    t = TYPES[dt]
    z = torch.linspace(-12, 4, m * 8, device=dev).to(t).view(m, 8)
    y = D.linear_act(z, torch.eye(8, device=dev, dtype=t), None, "gelu").double()
    z = z.double()
    ref = z * 0.5 * torch.erfc(-z / math.sqrt(2))  # 1 + erf would cancel, in 64 bits too: off by 1e-16, more than the values from z = -8.3 on
    e = z.abs() * 0.75e-7 + 2.0 ** -20 * ref.abs()
    e = torch.where(z < -8, torch.minimum(e, 0.05 * ref.abs()), e)
    within(y, ref, u_of(t) * (ref.abs() + e) + e + tiny_of(t), "gelu")
