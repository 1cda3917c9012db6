"""The dense feed-forward operators (norm with residual, projection with bias / activation / residual, gated projection, FP8 forms) against
their formulas in 64 bits.  Bounds count roundings: u = half a step of the result's type for each value that is stored, 2^-23 per addition of a
sum relative to the sum of magnitudes (the tensor cores may truncate), and what the formula makes of the error of a stored intermediate."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


def u_of(t):
    return torch.finfo(t).eps / 2


def tiny_of(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps  # the smallest subnormal: results below the normal range


def act64(name, z):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def dact64(name, z):
    z = z.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act64(name, z).sum(), z)[0]


# |act'| <= 1.13 and |act''| <= 1.0 for all of them (silu: 1.10, 0.5; gelu: 1.13, 0.80; gelu_tanh: 1.13, 0.80; relu: its slope does not change
# under a rounding of z, which keeps z's sign)
SLOPE, CURVE = 1.13, 1.0
# the activations are evaluated in fp32 with a handful of roundings and special-function results of 2 ulp each, relative to |z| (+ 1 for the slope)
ACT_EVAL = 2.0 ** -19


def within(got, ref, bound, what=""):
    got = got.detach().double().cpu()
    ref, bound = ref.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    worst = ((got - ref).abs() - bound).max().item() if got.numel() else 0.0
    ratio = ((got - ref).abs() / bound.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 0, f"{what}: error / bound up to {ratio:.3g}"


def randn(shape, seed, dev, dtype, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


# ------------------------------------------------------------------ norm
SUM_REL = 2.0 ** -18  # a mean of positive squares: 64 additions at most in a row (serial part of a thread + trees), rsqrt, products: < 64 * 2^-24


def norm64(x, r, w, eps):
    s = x.double() + (r.double() if r is not None else 0)
    n = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    return s, n, n * (w.double() if w is not None else 1)


NORM_SHAPES = [(1, 4096), (5, 1), (3, 7), (4, 32), (9, 250), (7, 512), (2, 1000), (3, 4097), (6, 5120), (2, 8192), (2, 8200), (3, 16384), (700, 64), (1500, 264), (400, 5120), (310, 8192)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm_forward_backward(D, dev, dt, rows, dim):
    t = TYPES[dt]
    for wt, with_res in ((t, True), (torch.float32, True), (t, False), (None, True)):
        x = randn((rows, dim), 1, dev, t).requires_grad_(True)
        r = randn((rows, dim), 2, dev, t, 2.0).requires_grad_(True) if with_res else None
        w = (1 + randn((dim,), 3, dev, torch.float32, 0.2)).to(wt).requires_grad_(True) if wt else None
        y, s = D.add_rms_norm(x, r, w, 1e-5)
        s64, n64, y64 = norm64(x.detach(), r.detach() if r is not None else None, w.detach() if w is not None else None, 1e-5)
        within(y, y64, (u_of(t) + SUM_REL) * y64.abs() + tiny_of(t), "y")
        if with_res:
            within(s, s64, u_of(t) * (1 + 2.0 ** -10) * s64.abs() + 2.0 ** -24 * s64.abs() + tiny_of(t), "s")
        else:
            assert s is x
        gy, gs = randn((rows, dim), 4, dev, t), randn((rows, dim), 5, dev, t)
        leaves = [v for v in (x, r, w) if v is not None]
        grads = dict(zip([n for n, v in (("x", x), ("r", r), ("w", w)) if v is not None],
                         torch.autograd.grad((y, s) if with_res else (y,), leaves, (gy, gs) if with_res else (gy,))))
        w64 = w.detach().double() if w is not None else torch.ones(dim, device=dev, dtype=torch.float64)
        h = gy.double() * w64
        rinv = 1 / torch.sqrt(s64.square().mean(-1, keepdim=True) + 1e-5)
        ds = rinv * (h - n64 * (h * n64).mean(-1, keepdim=True)) + (gs.double() if with_res else 0)
        scale = rinv * (h.abs() + n64.abs() * (h * n64).abs().mean(-1, keepdim=True))
        b = u_of(t) * ds.abs() + 4 * SUM_REL * scale + tiny_of(t) + (2.0 ** -23 * gs.double().abs() if with_res else 0)
        within(grads["x"], ds, b, "dx")
        if with_res:
            assert torch.equal(grads["r"], grads["x"])
        if w is not None:
            dw = (gy.double() * n64).sum(0)
            mag = (gy.double() * n64).abs().sum(0)
            within(grads["w"], dw, u_of(wt) * dw.abs() + (2 * SUM_REL + rows * 2.0 ** -23) * mag + tiny_of(wt), "dw")


def test_norm_gradients_against_differences(D, dev):
    x, r = randn((3, 40), 11, dev, torch.float32).requires_grad_(True), randn((3, 40), 12, dev, torch.float32).requires_grad_(True)
    w = (1 + randn((40,), 13, dev, torch.float32, 0.3)).requires_grad_(True)
    gy, gs = randn((3, 40), 14, dev, torch.float32), randn((3, 40), 15, dev, torch.float32)
    y, s = D.add_rms_norm(x, r, w, 1e-6)
    grads = torch.autograd.grad((y, s), (x, r, w), (gy, gs))

    def loss(a, b, c):
        s64, _, y64 = norm64(a, b, c, 1e-6)
        return ((y64 * gy.double()).sum() + (s64 * gs.double()).sum()).item()

    vals = [v.detach().double() for v in (x, r, w)]
    for i in range(3):
        d = torch.randn(vals[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(dev)
        h = 1e-4
        up, dn = list(vals), list(vals)
        up[i], dn[i] = vals[i] + h * d, vals[i] - h * d
        num = (loss(*up) - loss(*dn)) / (2 * h)
        got = (grads[i].double() * d).sum().item()
        # central differences: h^2 = 1e-8 times third derivatives of order 10, and fp32 gradients
        assert abs(num - got) <= 1e-5 * (grads[i].double().abs() * d.abs()).sum().item()


def check_codes(q8, sf, y64, scale_rel):
    """codes and scales against the 64-bit y: the scale is the smallest power of two that fits (either neighbour where the largest value of the group lies
    within scale_rel of the border), every code the nearest e4m3 value up to that relative error."""
    rows, dim = y64.shape
    v8 = q8.view(torch.float8_e4m3fn).double()
    e = sf.double() - 127
    amax = y64.view(rows, -1, 32).abs().amax(-1).clamp_min(1e-4)
    fits = lambda a: torch.ceil(torch.log2(a / 448) - 1e-12)  # noqa: E731
    lo, hi = fits(amax * (1 - scale_rel)), fits(amax * (1 + scale_rel))
    assert ((e >= lo) & (e <= hi)).all()
    v = y64 / torch.exp2(e).repeat_interleave(32, 1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(2.0 ** -6, 448))) - 3)
    assert ((v8 - v.clamp(-448, 448)).abs() <= step / 2 * (1 + 1e-9) + scale_rel * v.abs()).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,dim", [(1, 4096), (3, 32), (70, 96), (5, 1024), (4099, 160), (2, 5120), (2, 16384), (400, 4128), (330, 8192)])
def test_norm_quant(D, dev, dt, rows, dim):
    t = TYPES[dt]
    x, r = randn((rows, dim), 21, dev, t), randn((rows, dim), 22, dev, t)
    w = 1 + randn((dim,), 23, dev, torch.float32, 0.5)
    q8, sf, s, y = D.add_rms_norm_quant(x, r, w, 1e-6, want_y=True)
    assert q8.shape == (rows, dim) and sf.shape == (rows, dim // 32) and q8.dtype == sf.dtype == torch.uint8
    s64, _, y64 = norm64(x, r, w, 1e-6)
    check_codes(q8, sf, y64, SUM_REL)
    y2, s2 = D.add_rms_norm(x, r, w, 1e-6)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    q8b, sfb, _ = D.add_rms_norm_quant(x, r, w, 1e-6)
    assert torch.equal(q8, q8b) and torch.equal(sf, sfb)
    q8c, sfc, sc = D.add_rms_norm_quant(s, None, w, 1e-6)  # no residual
    assert sc is s
    check_codes(q8c, sfc, norm64(s, None, w, 1e-6)[2], SUM_REL)


def test_norm_special_rows(D, dev):
    x = randn((6, 128), 31, dev, torch.bfloat16)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4, 64:] = 0  # groups of zeros beside groups of values
    ref = D.add_rms_norm(x[[0, 5]].contiguous(), None, None, 1e-6)[0]
    y, _ = D.add_rms_norm(x, None, None, 1e-6)
    assert torch.equal(y[[0, 5]], ref) and (y[1] == 0).all() and y[3].isnan().all()
    assert y[2, 5].isnan() and (y[2, :5] == 0).all()  # x / inf = 0, inf / inf = NaN
    q8, sf, _ = D.add_rms_norm_quant(x, None, None, 1e-6)
    v = q8.view(torch.float8_e4m3fn).float()
    assert (v[1] == 0).all() and (v[4, 64:] == 0).all() and v[3].isnan().all()
    # a group of zeros takes the scale of the floor 1e-4: the smallest 2^e with 1e-4 / 2^e <= 448
    assert (sf[1].int() == 127 + math.ceil(math.log2(1e-4 / 448))).all()


def test_norm_strides_and_shapes(D, dev):
    big, rbig = randn((12, 200), 41, dev, torch.bfloat16), randn((12, 200), 42, dev, torch.bfloat16)
    w = randn((96,), 43, dev, torch.bfloat16)
    for sl in (slice(0, 96), slice(8, 104), slice(3, 99)):  # aligned rows, aligned offset, odd offset
        a, b = big[:, sl], rbig[:, sl]
        y, s = D.add_rms_norm(a, b, w, 1e-6)
        y2, s2 = D.add_rms_norm(a.contiguous(), b.contiguous(), w, 1e-6)
        assert torch.equal(s, s2)  # another vector width adds the squares in another order: a rounding of y may differ
        within(y, y2, u_of(torch.bfloat16) * 2 * y2.double().abs() + 1e-30)
        q, f, _ = D.add_rms_norm_quant(a, b, w, 1e-6)
        check_codes(q, f, norm64(a, b, w, 1e-6)[2], SUM_REL)
    x3 = randn((2, 3, 96), 44, dev, torch.bfloat16)
    y3, _ = D.add_rms_norm(x3, None, w, 1e-6)
    assert y3.shape == x3.shape and torch.equal(y3.view(6, 96), D.add_rms_norm(x3.view(6, 96), None, w, 1e-6)[0])
    xt = randn((96, 5), 45, dev, torch.bfloat16).t()  # inner stride 5
    assert torch.equal(D.add_rms_norm(xt, None, w)[0], D.add_rms_norm(xt.contiguous(), None, w)[0])
    xe = randn((1, 96), 46, dev, torch.bfloat16).expand(4, 96)  # one row for all
    assert torch.equal(D.add_rms_norm(xe, None, w)[0], D.add_rms_norm(xe.contiguous(), None, w)[0])
    assert D.add_rms_norm(x3[:, :0], None, w)[0].shape == (2, 0, 96)
    assert D.add_rms_norm_quant(x3[:, :0], None, w)[0].shape == (0, 96)


def test_norm_partial_gradients(D, dev):
    x, r = (randn((4, 64), s, dev, torch.bfloat16).requires_grad_(True) for s in (51, 52))
    w = randn((64,), 53, dev, torch.float32).requires_grad_(True)
    gy = randn((4, 64), 54, dev, torch.bfloat16)
    y, s = D.add_rms_norm(x, r, w)
    full = torch.autograd.grad(y, (x, r, w), gy, retain_graph=True)
    assert torch.equal(torch.autograd.grad(s, x, gy, retain_graph=True)[0], gy)  # the sum alone
    y2, _ = D.add_rms_norm(x.detach(), r, w)
    assert torch.equal(torch.autograd.grad(y2, r, gy)[0], full[1])
    y3, _ = D.add_rms_norm(x, r.detach(), w.detach())
    assert torch.equal(torch.autograd.grad(y3, x, gy)[0], full[0])
    # leaves that accumulate: the shared gradient tensor is not changed through the other leaf
    for _ in range(2):
        y, s = D.add_rms_norm(x, r, w)
        torch.autograd.backward((y,), (gy,))
    assert torch.equal(x.grad, (full[0].float() * 2).to(torch.bfloat16)) and torch.equal(r.grad, x.grad)
    xe = randn((1, 64), 55, dev, torch.float32).requires_grad_(True)  # a broadcast input
    ye, _ = D.add_rms_norm(xe.expand(4, 64), None, w)
    ge = torch.autograd.grad(ye, xe, gy.float())[0]
    each = torch.autograd.grad(D.add_rms_norm(xe, None, w)[0], xe, gy.float().sum(0, keepdim=True))[0]
    within(ge, each, 1e-5 * each.double().abs().max().expand_as(each))


# ------------------------------------------------------------------ projection
def gamma(k):
    return (k + 8) * 2.0 ** -23


def linear_bounds(x, w, b, act, r, t):
    """(reference, bound, z64, bound of z before its rounding)."""
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    ez = gamma(x.shape[1]) * mag
    if b is not None:
        z = z + b.double()
        ez = ez + 2.0 ** -23 * (mag + b.double().abs())
    y = act64(act, z)
    e = SLOPE * ez + ACT_EVAL * z.abs()
    if r is not None:
        y = y + r.double()
        e = e + 2.0 ** -23 * (z.abs() + r.double().abs())
    return y, u_of(t) * (y.abs() + e) + e + tiny_of(t), z, ez


LINEAR_SHAPES = [(1, 8, 8), (1, 1, 1), (1, 4096, 2048), (2, 300, 77), (3, 128, 64), (5, 130, 1000), (8, 256, 512), (9, 264, 328), (16, 512, 4096), (17, 136, 520), (32, 200, 192),
                 (33, 1001, 230), (64, 384, 1024), (100, 257, 200), (129, 260, 136), (130, 256, 2000), (257, 640, 72), (300, 2048, 576), (1000, 96, 40)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
def test_linear_act_forward(D, dev, dt, m, n, k):
    t = TYPES[dt]
    x, w = randn((m, k), 1, dev, t), randn((n, k), 2, dev, t, 1 / math.sqrt(k))
    b, r = randn((n,), 3, dev, t), randn((m, n), 4, dev, t)
    for i, act in enumerate(ACTS):
        bb, rr = (b if i != 1 else None), (r if i % 2 == 0 else None)
        y = D.linear_act(x, w, bb, act, rr)
        ref, bound, _, _ = linear_bounds(x, w, bb, act, rr, t)
        within(y, ref, bound, f"{act}")
        assert torch.equal(y, D.linear_act(x, w, bb, act, rr))  # the same from run to run


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (4, 64, 128), (7, 33, 50), (64, 128, 64), (130, 200, 136), (200, 1001, 72), (257, 136, 330), (512, 384, 256)])
def test_linear_act_backward(D, dev, dt, m, n, k):
    t = TYPES[dt]
    u = u_of(t)
    for i, act in enumerate(ACTS):
        x, w = randn((m, k), 1, dev, t).requires_grad_(True), randn((n, k), 2, dev, t, 1 / math.sqrt(k)).requires_grad_(True)
        b, r = randn((n,), 3, dev, t).requires_grad_(True), randn((m, n), 4, dev, t).requires_grad_(True)
        gy = randn((m, n), 5, dev, t)
        y = D.linear_act(x, w, b, act, r)
        dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), gy)
        ref, bound, z, ez = linear_bounds(x.detach(), w.detach(), b.detach(), act, r.detach(), t)
        within(y, ref, bound, "y")
        assert torch.equal(dr, gy)
        g = gy.double()
        dz = g * dact64(act, z)
        if act is None:
            edz = torch.zeros_like(dz)
        else:  # the stored z is off by ez + u |z|, the slope by CURVE times that and its evaluation; then dz is rounded
            slope_err = (0.0 if act == "relu" else CURVE) * (ez + u * z.abs() + tiny_of(t)) + ACT_EVAL * (1 + z.abs())
            if act == "relu":
                slope_err = slope_err + (z.abs() <= ez + tiny_of(t)).double()  # z of either sign
            edz = g.abs() * slope_err
        edz_r = edz + (u * (dz.abs() + edz) + tiny_of(t) if act is not None else 0)
        x64, w64 = x.detach().double(), w.detach().double()
        ref_dx, ref_dw = dz @ w64, dz.t() @ x64
        within(dx, ref_dx, (lambda e: e + u * (ref_dx.abs() + e) + tiny_of(t))(edz_r @ w64.abs() + gamma(n) * ((dz.abs() + edz_r) @ w64.abs())), f"dx {act}")
        within(dw, ref_dw, (lambda e: e + u * (ref_dw.abs() + e) + tiny_of(t))(edz_r.t() @ x64.abs() + gamma(m) * ((dz.abs() + edz_r).t() @ x64.abs())), f"dw {act}")
        ref_db = dz.sum(0)
        within(db, ref_db, (lambda e: e + u * (ref_db.abs() + e) + tiny_of(t))(edz.sum(0) + gamma(m) * (dz.abs() + edz).sum(0)), f"db {act}")


def test_linear_gradients_against_differences(D, dev):
    """The direction derivative of the 64-bit formula against the kernel's gradients: they are rounded to 11 bits, sums of k of them with random
    signs stay within a few roundings of the sum of magnitudes."""
    m, n, k = 33, 40, 56
    x, w, b = (randn(s, i, dev, torch.float16, 0.5).requires_grad_(True) for i, s in enumerate(((m, k), (n, k), (n,))))
    gy = randn((m, n), 9, dev, torch.float16)
    for act in ("silu", "gelu", "gelu_tanh"):
        grads = torch.autograd.grad(D.linear_act(x, w, b, act), (x, w, b), gy)
        vals = [v.detach().double() for v in (x, w, b)]
        loss = lambda a, c, d: (act64(act, a @ c.t() + d) * gy.double()).sum().item()  # noqa: E731
        for i in range(3):
            d = torch.randn(vals[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(dev)
            up, dn = list(vals), list(vals)
            up[i], dn[i] = vals[i] + 1e-5 * d, vals[i] - 1e-5 * d
            num, got = (loss(*up) - loss(*dn)) / 2e-5, (grads[i].double() * d).sum().item()
            assert abs(num - got) <= 4 * u_of(torch.float16) * (grads[i].double().abs() * d.abs()).sum().item()


def test_linear_strides(D, dev):
    t = torch.bfloat16
    xb, wb, rb = randn((40, 300), 1, dev, t), randn((72, 300), 2, dev, t, 0.1), randn((40, 100), 3, dev, t)
    for xo, wo, ro in ((0, 0, 0), (8, 16, 8), (3, 8, 1), (8, 5, 0)):
        x, w, r = xb[:, xo:xo + 256], wb[:, wo:wo + 256], rb[:, ro:ro + 72]
        assert torch.equal(D.linear_act(x, w, None, "silu", r), D.linear_act(x.contiguous(), w.contiguous(), None, "silu", r.contiguous()))
    x3 = randn((2, 5, 64), 4, dev, t)
    w = randn((24, 64), 5, dev, t)
    y3 = D.linear_act(x3, w)
    assert y3.shape == (2, 5, 24) and torch.equal(y3.view(10, 24), D.linear_act(x3.view(10, 64), w))
    assert torch.equal(D.linear_act(x3[0, 0], w), y3[0, 0]) or D.linear_act(x3[0, 0], w).shape == (24,)
    wt = randn((64, 24), 6, dev, t).t()
    assert torch.equal(D.linear_act(x3, wt), D.linear_act(x3, wt.contiguous()))
    assert D.linear_act(x3[:0], w).shape == (0, 5, 24)
    xe = x3[:1, :1].expand(3, 4, 64)
    assert torch.equal(D.linear_act(xe, w), D.linear_act(xe.contiguous(), w))
    # gradients of rows that had to be copied, and of a gradient that arrives expanded
    xo = xb[:, 3:53].detach().requires_grad_(True)
    wo = wb[:, 5:55].detach().requires_grad_(True)
    dx, dw = torch.autograd.grad(D.linear_act(xo, wo, None, "gelu").sum(), (xo, wo))
    xc, wc = xo.detach().contiguous().requires_grad_(True), wo.detach().contiguous().requires_grad_(True)
    dx2, dw2 = torch.autograd.grad(D.linear_act(xc, wc, None, "gelu"), (xc, wc), torch.ones(40, 72, device=dev, dtype=t))
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    # no rows: gradients of weight and bias are zeros
    b0 = randn((24,), 7, dev, t).requires_grad_(True)
    w0 = w.detach().requires_grad_(True)
    g = torch.autograd.grad(D.linear_act(x3[:0], w0, b0, "silu").sum(), (w0, b0))
    assert (g[0] == 0).all() and (g[1] == 0).all() and g[0].shape == w0.shape


def test_linear_special_values(D, dev):
    x, w = randn((5, 64), 1, dev, torch.bfloat16), randn((40, 64), 2, dev, torch.bfloat16)
    ref = D.linear_act(x, w, None, "relu")
    x2 = x.clone()
    x2[1, 3], x2[3, 0] = float("nan"), float("inf")
    y = D.linear_act(x2, w, None, "relu")
    assert torch.equal(y[[0, 2, 4]], ref[[0, 2, 4]]) and y[1].isnan().all()
    assert ((y[3] == float("inf")) | (y[3] == 0)).all() and torch.equal(y[3] > 0, w[:, 0] > 0)
    big = torch.full((1, 8), 200.0, device=dev, dtype=torch.bfloat16)  # activations at both ends
    one = torch.cat([torch.ones(1, 8), -torch.ones(1, 8)]).to(dev, torch.bfloat16)
    for act in ("silu", "gelu", "gelu_tanh"):
        v = D.linear_act(big, one, None, act).float()[0].tolist()
        assert v[0] == 1600.0 and v[1] == 0.0, (act, v)


def test_offsets_past_32_bits(D, dev):
    """Rows whose element offsets pass 2^31, in x, the residual, the norm's inputs and the weights."""
    m, ld = 140000, 16384
    buf = torch.empty(m, ld, device=dev, dtype=torch.bfloat16)
    r, xs = buf[:, 16000:16008], buf[:, 8000:8064]
    r.copy_(randn((m, 8), 1, dev, torch.bfloat16))
    x, w = randn((m, 64), 2, dev, torch.bfloat16), randn((8, 64), 3, dev, torch.bfloat16, 0.1)
    assert torch.equal(D.linear_act(x, w, None, None, r), D.linear_act(x, w, None, None, r.contiguous()))
    xs.copy_(x)
    assert torch.equal(D.linear_act(xs, w), D.linear_act(x, w))
    assert torch.equal(D.add_rms_norm(xs, xs)[0], D.add_rms_norm(x, x)[0])
    xg, xsg = x.clone().requires_grad_(True), xs.detach().requires_grad_(True)
    gy = randn((m, 64), 4, dev, torch.bfloat16)
    assert torch.equal(torch.autograd.grad(D.add_rms_norm(xg)[0], xg, gy)[0], torch.autograd.grad(D.add_rms_norm(xsg)[0], xsg, gy)[0])
    del buf, r, xs, xsg
    n, k = 600000, 4096
    big = torch.empty(n, k, device=dev, dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, 31, 300000, 524288, 524289, 599998, 599999], device=dev)
    big[rows] = randn((8, k), 5, dev, torch.bfloat16, 1 / 64)
    for m in (2, 12, 40):  # streaming kernel, streaming kernel with two groups of rows, tensor cores
        x = randn((m, k), 6, dev, torch.bfloat16)
        ref, bound, _, _ = linear_bounds(x, big[rows], None, None, None, torch.bfloat16)
        within(D.linear_act(x, big)[:, rows], ref, bound, f"m {m}")


# ------------------------------------------------------------------ gated projection
def gated_ref(x, w13, act, limit, t):
    inter = w13.shape[0] // 2
    gu = x.double() @ w13.double().t()
    egu = gamma(x.shape[1]) * (x.double().abs() @ w13.double().abs().t())
    g, u = gu[:, :inter], gu[:, inter:]
    eg, eu = egu[:, :inter], egu[:, inter:]
    gc, uc = (g.clamp(max=limit), u.clamp(-limit, limit)) if limit > 0 else (g, u)
    a = act64(act, gc)
    h = a * uc
    ea = SLOPE * eg + ACT_EVAL * gc.abs()
    e = ea * (uc.abs() + eu) + a.abs() * eu + 2.0 ** -23 * h.abs()
    return h, u_of(t) * (h.abs() + e) + e + tiny_of(t), (g, u, gc, uc, a, eg, eu, ea)


GATED_SHAPES = [(1, 8, 16), (1, 2048, 4096), (2, 1, 3), (4, 100, 64), (8, 256, 512), (9, 136, 200), (16, 72, 4096), (33, 200, 130), (64, 129, 72), (130, 264, 256), (257, 512, 136), (300, 96, 1000)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("m,inter,k", GATED_SHAPES)
def test_gated_forward(D, dev, dt, m, inter, k):
    t = TYPES[dt]
    x, w = randn((m, k), 1, dev, t), randn((2 * inter, k), 2, dev, t, 2 / math.sqrt(k))
    for act, limit in (("silu", 0.0), ("silu", 1.5), ("gelu", 0.0), ("gelu_tanh", 2.0), ("relu", 0.0), (None, 1.0)):
        h = D.gated_linear(x, w, act, limit)
        ref, bound, _ = gated_ref(x, w, act, limit, t)
        within(h, ref, bound, f"{act} {limit}")
        assert torch.equal(h, D.gated_linear(x, w, act, limit))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("m,inter,k", [(1, 8, 16), (3, 5, 7), (9, 136, 200), (64, 129, 72), (130, 264, 256), (300, 96, 330)])
def test_gated_backward(D, dev, dt, m, inter, k):
    t = TYPES[dt]
    u_ = u_of(t)
    for act, limit in (("silu", 0.0), ("silu", 1.5), ("gelu", 0.0), ("gelu_tanh", 2.0), ("relu", 1.0), (None, 0.0)):
        x, w = randn((m, k), 1, dev, t).requires_grad_(True), randn((2 * inter, k), 2, dev, t, 2 / math.sqrt(k)).requires_grad_(True)
        gy = randn((m, inter), 3, dev, t)
        h = D.gated_linear(x, w, act, limit)
        dx, dw = torch.autograd.grad(h, (x, w), gy)
        assert torch.equal(h, D.gated_linear(x.detach(), w.detach(), act, limit))  # keeping g and u changes nothing
        _, _, (g, u, gc, uc, a, eg, eu, ea) = gated_ref(x.detach(), w.detach(), act, limit, t)
        gy64, da = gy.double(), dact64(act, gc)
        pg, pu = ((g <= limit).double(), (u.abs() <= limit).double()) if limit > 0 else (torch.ones_like(g), torch.ones_like(u))
        dg, du = gy64 * uc * da * pg, gy64 * a * pu
        # stored g and u: off by eg + 2 u |g| (one rounding; next to the limit the clamp moves a value by at most another)
        sg, su = eg + 2 * u_ * gc.abs() + tiny_of(t), eu + 2 * u_ * uc.abs() + tiny_of(t)
        slope = (0.0 if act in ("relu", None) else CURVE) * sg + (ACT_EVAL * (1 + gc.abs()) if act else 0)
        if act == "relu":
            slope = slope + (g.abs() <= eg + tiny_of(t)).double()
        near_g = ((g - limit).abs() <= eg).double() if limit > 0 else 0  # either side of the clamp
        near_u = ((u.abs() - limit).abs() <= eu).double() if limit > 0 else 0
        edg = gy64.abs() * (su * (da.abs() + slope) + uc.abs() * slope) * 1.01 + near_g * gy64.abs() * 1.2 * (uc.abs() + su)
        edu = gy64.abs() * (SLOPE * sg + ACT_EVAL * gc.abs()) * 1.01 + near_u * gy64.abs() * 1.2 * (gc.abs() + sg)
        d, e = torch.cat([dg, du], 1), torch.cat([edg, edu], 1)
        e = e + u_ * (d.abs() + e) + tiny_of(t)
        x64, w64 = x.detach().double(), w.detach().double()
        rdx, rdw = d @ w64, d.t() @ x64
        within(dx, rdx, (lambda b: b + u_ * (rdx.abs() + b) + tiny_of(t))(e @ w64.abs() + gamma(2 * inter) * ((d.abs() + e) @ w64.abs())), f"dx {act} {limit}")
        within(dw, rdw, (lambda b: b + u_ * (rdw.abs() + b) + tiny_of(t))(e.t() @ x64.abs() + gamma(m) * ((d.abs() + e).t() @ x64.abs())), f"dw {act} {limit}")


def test_gated_gradients_against_differences(D, dev):
    m, inter, k = 20, 24, 40
    x, w = randn((m, k), 1, dev, torch.float16, 0.5).requires_grad_(True), randn((2 * inter, k), 2, dev, torch.float16, 0.3).requires_grad_(True)
    gy = randn((m, inter), 3, dev, torch.float16)
    grads = torch.autograd.grad(D.gated_linear(x, w, "silu"), (x, w), gy)
    vals = [x.detach().double(), w.detach().double()]

    def loss(a, c):
        gu = a @ c.t()
        return (act64("silu", gu[:, :inter]) * gu[:, inter:] * gy.double()).sum().item()

    for i in range(2):
        d = torch.randn(vals[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(dev)
        up, dn = list(vals), list(vals)
        up[i], dn[i] = vals[i] + 1e-5 * d, vals[i] - 1e-5 * d
        num, got = (loss(*up) - loss(*dn)) / 2e-5, (grads[i].double() * d).sum().item()
        assert abs(num - got) <= 4 * u_of(torch.float16) * (grads[i].double().abs() * d.abs()).sum().item()


def test_gated_clamp_borders(D, dev):
    """Values that lie on the limit pass their gradient, values above it do not, whatever the 16-bit rounding of the kept g and u does: with an identity
    weight g and u are inputs."""
    for t, limit in ((torch.bfloat16, 1.5), (torch.bfloat16, 1.503), (torch.float16, 1.503), (torch.float16, 10.0)):
        eps = torch.finfo(t).eps
        base = torch.tensor([limit], dtype=torch.float64)
        vals = torch.cat([base * (1 + k * eps) for k in (-3, -2, -1, -0.5, 0, 0.5, 1, 2, 3)] + [-base * (1 + k * eps) for k in (-2, -1, 0, 1, 2)]).to(dev, t)
        m = vals.numel()
        x = torch.zeros(m, 16, device=dev, dtype=t)
        x[:, 0], x[:, 1] = vals, vals.flip(0)
        w = torch.zeros(2, 16, device=dev, dtype=t)
        w[0, 0], w[1, 1] = 1, 1
        x.requires_grad_(True)
        h = D.gated_linear(x, w, None, limit)
        dx = torch.autograd.grad(h, x, torch.ones_like(h))[0].double()
        g, u = x.detach()[:, 0].double(), x.detach()[:, 1].double()
        lim32 = float(torch.tensor(limit, dtype=torch.float32))
        pg, pu = (g <= lim32), (u.abs() <= lim32)
        assert torch.equal(dx[:, 0] != 0, pg) and torch.equal(dx[:, 1] != 0, pu), (t, limit)


# ------------------------------------------------------------------ FP8 projection
def quantise_block(v, rows):
    n, k = v.shape
    nb = -(-n // rows)
    full = torch.zeros(nb * rows, k, device=v.device)
    full[:n] = v
    b = full.view(nb, rows, k // 32, 32)
    e = torch.ceil(torch.log2(b.abs().amax(dim=(1, 3)).clamp_min(1e-4) / 448) - 1e-6)
    q = (b / torch.exp2(e)[:, None, :, None]).clamp(-448, 448).view(nb * rows, k)[:n]
    return q.to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), (e + 127).to(torch.uint8).contiguous()


def value8(q, s, rows):
    return q.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127).repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(32, 1)


@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 4096, 4096), (3, 100, 256), (8, 4096, 2048), (9, 512, 640), (16, 33, 1152), (17, 300, 128), (40, 272, 384), (64, 256, 512), (65, 160, 256),
                                   (130, 264, 384), (300, 1000, 640), (520, 512, 1024)])
def test_linear_act_q8(D, dev, m, n, k):
    t = torch.bfloat16
    x8, xsf = quantise_block(randn((m, k), 1, dev, torch.float32) * torch.exp2(torch.arange(m, device=dev) % 7 - 3.0)[:, None], 1)
    w8, s8 = quantise_block(randn((n, k), 2, dev, torch.float32, 1 / math.sqrt(k)), 32)
    b, r = randn((n,), 3, dev, t), randn((m, n), 4, dev, t)
    xv, wv = value8(x8, xsf, 1), value8(w8, s8, 32)
    for i, act in enumerate(ACTS):
        bb, rr = (b if i != 1 else None), (r if i % 2 == 0 else None)
        y = D.linear_act_q8(x8, xsf, w8, s8, bb, act, rr)
        ref, bound, _, _ = linear_bounds(xv, wv, bb, act, rr, t)
        within(y, ref, bound, f"{act}")
        assert torch.equal(y, D.linear_act_q8(x8, xsf, w8, s8, bb, act, rr))
    wide = torch.full((s8.shape[0], s8.shape[1] + 4), 99, device=dev, dtype=torch.uint8)  # scale rows longer than K / 32
    wide[:, : s8.shape[1]] = s8
    assert torch.equal(D.linear_act_q8(x8, xsf, w8, wide, b), D.linear_act_q8(x8, xsf, w8, s8, b))


def test_linear_act_q8_matches_exact_dequantisation(D, mods, dev):
    """Every e4m3 code against every e4m3 code: one k carries a value, the rest is zero, so the product is exact in fp32."""
    codes = torch.arange(256, dtype=torch.uint8, device=dev)
    codes = codes[(codes & 0x7F) != 0x7F]  # without the NaNs
    m = codes.numel()
    x8, w8 = torch.zeros(m, 128, dtype=torch.uint8, device=dev), torch.zeros(m, 128, dtype=torch.uint8, device=dev)
    x8[:, 77], w8[:, 77] = codes, codes
    xsf = (torch.arange(m, device=dev) % 9 + 123)[:, None].expand(m, 4).to(torch.uint8).contiguous()
    s8 = (torch.arange((m + 31) // 32, device=dev) % 5 + 125)[:, None].expand(-1, 4).to(torch.uint8).contiguous()
    ref = (value8(x8, xsf, 1) @ value8(w8, s8, 32).t()).to(torch.bfloat16)
    assert torch.equal(D.linear_act_q8(x8, xsf, w8, s8), ref)
    for lo, hi in ((0, 1), (3, 11), (100, 116), (50, 90)):
        assert torch.equal(D.linear_act_q8(x8[lo:hi], xsf[lo:hi], w8, s8), ref[lo:hi])


# ------------------------------------------------------------------ together
def ffn64(x, r, nw, w13, w2, limit):
    s, _, y = norm64(x, r, nw, 1e-6)
    inter = w13.shape[0] // 2
    gu = y @ w13.double().t()
    g, u = gu[:, :inter], gu[:, inter:]
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return (act64("silu", g) * u) @ w2.double().t() + s


@pytest.mark.parametrize("m", [1, 5, 70, 300])
def test_block_trains(D, dev, m):
    """norm -> gated projection -> down projection with the residual, forward and all gradients.  Each of the three steps rounds to 8 bits of mantissa;
    relative to the norm of the result the roundings add up like independent errors of u / sqrt(3) each: y, h, out forward (amplified by less than 2 on
    the way), and as many again backward; 8 u bounds the sum with room for two standard deviations."""
    dim, inter, t = 256, 192, torch.bfloat16
    P = {"x": randn((m, dim), 1, dev, t), "r": randn((m, dim), 2, dev, t), "nw": 1 + randn((dim,), 3, dev, torch.float32, 0.2),
         "w13": randn((2 * inter, dim), 4, dev, t, 1 / 16), "w2": randn((dim, inter), 5, dev, t, 1 / 14)}
    for v in P.values():
        v.requires_grad_(True)
    out = D.DenseFFN(P["nw"], P["w13"], P["w2"], limit=3.0)(P["x"], P["r"])
    gy = randn((m, dim), 6, dev, t)
    grads = torch.autograd.grad(out, list(P.values()), gy)
    Q = {n: v.detach().double().requires_grad_(True) for n, v in P.items()}
    ref = ffn64(Q["x"], Q["r"], Q["nw"], Q["w13"], Q["w2"], 3.0)
    rg = torch.autograd.grad(ref, list(Q.values()), gy.double())
    for name, a, b in zip(["out", *P], [out, *grads], [ref, *rg]):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= 8 * u_of(t), (name, rel)


@pytest.mark.parametrize("m", [1, 8, 70, 300])
def test_block_in_fp8(D, mods, dev, m):
    """The FP8 block against the same steps in 64 bits on the same quantised weights: what is left is the rounding of the normed rows and of h to e4m3 (a
    relative error of at most 2^-4 each, 2^-4 / sqrt(3) in the mean), the latter doubled through the product."""
    dim, inter = 512, 256
    sh = mods.synth.make_shared(dim, inter, seed=3, kind="e8m0", std=0.08)
    w13, w2 = mods.w8.W8(sh["w13"].to(dev), sh["s13"].to(dev)), mods.w8.W8(sh["w2"].to(dev), sh["s2"].to(dev))
    nw = 1 + randn((dim,), 4, dev, torch.float32, 0.2)
    x, r = randn((m, dim), 1, dev, torch.bfloat16), randn((m, dim), 2, dev, torch.bfloat16)
    out = D.DenseFFN(nw, w13, w2, limit=10.0)(x, r)
    ref = ffn64(x, r, nw, w13.bf16(), w2.bf16(), 10.0)
    branch, got = ref - (x.double() + r.double()), out.double() - (x.double() + r.double())
    assert ((got - branch).norm() / branch.norm()).item() <= 3 * 2.0 ** -4
    assert mods.cukern.device_error(dev) == 0


def test_other_stream_and_device_argument(D, dev):
    x, w13, w2 = randn((40, 256), 1, dev, torch.bfloat16), randn((256, 256), 2, dev, torch.bfloat16, 0.1), randn((256, 128), 3, dev, torch.bfloat16, 0.1)
    blk = D.DenseFFN(None, w13, w2)
    ref = blk(x, x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    outs = []
    with torch.cuda.stream(st):
        x2 = x * 1  # produced on this stream: the kernels must follow it there
        for _ in range(3):
            outs.append(blk(x2, x2))
    more = blk(x, x)  # at the same time on the default stream
    st.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs) and torch.equal(more, ref)


def test_two_captured_graphs(D, dev):
    """Forward and backward captured into two graphs over static inputs, replayed with new values in turn and at the same time on two streams."""
    dim, inter, m = 256, 128, 37

    def make(seed):
        P = [randn((m, dim), seed, dev, torch.bfloat16), randn((dim,), seed + 1, dev, torch.bfloat16), randn((2 * inter, dim), seed + 2, dev, torch.bfloat16, 0.1),
             randn((dim, inter), seed + 3, dev, torch.bfloat16, 0.1)]
        return [p.requires_grad_(True) for p in P]

    def step(P, gy):
        out = D.DenseFFN(P[1], P[2], P[3], limit=2.0)(P[0], None)
        return [out.detach(), *torch.autograd.grad(out, P, gy)]

    gy = randn((m, dim), 9, dev, torch.bfloat16)
    graphs, outs, params = [], [], []
    side = torch.cuda.Stream()
    for k in range(2):
        P = make(100 * k)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(P, gy)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = step(P, gy)
        graphs.append(g), outs.append(o), params.append(P)
    for trial in range(2):
        refs = []
        for k in range(2):
            new = make(1000 * trial + 100 * k + 7)
            with torch.no_grad():
                for a, b in zip(params[k], new):
                    a.copy_(b)
            refs.append([t.clone() for t in step(new, gy)])
        torch.cuda.synchronize()
        s2 = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in zip(outs[k], refs[k]):
                assert torch.equal(a, b)


def test_no_device_error_left(mods, dev):
    assert mods.cukern.device_error(dev) == 0


def test_no_second_derivatives(D, dev):
    """Gradients with create_graph are the same values and refuse to be differentiated again."""
    x, w = randn((8, 64), 1, dev, torch.bfloat16).requires_grad_(True), randn((16, 64), 2, dev, torch.bfloat16).requires_grad_(True)
    n, w13 = randn((64,), 3, dev, torch.bfloat16).requires_grad_(True), randn((32, 64), 4, dev, torch.bfloat16).requires_grad_(True)
    xs = randn((8, 80), 5, dev, torch.bfloat16)[:, 3:67].requires_grad_(True)  # rows that take the other way through the host code
    for f, leaves in ((lambda: D.linear_act(x, w, None, "gelu"), (x, w)), (lambda: D.gated_linear(x, w13), (x, w13)), (lambda: D.add_rms_norm(x, None, n)[0], (x, n)),
                      (lambda: D.linear_act(xs, w, None, "gelu"), (xs, w)), (lambda: D.gated_linear(xs, w13), (xs, w13)), (lambda: D.add_rms_norm(xs, None, n)[0], (xs, n))):
        y = f()
        plain = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        graph = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, graph))
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            torch.autograd.grad(graph[0].float().sum(), leaves[1])


@pytest.mark.parametrize("n", [64, 50])  # 50: rows that the kernels cannot fetch, another way through the host code
def test_gradients_of_some_inputs(D, dev, n):
    """Whatever subset of the inputs wants a gradient, each gets the one of the full call."""
    t, k, m = torch.bfloat16, 72, 19
    vals = {"x": randn((m, k), 1, dev, t), "w": randn((n, k), 2, dev, t, 0.1), "bias": randn((n,), 3, dev, t), "residual": randn((m, n), 4, dev, t)}
    gy = randn((m, n), 5, dev, t)
    full = {a: v.clone().requires_grad_(True) for a, v in vals.items()}
    ref = dict(zip(full, torch.autograd.grad(D.linear_act(act="gelu", **full), list(full.values()), gy)))
    for names in (("x",), ("w",), ("bias",), ("residual",), ("x", "residual"), ("w", "bias"), ("bias", "residual")):
        for drop in (None, "bias", "residual"):
            if drop in names:
                continue
            args = {a: v.clone().requires_grad_(a in names) for a, v in vals.items() if a != drop}
            got = torch.autograd.grad(D.linear_act(act="gelu", **args), [args[a] for a in names], gy)
            for a, g in zip(names, got):
                if drop != "bias":  # without the bias the slopes are others
                    assert torch.equal(g, ref[a]), (names, drop, a)
                assert g.shape == vals[a].shape and g.isfinite().all()
    w13 = randn((2 * n, k), 6, dev, t, 0.1)
    xg, wg = vals["x"].clone().requires_grad_(True), w13.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(D.gated_linear(xg, wg, limit=2.0), (xg, wg), gy)
    assert torch.equal(torch.autograd.grad(D.gated_linear(xg, w13, limit=2.0), xg, gy)[0], dx)
    assert torch.equal(torch.autograd.grad(D.gated_linear(vals["x"], wg, limit=2.0), wg, gy)[0], dw)
    nw, r = randn((k,), 7, dev, t), randn((m, k), 8, dev, t)
    gk = randn((m, k), 9, dev, t)
    P = [v.clone().requires_grad_(True) for v in (vals["x"], r, nw)]
    ref3 = torch.autograd.grad(D.add_rms_norm(*P)[0], P, gk)
    for mask in range(1, 8):
        Q = [v.clone().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((vals["x"], r, nw))]
        want = [i for i in range(3) if mask >> i & 1]
        got = torch.autograd.grad(D.add_rms_norm(*Q)[0], [Q[i] for i in want], gk)
        assert all(torch.equal(g, ref3[i]) for g, i in zip(got, want))
    q = nw.clone().requires_grad_(True)
    full2 = torch.autograd.grad(D.add_rms_norm(vals["x"], None, q)[0], q, gk)[0]
    x2 = vals["x"].clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(D.add_rms_norm(x2, None, q)[0], (x2, q), gk)[1], full2)
