"""The FP8 block step by step: every step's input is the codes of the step before, so that each is held to its own roundings."""
import importlib

import pytest
import torch

from test_gpu_dense import ACT_EVAL, SLOPE, SUM_REL, act64, check_codes, gamma, linear_bounds, norm64, randn, u_of, value8, within

pytestmark = pytest.mark.gpu
T = torch.bfloat16


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


def block(D, mods, dev, dim, inter, limit):
    sh = mods.synth.make_shared(dim, inter, seed=3, kind="e8m0", std=0.08)
    w13, w2 = mods.w8.W8(sh["w13"].to(dev), sh["s13"].to(dev)), mods.w8.W8(sh["w2"].to(dev), sh["s2"].to(dev))
    nw = 1 + randn((dim,), 4, dev, torch.float32, 0.2)
    return D.DenseFFN(nw, w13, w2, limit=limit), nw, w13, w2


@pytest.mark.parametrize("limit", [10.0, 0.4, 0.0])
@pytest.mark.parametrize("m,dim,inter", [(1, 512, 256), (8, 512, 256), (17, 384, 640), (64, 512, 256), (65, 512, 256), (300, 512, 256), (1500, 1024, 1152)])
def test_steps(D, mods, dev, monkeypatch, m, dim, inter, limit):
    ffn, nw, w13, w2 = block(D, mods, dev, dim, inter, limit)
    x, r = randn((m, dim), 1, dev, T), randn((m, dim), 2, dev, T)
    seen = {}
    gate_up, down = mods.cukern.mx_grouped, D.linear_act_q8

    def see_gate_up(*a, **k):
        seen["h"] = gate_up(*a, **k)
        return seen["h"]

    def see_down(*a, **k):
        seen["down"] = (a, k)
        return down(*a, **k)

    monkeypatch.setattr(mods.cukern, "mx_grouped", see_gate_up)
    monkeypatch.setattr(D, "linear_act_q8", see_down)
    out = ffn(x, r)
    # 1. norm: the operator's own test holds it; the block must use its codes and its sum
    q8, sf, s = D.add_rms_norm_quant(x, r, nw, 1e-6)
    check_codes(q8, sf, norm64(x, r, nw, 1e-6)[2], SUM_REL)
    # 2. gate and up on those codes, clamped, silu, product, a rounding to bf16, then to e4m3 with one scale per 32
    xv, wv = value8(q8, sf, 1), value8(mods.w8.unpermute_k(w13.w8), w13.s8, 32)
    gu, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    e = gamma(dim) * mag
    g, u, eg, eu = gu[:, :inter], gu[:, inter:], e[:, :inter], e[:, inter:]
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    a = act64("silu", g)
    h = a * u
    eh = (SLOPE * eg + ACT_EVAL * g.abs()) * (u.abs() + eu) + a.abs() * eu + 2.0 ** -22 * h.abs()
    eh = eh + u_of(T) * (h.abs() + eh) + 2.0 ** -126  # the rounding to bf16
    h8, hsf = seen["h"]
    v8, es = h8.view(torch.float8_e4m3fn).double(), hsf.double() - 127
    amax, eamax = h.abs().view(m, -1, 32).amax(-1), eh.view(m, -1, 32).amax(-1)
    fits = lambda v: torch.ceil(torch.log2(v.clamp_min(float(torch.tensor(1e-4))) / 448) - 1e-12)  # noqa: E731
    assert ((es >= fits(amax - eamax)) & (es <= fits(amax + eamax))).all()
    scale = torch.exp2(es).repeat_interleave(32, 1)
    v, ev = h / scale, eh / scale
    step = torch.exp2(torch.floor(torch.log2((v.abs() + ev).clamp(2.0 ** -6, 448))) - 3)
    assert ((v8 - v.clamp(-448, 448)).abs() <= step / 2 + ev).all()
    # 3. the down projection on those codes, with the sum added
    ref, bound, _, _ = linear_bounds(value8(h8, hsf, 1), value8(mods.w8.unpermute_k(w2.w8), w2.s8, 32), None, None, s, T)
    within(out, ref, bound, "block")
    (a8, asf, *_), kw = seen["down"]
    assert a8.data_ptr() == h8.data_ptr() and asf.data_ptr() == hsf.data_ptr() and torch.equal(kw["residual"], s)
    assert torch.equal(out, ffn(x, r)) and mods.cukern.device_error(dev) == 0


def test_two_captured_graphs_of_the_block(D, mods, dev):
    """Two graphs of FP8 blocks replayed at the same time on two streams, beside an eager call: the same bits as alone."""
    ffn, *_ = block(D, mods, dev, 512, 256, 10.0)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, ins, outs = [], [], []
    for m in (8, 300):
        x = randn((m, 512), m, dev, T)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ffn(x, x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = ffn(x, x)
        graphs.append(g), ins.append(x), outs.append(o)
    for trial in range(3):
        refs = []
        for x in ins:
            x.copy_(randn(x.shape, 100 + trial, dev, T))
            refs.append(ffn(x, x))
        y = randn((70, 512), 200 + trial, dev, T)
        ref_y = ffn(y, y)
        torch.cuda.synchronize()
        for _ in range(4):
            with torch.cuda.stream(side):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
            got = ffn(y, y)
        torch.cuda.synchronize()
        assert torch.equal(got, ref_y) and all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_limits_that_are_refused(D, mods, dev):
    """As in 16 bits."""
    for limit in (-1.0, float("nan")):
        with pytest.raises(AssertionError, match="limit"):
            block(D, mods, dev, 512, 256, limit)
