"""CPU: what the backward passes of the dense operators hand to the kernels.  The calls into the library are recorded, not made: a read through an address or
a stride that does not belong to the tensor at hand shows here without a GPU."""
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


class Recorder:
    def __init__(self, D, monkeypatch):
        self.calls = []
        monkeypatch.setattr(D, "_call", lambda name, index, *args: self.calls.append((name, args)))
        monkeypatch.setattr(D, "_size", lambda name, index, *args: 0)

    def of(self, name):
        return [a for n, a in self.calls if n == name]


class Hooks(torch.autograd.graph.saved_tensors_hooks):
    """Hands back what `unpack` makes of each saved tensor and keeps it."""

    def __init__(self, unpack):
        self.back = []

        def un(t):
            t = unpack(t)
            self.back.append(t)
            return t

        super().__init__(lambda t: t, un)


def dense_copy(t):
    return torch.empty(t.shape, dtype=t.dtype).copy_(t)  # as save_on_cpu does: whatever the strides were, contiguous now


def in_wider_rows(t):
    buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype)
    out = buf[..., 8:8 + t.shape[-1]]
    return out.copy_(t)


def backward(f, hooks):
    with hooks:
        y = f()
    out = y[0] if isinstance(y, tuple) else y
    torch.autograd.backward(out, torch.ones_like(out))


def holds(base, ld, rows, cols, mn, tensors):
    """Whether the operand [rows, cols] (element (i, k) at base[i * ld + k], or base[k * ld + i]) lies within one of the tensors' memory, read at its strides."""
    outer, inner = (cols, rows) if mn else (rows, cols)
    for t in tensors:
        r = t.reshape(-1, t.shape[-1]) if t.is_contiguous() else t
        if t.data_ptr() == base and r.dim() == 2 and r.shape[0] == outer and inner <= r.shape[1] and (outer == 1 or r.stride(0) == ld) and r.stride(1) == 1:
            return True
    return False


@pytest.mark.parametrize("unpack", [dense_copy, in_wider_rows])
@pytest.mark.parametrize("which", ["linear", "gated"])
def test_products_read_the_tensors_that_hooks_return(D, monkeypatch, unpack, which):
    rec, made = Recorder(D, monkeypatch), []
    aligned = D._aligned
    monkeypatch.setattr(D, "_aligned", lambda x, w, K: made.append(aligned(x, w, K)) or made[-1])
    big, wide = torch.zeros(20, 304, dtype=torch.bfloat16), torch.zeros(48, 320, dtype=torch.bfloat16)
    x, w = big[:, 8:264].requires_grad_(True), wide[:, :256].requires_grad_(True)
    hooks = Hooks(unpack)
    f = (lambda: D._LinearAct.apply(x, w, None, 3, None)) if which == "linear" else (lambda: D._GatedLinear.apply(x, w, 2, 0.0))
    backward(f, hooks)
    products = rec.of("b200_dense_product")
    assert len(products) == 2
    live = hooks.back + [m[0] for m in made]
    for a, a_ld, a_mn, b, b_ld, b_mn, _, M, N, K, *_ in products:
        assert holds(b, b_ld, N, K, b_mn, live), (M, N, K, b_ld)
    z = rec.of("b200_linear_act_bwd" if which == "linear" else "b200_gated_linear_bwd")[0]
    assert z[3] == 48 and (unpack is in_wider_rows or holds(z[2], z[3], 20, 48, 0, live))  # wider rows are copied to dense ones first


@pytest.mark.parametrize("unpack", [dense_copy, in_wider_rows])
def test_norm_reads_the_tensors_that_hooks_return(D, monkeypatch, unpack):
    rec = Recorder(D, monkeypatch)
    big = torch.zeros(20, 304, dtype=torch.bfloat16)
    x, r = big[:, 8:72].requires_grad_(True), big[:, 80:144].requires_grad_(True)
    w = torch.zeros(64).requires_grad_(True)
    hooks = Hooks(unpack)
    backward(lambda: D._AddRmsNorm.apply(x, r, w, 1e-6), hooks)
    a = rec.of("b200_add_rms_norm_bwd")[0]
    assert holds(a[0], a[1], 20, 64, 0, hooks.back) and holds(a[2], a[3], 20, 64, 0, hooks.back)
    assert a[4] in [t.data_ptr() for t in hooks.back if t.dim() == 1]


@pytest.mark.parametrize("unpack", [lambda t: t[..., :-8], lambda t: t.to(torch.float64), lambda t: t.to("meta")])
def test_another_tensor_from_a_hook_is_refused(D, monkeypatch, unpack):
    Recorder(D, monkeypatch)
    x, w = torch.zeros(20, 256, dtype=torch.bfloat16, requires_grad=True), torch.zeros(48, 256, dtype=torch.bfloat16, requires_grad=True)
    n = torch.zeros(256, dtype=torch.bfloat16, requires_grad=True)
    for f in (lambda: D._LinearAct.apply(x, w, None, 3, None), lambda: D._GatedLinear.apply(x, w, 2, 0.0), lambda: D._AddRmsNorm.apply(x, x, n, 1e-6)):
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            backward(f, Hooks(unpack))


def test_forward_mode_is_refused(D, monkeypatch):
    """A result without a tangent would count as one whose derivative is zero."""
    import torch.autograd.forward_ad as fw
    monkeypatch.setattr(D.L, "require_cuda", lambda *t: torch.device("cpu"))
    rec = Recorder(D, monkeypatch)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    with fw.dual_level():
        dual = lambda *s: fw.make_dual(bf(*s), bf(*s))  # noqa: E731
        for call in (lambda: D.linear_act(dual(2, 64), bf(8, 64)), lambda: D.linear_act(bf(2, 64), dual(8, 64)), lambda: D.linear_act(bf(2, 64), bf(8, 64), dual(8)),
                     lambda: D.linear_act(bf(2, 64), bf(8, 64), residual=dual(2, 8)), lambda: D.gated_linear(dual(2, 64), bf(8, 64)), lambda: D.gated_linear(bf(2, 64), dual(8, 64)),
                     lambda: D.add_rms_norm(dual(2, 64)), lambda: D.add_rms_norm(bf(2, 64), dual(2, 64)), lambda: D.add_rms_norm(bf(2, 64), None, dual(64)),
                     lambda: D.add_rms_norm_quant(dual(2, 64)), lambda: D.linear_act_q8(u8(2, 128), u8(2, 4), u8(8, 128), u8(1, 4), bias=dual(8)),
                     lambda: D.linear_act_q8(u8(2, 128), u8(2, 4), u8(8, 128), u8(1, 4), residual=dual(2, 8))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not rec.calls
        D.linear_act(bf(2, 64), bf(8, 64))  # without tangents a level changes nothing
        assert len(rec.calls) == 1


TWICE = "differentiate twice"


def python_calls(D):
    """Each operator's Python route on leaves; the values are whatever the memory holds, the graph is what is looked at."""
    leaf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, requires_grad=True)  # noqa: E731
    x, w, b, r = leaf(4, 64), leaf(16, 64), leaf(16), leaf(4, 16)
    n, s = leaf(64), leaf(4, 64)
    w13 = leaf(32, 64)
    return [("linear", (x, w, b, r), lambda: D._LinearAct.apply(x, w, b, 3, r)), ("gated", (x, w13), lambda: D._GatedLinear.apply(x, w13, 2, 0.0)), ("norm", (x, s, n), lambda: D._AddRmsNorm.apply(x, s, n, 1e-6)[0])]


def check_guard(calls):
    for name, leaves, f in calls:
        for gy_wants in (False, True):
            y = f()
            gy = torch.ones_like(y).requires_grad_(gy_wants)
            gs = torch.autograd.grad(y, leaves, gy, create_graph=True)
            for i, g in enumerate(gs[:2]):  # x and w (or the norm's residual) depend on all the others
                loss = y.float().sum() + g.float().square().sum()
                for leaf in leaves[:2] + ((gy,) if gy_wants else ()):
                    with pytest.raises(RuntimeError, match=TWICE):
                        torch.autograd.grad(loss, leaf, retain_graph=True)
                with pytest.raises(RuntimeError, match=TWICE):
                    loss.backward(retain_graph=True)
            plain = torch.autograd.grad(y, leaves, gy.detach(), retain_graph=True)
            assert not any(g.requires_grad for g in plain)


def test_second_derivatives_raise_on_the_way_to_any_input(D, monkeypatch):
    Recorder(D, monkeypatch)
    check_guard(python_calls(D))


def check_free(linear, dtype=torch.bfloat16, device="cpu"):
    """Gradients that depend on nothing that wants one stay as they are; the residual's is the incoming one and can be differentiated again; without an activation
    the gradient of x depends on w alone and that of w on x alone."""
    t = lambda *s: torch.ones(*s, dtype=dtype, device=device)  # noqa: E731
    for act in (None, "relu"):
        x = t(4, 64).requires_grad_(True)
        y = linear(x, t(16, 64), t(16), act, t(4, 16))
        assert not torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)[0].requires_grad
        b = t(16).requires_grad_(True)
        y = linear(t(4, 64), t(16, 64), b, act, None)
        assert not torch.autograd.grad(y, b, torch.ones_like(y), create_graph=True)[0].requires_grad
    r, x = t(4, 16).requires_grad_(True), t(4, 64).requires_grad_(True)
    y = linear(x, t(16, 64), None, "silu", r)
    v = t(4, 16).requires_grad_(True)
    dr = torch.autograd.grad(y, r, v, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad((dr * dr).sum(), v)[0], 2 * v.detach())
    for act in (None, "relu"):
        x, w, b = t(4, 64).requires_grad_(True), t(16, 64).requires_grad_(True), t(16).requires_grad_(True)
        y = linear(x, w, b, act, None)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y), create_graph=True)
        assert dx.requires_grad and dw.requires_grad and not db.requires_grad
        for g, free, bound in ((dx, x, w), (dw, w, x)):
            assert torch.autograd.grad(g.float().sum(), (free, b), allow_unused=True, retain_graph=True) == (None, None)
            torch.autograd.grad(y.float().sum() + g.float().sum(), (free, b), retain_graph=True)
            with pytest.raises(RuntimeError, match=TWICE):
                torch.autograd.grad(y.float().sum() + g.float().sum(), bound, retain_graph=True)


def test_gradients_that_depend_on_nothing_are_free(D, monkeypatch):
    Recorder(D, monkeypatch)
    check_free(lambda x, w, b, act, r: D._LinearAct.apply(x, w, b, D._act_code(act), r))
