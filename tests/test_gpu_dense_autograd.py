"""The dense operators under the tools of torch's autograd: saved-tensor hooks, derivatives of derivatives, forward-mode derivatives."""
import importlib

import pytest
import torch

from test_dense_autograd_host import check_free, check_guard

pytestmark = pytest.mark.gpu
T = torch.bfloat16


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


def randn(shape, seed, dev, dtype=T, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def operands(dev, kind, k=72):
    """x [20, k], w [48, k], residual [20, 48], bias [48] as leaves: dense, aligned slices of wider rows, or slices at an odd offset."""
    at = {"dense": None, "slices": 8, "odd": 3}[kind]

    def rows(r, c, seed, scale=1.0):
        if at is None:
            return randn((r, c), seed, dev, T, scale).requires_grad_(True)
        return randn((r, c + 48), seed, dev, T, scale)[:, at:at + c].requires_grad_(True)

    return {"x": rows(20, k, 1), "w": rows(48, k, 2, 0.2), "residual": rows(20, 48, 3), "bias": randn((48,), 4, dev).requires_grad_(True)}


def calls(D, dev, kind):
    """(name, leaves, function) of each differentiable operator on such operands."""
    P = operands(dev, kind)
    Q = operands(dev, kind)
    n = (1 + randn((72,), 5, dev, torch.float32, 0.2)).requires_grad_(True)
    R = operands(dev, kind)
    r = randn((20, 72), 6, dev).requires_grad_(True)
    return [("linear", list(P.values()), lambda: D.linear_act(P["x"], P["w"], P["bias"], "gelu", P["residual"])),
            ("product", [P["x"], P["w"]], lambda: D.linear_act(P["x"], P["w"])),
            ("gated", [Q["x"], Q["w"]], lambda: D.gated_linear(Q["x"], Q["w"], limit=2.0)),
            ("norm", [R["x"], r, n], lambda: D.add_rms_norm(R["x"], r, n)[0])]


def wider(offset):
    def unpack(t):
        buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype, device=t.device)
        return buf[..., offset:offset + t.shape[-1]].copy_(t)
    return unpack


@pytest.mark.parametrize("kind", ["dense", "slices", "odd"])
@pytest.mark.parametrize("hook", ["save_on_cpu", "clone", "wider", "wider_odd"])
def test_saved_tensor_hooks(D, dev, kind, hook):
    """Whatever strides and addresses a hook hands back, the gradients are those of the call without it.  Operands off 16 bytes go through the same products (as
    copies); the norm adds them up in another order: within a rounding of 2^-8 and the fp32 sums."""
    for name, leaves, f in calls(D, dev, kind):
        y = f()
        gy = randn(y.shape, 9, dev)
        ref = torch.autograd.grad(y, leaves, gy)
        if hook == "save_on_cpu":
            ctx = torch.autograd.graph.save_on_cpu()
        else:
            ctx = torch.autograd.graph.saved_tensors_hooks(lambda t: t, {"clone": torch.clone, "wider": wider(8), "wider_odd": wider(3)}[hook])
        with ctx:
            y2 = f()
        got = torch.autograd.grad(y2, leaves, gy)
        assert torch.equal(y, y2)
        for a, b in zip(got, ref):
            if name == "norm" and (kind == "odd" or hook == "wider_odd"):
                assert ((a - b).double().abs() <= 2.0 ** -8 * b.double().abs() + 2.0 ** -16 * b.double().abs().max()).all(), (name, hook)
            else:
                assert torch.equal(a, b), (name, hook)


@pytest.mark.parametrize("kind", ["dense", "slices"])
@pytest.mark.parametrize("unpack", [lambda t: t[..., :-8], lambda t: t.double(), lambda t: t.cpu()])
def test_other_tensors_from_hooks_are_refused(D, dev, kind, unpack):
    for name, leaves, f in calls(D, dev, kind):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = f()
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.parametrize("kind", ["dense", "odd"])
def test_forward_mode_is_refused(D, dev, kind):
    """Whichever input carries the tangent, with and without a gradient wanted or recorded."""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        for grad in (False, True):
            for recorded in (False, True):
                for which in ("x", "w", "bias", "residual"):
                    P = {a: t.detach().requires_grad_(grad) for a, t in operands(dev, kind).items()}
                    n = randn((72,), 5, dev).requires_grad_(grad)
                    P[which] = fw.make_dual(P[which], torch.ones_like(P[which]))
                    with torch.set_grad_enabled(recorded):
                        fs = [lambda: D.linear_act(P["x"], P["w"], P["bias"], "gelu", P["residual"])]
                        if which in ("x", "w"):
                            fs.append(lambda: D.gated_linear(P["x"], P["w"]))
                        if which == "x":
                            fs += [lambda: D.add_rms_norm(P["x"]), lambda: D.add_rms_norm(P["x"], None, n), lambda: D.add_rms_norm(P["x"].detach() * 0, P["x"]),
                                   lambda: D.add_rms_norm_quant(torch.cat([P["x"]] * 4, 1))]
                        for f in fs:
                            with pytest.raises(NotImplementedError, match="forward-mode"):
                                f()
    x, w = randn((4, 64), 1, dev), randn((8, 64), 2, dev)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda a: D.linear_act(a, w), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("kind", ["dense", "slices", "odd"])  # dense: the extension's functions; slices and odd offsets: dense.py's
def test_second_derivatives_raise_on_the_way_to_any_input(D, dev, kind):
    """Constant and differentiable incoming gradients, whichever leaf is asked for; and a penalty on a gradient does not train without its own gradient."""
    check_guard([(name, tuple(leaves), f) for name, leaves, f in calls(D, dev, kind) if name != "product"])
    for name, leaves, f in calls(D, dev, kind):
        y = f()
        gy = randn(y.shape, 9, dev)
        plain = torch.autograd.grad(y, leaves, gy, retain_graph=True)
        graph = torch.autograd.grad(y, leaves, gy, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, graph))


@pytest.mark.parametrize("odd", [False, True])
def test_gradients_that_depend_on_nothing_are_free(D, dev, odd):
    def linear(x, w, b, act, r):
        if odd:  # rows that are no view of 16-byte ones: dense.py's functions
            x = torch.cat([x, x], 1)[:, 3:67]
        return D.linear_act(x, w, b, act, r)
    check_free(linear, T, dev)


@pytest.mark.parametrize("kind", ["dense", "slices", "odd"])
def test_checkpointed_calls(D, dev, kind):
    """torch.utils.checkpoint hands the tensors of a second forward pass to the backward pass: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    for name, leaves, f in calls(D, dev, kind):
        y = f()
        gy = randn(y.shape, 9, dev)
        ref = torch.autograd.grad(y, leaves, gy)
        y2 = checkpoint(f, use_reentrant=False)
        got = torch.autograd.grad(y2, leaves, gy)
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(got, ref)), name
