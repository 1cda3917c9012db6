"""CPU: argument checks of the dense operators, in Python and at the C boundary (every refusal comes before anything is launched)."""
import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


def test_cpu_tensors_are_refused(D):
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    for call in (lambda: D.add_rms_norm(x), lambda: D.add_rms_norm_quant(x), lambda: D.linear_act(x, w), lambda: D.gated_linear(x, w),
                 lambda: D.linear_act_q8(*(torch.zeros(2, 128, dtype=torch.uint8),) * 4)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_python_refusals(D, monkeypatch):
    monkeypatch.setattr(D.L, "require_cuda", lambda *t: torch.device("cpu"))  # the checks behind the device check
    bf = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    bad = [
        lambda: D.add_rms_norm(bf(2, 64, t=torch.float64)),
        lambda: D.add_rms_norm(bf(2, 20000)),
        lambda: D.add_rms_norm(bf(2, 64), bf(1, 64)),
        lambda: D.add_rms_norm(bf(2, 64), bf(2, 64, t=torch.float16)),
        lambda: D.add_rms_norm(bf(2, 64), None, bf(64, t=torch.float16)),
        lambda: D.add_rms_norm(bf(2, 64), None, bf(63)),
        lambda: D.add_rms_norm(bf(2, 64), eps=-1.0),
        lambda: D.add_rms_norm(bf(2, 64), eps=float("nan")),
        lambda: D.add_rms_norm_quant(bf(2, 48)),
        lambda: D.add_rms_norm_quant(bf(2, 64).requires_grad_(True)),
        lambda: D.linear_act(bf(2, 64), bf(8, 64, t=torch.float16)),
        lambda: D.linear_act(bf(2, 64, t=torch.float32), bf(8, 64, t=torch.float32)),
        lambda: D.linear_act(bf(2, 64), bf(8, 32)),
        lambda: D.linear_act(bf(2, 64), bf(8, 64), bias=bf(7)),
        lambda: D.linear_act(bf(2, 64), bf(8, 64), bias=bf(8, t=torch.float32)),
        lambda: D.linear_act(bf(2, 64), bf(8, 64), act="tanh"),
        lambda: D.linear_act(bf(2, 64), bf(8, 64), residual=bf(1, 8)),
        lambda: D.gated_linear(bf(2, 64), bf(7, 64)),
        lambda: D.gated_linear(bf(2, 64), bf(8, 64), limit=-1.0),
        lambda: D.gated_linear(bf(2, 64), bf(8, 64), act="swish"),
        lambda: D.linear_act_q8(u8(2, 64), u8(2, 2), u8(8, 64), u8(1, 2)),
        lambda: D.linear_act_q8(u8(2, 128), u8(2, 3), u8(8, 128), u8(1, 4)),
        lambda: D.linear_act_q8(u8(2, 128), u8(2, 4), u8(40, 128), u8(1, 4)),
        lambda: D.linear_act_q8(bf(2, 128), u8(2, 4), u8(8, 128), u8(1, 4)),
        lambda: D.linear_act_q8(u8(2, 128), u8(2, 4), u8(8, 128), u8(1, 4), residual=bf(2, 9)),
        lambda: D.DenseFFN(None, bf(8, 64), bf(64, 5)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was accepted")


def test_c_boundary_refusals(mods):
    """Return codes of calls with addresses that are never followed: the checks come first."""
    lib = mods.lib.lib()
    p = ctypes.c_void_p(1 << 20)
    odd = ctypes.c_void_p((1 << 20) + 2)
    n = ctypes.c_void_p(0)
    BAD_ARG, BAD_SHAPE, BAD_ALIGN, WORKSPACE, UNSUPPORTED, TOO_LARGE = -1, -2, -3, -4, -5, -6
    norm = lib.b200_add_rms_norm
    assert norm(p, 64, n, 0, n, 0, 0, -1, 64, 1e-6, p, n, n, n, n) == BAD_ARG
    assert norm(p, 64, n, 0, n, 0, 0, 2, 64, -1.0, p, n, n, n, n) == BAD_ARG
    assert norm(p, 64, n, 0, n, 0, 0, 2, 64, float("nan"), p, n, n, n, n) == BAD_ARG
    assert norm(p, 64, n, 0, n, 0, 3, 2, 64, 1e-6, p, n, n, n, n) == UNSUPPORTED
    assert norm(p, 20000, n, 0, n, 0, 0, 2, 20000, 1e-6, p, n, n, n, n) == TOO_LARGE
    assert norm(p, 63, n, 0, n, 0, 0, 2, 64, 1e-6, p, n, n, n, n) == BAD_SHAPE
    assert norm(p, 64, n, 0, n, 0, 0, 2, 64, 1e-6, n, n, n, n, n) == BAD_ARG
    assert norm(p, 64, n, 0, n, 0, 0, 2, 64, 1e-6, p, n, p, n, n) == BAD_ARG
    assert norm(p, 48, n, 0, n, 0, 0, 2, 48, 1e-6, p, n, p, p, n) == BAD_SHAPE
    assert norm(n, 64, n, 0, n, 0, 0, 0, 64, 1e-6, p, n, n, n, n) == 0
    bwd = lib.b200_add_rms_norm_bwd
    assert bwd(p, 64, n, 0, n, 0, 0, 2, 64, 1e-6, n, n, p, n, n, 0, n) == BAD_ARG
    assert bwd(p, 64, n, 0, n, 0, 0, 2, 64, 1e-6, p, n, p, p, n, 0, n) == BAD_ARG  # a weight gradient without a weight
    lin = lib.b200_linear_act
    assert lin(p, 64, p, 64, 2, 2, 8, 64, n, 0, n, 0, p, 8, n, 0, n) == UNSUPPORTED
    assert lin(p, 64, p, 64, 0, 2, 8, 64, n, 9, n, 0, p, 8, n, 0, n) == UNSUPPORTED
    assert lin(p, 64, p, 64, 0, 2, 0, 64, n, 0, n, 0, p, 8, n, 0, n) == BAD_SHAPE
    assert lin(p, 64, p, 64, 0, 2, 8, 0, n, 0, n, 0, p, 8, n, 0, n) == BAD_SHAPE
    assert lin(p, 64, p, 64, 0, 2, 8, 64, n, 0, n, 0, p, 7, n, 0, n) == BAD_SHAPE
    assert lin(p, 64, p, 64, 0, 2, 8, 64, n, 0, p, 7, p, 8, n, 0, n) == BAD_SHAPE
    assert lin(p, 60, p, 64, 0, 2, 8, 60, n, 0, n, 0, p, 8, n, 0, n) == BAD_ALIGN
    assert lin(odd, 64, p, 64, 0, 2, 8, 64, n, 0, n, 0, p, 8, n, 0, n) == BAD_ALIGN
    assert lin(p, 56, p, 64, 0, 2, 8, 64, n, 0, n, 0, p, 8, n, 0, n) == BAD_SHAPE
    assert lin(p, 64, n, 64, 0, 2, 8, 64, n, 0, n, 0, p, 8, n, 0, n) == BAD_ARG
    assert lin(n, 64, n, 64, 0, 0, 8, 64, n, 0, n, 0, n, 8, n, 0, n) == 0
    lb = lib.b200_linear_act_bwd
    assert lb(p, 8, n, 0, 2, 0, 2, 8, p, 8, n, n, 0, n) == BAD_ARG  # silu without its pre-activation
    assert lb(p, 8, p, 8, 2, 0, 2, 8, p, 8, p, n, 0, n) == WORKSPACE
    assert lb(p, 8, p, 8, 2, 0, 2, 8, n, 0, n, n, 0, n) == BAD_ARG
    gl = lib.b200_gated_linear
    assert gl(p, 64, p, 64, 0, 2, 0, 64, 2, 0.0, p, 8, n, 0, n) == BAD_SHAPE
    assert gl(p, 64, p, 64, 0, 2, 8, 64, 2, -1.0, p, 8, n, 0, n) == BAD_SHAPE
    assert gl(p, 64, p, 64, 0, 2, 8, 64, 2, 0.0, p, 8, p, 15, n) == BAD_SHAPE
    gb = lib.b200_gated_linear_bwd
    assert gb(p, 8, p, 15, 2, 0.0, 0, 2, 8, p, 16, n) == BAD_SHAPE
    assert gb(p, 8, n, 16, 2, 0.0, 0, 2, 8, p, 16, n) == BAD_ARG
    dp = lib.b200_dense_product
    assert dp(p, 64, 1, p, 64, 0, 0, 64, 64, 8, p, 64, n) == UNSUPPORTED
    assert dp(p, 60, 0, p, 64, 1, 0, 8, 64, 60, p, 64, n) == BAD_ALIGN
    assert dp(p, 64, 0, p, 56, 1, 0, 8, 64, 64, p, 64, n) == BAD_SHAPE
    assert lib.b200_align_rows(p, 9, odd, 4, n, 0, n, 0, 9, 16, n) == BAD_ALIGN
    assert lib.b200_align_rows(p, 9, p, 4, n, 0, n, 0, 9, 12, n) == BAD_ALIGN
    assert lib.b200_align_rows(p, 9, p, 4, n, 0, n, 0, 9, 8, n) == BAD_SHAPE
    assert lib.b200_align_rows(p, 9, p, 4, n, 9, n, 2, 9, 16, n) == BAD_ARG
    assert lib.b200_align_rows(n, 9, n, 0, n, 0, n, 0, 9, 16, n) == 0
    q8 = lib.b200_linear_act_q8
    assert q8(p, p, p, p, 2, 2, 8, 64, n, 0, n, 0, p, 8, p, 1 << 30, n) == BAD_SHAPE
    assert q8(p, p, p, p, 3, 2, 8, 128, n, 0, n, 0, p, 8, p, 1 << 30, n) == BAD_SHAPE
    assert q8(odd, p, p, p, 4, 2, 8, 128, n, 0, n, 0, p, 8, p, 1 << 30, n) == BAD_ALIGN
    assert lib.b200_linear_act_q8_workspace_bytes(2, 8, 128) == 0  # decode-sized calls need none
    need = lib.b200_linear_act_q8_workspace_bytes(32, 8, 128)
    assert need > 0 and q8(p, p, p, p, 4, 32, 8, 128, n, 0, n, 0, p, 8, p, need - 1, n) == WORKSPACE
    assert q8(p, p, p, p, 4, 32, 8, 128, n, 0, n, 0, p, 8, n, need, n) == WORKSPACE
    assert b"shape" in lib.b200_error_string(BAD_SHAPE) or lib.b200_error_string(BAD_SHAPE)
