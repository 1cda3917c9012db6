"""CPU: sizes at the ends of what the dense operators count in 32 bits."""
import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


@pytest.mark.parametrize("count", [(1 << 30) + 1, (1 << 31) + 5, (1 << 32) + 5])
def test_counts_past_the_limit_are_refused(D, monkeypatch, count):
    """2^32 + 5 rows are not five rows."""
    monkeypatch.setattr(D.L, "require_cuda", lambda *t: torch.device("cpu"))
    made = []
    monkeypatch.setattr(D, "_call", lambda name, index, *args: made.append(name))
    row = lambda w, t=torch.bfloat16: torch.zeros(1, w, dtype=t).expand(count, w)  # noqa: E731  one row in memory
    u8 = torch.uint8
    z = lambda *s: torch.zeros(*s, dtype=u8)  # noqa: E731
    for call in (lambda: D.linear_act(row(1), torch.zeros(1, 1, dtype=torch.bfloat16)), lambda: D.linear_act(torch.zeros(1, 1, dtype=torch.bfloat16), row(1)),
                 lambda: D.linear_act(row(1).t(), row(1).t()), lambda: D.gated_linear(row(1), torch.zeros(2, 1, dtype=torch.bfloat16)),
                 lambda: D.gated_linear(torch.zeros(1, 1, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.bfloat16).expand(count // 2 * 2 + 2, 1)),
                 lambda: D.gated_linear(row(1).t(), torch.zeros(1, 1, dtype=torch.bfloat16).expand(2, count)),
                 lambda: D.linear_act_q8(row(128, u8), row(4, u8), z(32, 128), z(1, 4)),
                 lambda: D.linear_act_q8(z(1, 128), z(1, 4), row(128, u8), z(1, 4).expand((count + 31) // 32, 4))):
        with pytest.raises(AssertionError, match="2\\^30"):
            call()
    assert not made


def test_counts_past_the_limit_at_the_c_boundary(mods):
    lib = mods.lib.lib()
    p, n, m = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), (1 << 30) + 1
    TOO_LARGE = -6
    assert lib.b200_linear_act(p, 64, p, 64, 0, m, 8, 64, n, 0, n, 0, p, 8, n, 0, n) == TOO_LARGE
    assert lib.b200_linear_act(p, 64, p, 64, 0, 32, m, 64, n, 0, n, 0, p, 1 << 31, n, 0, n) == TOO_LARGE
    assert lib.b200_linear_act(p, 1 << 31, p, 1 << 31, 0, 32, 8, m, n, 0, n, 0, p, 8, n, 0, n) == TOO_LARGE
    assert lib.b200_gated_linear(p, 64, p, 64, 0, m, 8, 64, 2, 0.0, p, 8, n, 0, n) == TOO_LARGE
    assert lib.b200_dense_product(p, 64, 0, p, 64, 0, 0, m, 8, 64, p, 8, n) == TOO_LARGE
    assert lib.b200_linear_act_bwd(p, 8, n, 0, 0, 0, m, 8, p, 8, n, n, 0, n) == TOO_LARGE
    assert lib.b200_gated_linear_bwd(p, 8, p, 16, 2, 0.0, 0, m, 8, p, 16, n) == TOO_LARGE
    assert lib.b200_linear_act_q8(p, p, p, p, 4, m, 8, 128, n, 0, n, 0, p, 8, p, 1 << 40, n) == TOO_LARGE
    assert lib.b200_linear_act_q8(p, p, p, p, 4, 2, m, 128, n, 0, n, 0, p, 1 << 31, p, 1 << 40, n) == TOO_LARGE
