"""The dense operators at row counts past what a grid's second dimension holds (65535 blocks of 64 rows)."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
T = torch.bfloat16


@pytest.fixture(scope="module")
def D(pkg):
    return importlib.import_module("dsv41_b200.dense")


@pytest.mark.parametrize("n", [8, 5])
def test_training_step_of_many_rows(D, dev, n):
    """Rows are independent of one another: the same bits as in a call on some of them.  db is a sum over all rows in fp32: relative to the sum of the magnitudes
    off by 2^-23 for each addition that a value goes through, 8 in a thread, 8 over warps, 2048 parts of 64 rows in a thread and 32 over warps, and for the slopes."""
    m, k = 65535 * 64 + 77, 8
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(m, k, generator=g, device=dev).to(T).requires_grad_(True)
    w, b = (torch.randn(n, k, generator=g, device=dev).to(T).requires_grad_(True), torch.randn(n, generator=g, device=dev).to(T).requires_grad_(True))
    gy = torch.randn(m, n, generator=g, device=dev).to(T)
    y = D.linear_act(x, w, b, "silu")
    dx, db = torch.autograd.grad(y, (x, b), gy)
    for lo, hi in ((0, 1000), (65535 * 64 - 500, m)):
        xs = x.detach()[lo:hi].clone().requires_grad_(True)
        ys = D.linear_act(xs, w, b, "silu")
        assert torch.equal(ys, y[lo:hi]) and torch.equal(torch.autograd.grad(ys, xs, gy[lo:hi])[0], dx[lo:hi])
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    s = torch.sigmoid(z)
    dz = gy.double() * s * (1 + z * (1 - s))
    ref, mag = dz.sum(0), (gy.double().abs() * (1 + z.abs())).sum(0)
    eps = (8 + 8 + 2049 + 32) * 2.0 ** -23 + 2.0 ** -18
    assert ((db.double() - ref).abs() <= 2.0 ** -9 * 2 * ref.abs() + eps * mag).all()


@pytest.mark.parametrize("n", [8, 5])
def test_sums_over_many_rows_are_exact_on_integers(D, dev, n):
    """Values of -1, 0 and 1: every partial sum is an integer below 2^24, so that fp32 holds it whatever the order, and the results are its roundings."""
    m, k = 65535 * 64 + 77, 8
    g = torch.Generator(device=dev).manual_seed(2)
    three = lambda *s: torch.randint(-1, 2, s, generator=g, device=dev).to(T)  # noqa: E731
    x, w, b, gy = three(m, k), three(n, k).requires_grad_(True), three(n).requires_grad_(True), three(m, n)
    x[-80:], gy[-80:] = 1, 1  # rows that a sum without them would miss
    x.requires_grad_(True)
    dx, dw, db = torch.autograd.grad(D.linear_act(x, w, b), (x, w, b), gy)
    assert torch.equal(dw, (gy.double().t() @ x.detach().double()).to(T))
    assert torch.equal(db, gy.double().sum(0).to(T))
    assert torch.equal(dx, (gy.double() @ w.detach().double()).to(T))
