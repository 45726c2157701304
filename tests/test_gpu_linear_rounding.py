"""What is rounded between the gradients' steps (cavs_linear_bwd in bf16): D = drop(dY), once, and nothing else.

Without an activation D is a product of a bf16 value and dropout's factor in fp32, which torch's fp32 makes bit for bit; so the bound of dX and dW against products of D as
bf16 has it is the product's own, (K / 16 + 40) u sum |D| |W| (u = 2^-24), and half a step of the result."""
import pytest

from test_gpu_linear import Case, U, philox, torch


@pytest.mark.gpu
@pytest.mark.parametrize("n,K,N", [(300, 136, 264), (1024, 512, 1024), (70, 129, 75), (2, 1344, 1500)])
def test_d_is_rounded_once(n, K, N):
    c = Case("bf16", n, K, N, "none", 0.25)
    got = c.run(1)
    factor = torch.tensor(philox.factor(0.25), dtype=torch.float32, device="cuda")
    exact = torch.where(c.keep, c.dY.float() * factor, torch.zeros((), device="cuda"))
    D, X, W, half = exact.to(torch.bfloat16).double(), c.X.double(), c.W.double(), torch.finfo(torch.bfloat16).eps / 2
    for k, want, size, terms in (("dX", D @ W, D.abs() @ W.abs(), N), ("dW", D.t() @ X, D.abs().t() @ X.abs(), n)):
        assert bool(((got[k].double() - want).abs() <= (terms / 16 + 40) * U * size + half * want.abs()).all()), k
    exact = exact.double()
    assert bool(((got["db"].double() - exact.sum(0)).abs() <= (n / 256 + 40) * U * exact.abs().sum(0)).all())
