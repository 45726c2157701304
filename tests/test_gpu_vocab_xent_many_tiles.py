"""Losses of more tokens and classes than one dimension of a grid has room for."""
import copy

import pytest

from cavs_amd import hip
from test_gpu_vocab_xent import TYPES, U, Case, _device  # noqa: F401

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("type_,C", [("bf16", 525001), ("f32", 262501)])
def test_losses_of_more_tiles_than_a_grid_dimension_holds(type_, C):
    """A million tokens: 2^24 workgroups and more, 2^32 threads.  What is looked at are rows from everywhere, against the definition."""
    n, H = 1 << 20, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    code, t = TYPES[type_]
    c = Case.__new__(Case)
    c.code, c.t, c.n, c.H, c.C, c.pad, c.dloss, c.scale = code, t, n, H, C, (0, 0, 0, 0), None, 1.0
    c.X, c.W = torch.randn(n, H, generator=g, device="cuda").to(t), torch.randn(C, H, generator=g, device="cuda").to(t)
    c.b = torch.randn(C, generator=g, device="cuda")
    c.labels = torch.floor(torch.rand(n, generator=g, device="cuda") * C).clamp_(max=C - 1)
    o = {k: torch.full((n,), 7.0, device="cuda") for k in ("loss", "lse")}
    o["dX"], o["dW"], o["db"] = c.X, c.W, c.b  # (not written)
    need = hip.lib().cavs_vocab_xent_workspace(code, n, H, C, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    c.call("cavs_vocab_xent_fwd", o, ws, need)
    torch.cuda.synchronize()
    assert ((o["loss"] != 7) & o["loss"].isfinite()).all()
    rows = torch.cat([torch.arange(40), torch.arange(n // 2, n // 2 + 40), torch.arange(n - 40, n), torch.randint(0, n, (40,), generator=torch.Generator().manual_seed(2))]).cuda()
    some = copy.copy(c)
    some.X, some.labels, some.n = c.X[rows], c.labels[rows], len(rows)
    z = some.X.double() @ c.W.double().t() + c.b.double()
    lse = torch.logsumexp(z, 1)
    loss = lse - z[torch.arange(len(rows), device="cuda"), some.labels.long()]
    # bounds as of the other tests: a product's and the bias's roundings, the logarithm's and the sum's
    ez = (H / 16 + 8) * U * (some.X.double().abs() @ c.W.double().abs().t()) + U * z.abs()
    elog = ez.max(1).values + 16 * U + U * lse.abs()
    assert ((o["lse"][rows].double() - lse).abs() <= elog).all()
    assert ((o["loss"][rows].double() - loss).abs() <= elog + ez.max(1).values + U * loss.abs()).all()
