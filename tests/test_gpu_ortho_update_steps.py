"""Orthogonalised updates over the whole range of steps and coefficients: what rounding leaves beside a singular value of 0 grows with every
step, a-fold, and has to stay below what a bf16 result holds."""
import math

import pytest

from cavs_amd import hip
from test_gpu_ortho_update import NS, Case, _device, _steps, options  # noqa: F401

torch = pytest.importorskip("torch")

CUBIC, QUINTIC = (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(256, 256), (96, 160), (300, 130)])
@pytest.mark.parametrize("steps,ns", [(5, NS), (6, NS), (8, NS), (10, NS), (15, CUBIC), (16, CUBIC), (30, CUBIC), (10, QUINTIC), (16, QUINTIC)])
def test_a_gradient_of_few_directions_alone(size, steps, ns):
    """A bf16 gradient of small whole numbers, of rank 3 to the last bit: all but three singular values are 0, and what is left of the others is rounding.
    Three parts lose no more than fp32 does, but for up to four roundings a product (six products in two sets of accumulators, three left out) where fp32
    makes one; twice that for chance.  And half a step of bf16."""
    g = torch.Generator().manual_seed(steps + size[0])
    whole = lambda *s: torch.randint(-3, 4, s, generator=g).float()  # noqa: E731
    c = Case(1, "bf16", [size])
    G = whole(size[0], 3) @ whole(3, size[1])  # (27 at most: exact)
    c.G[0].copy_(G)
    o = options(steps=steps, ns=ns)
    c.run(o)
    torch.cuda.synchronize()
    xs = lambda t: _steps(G.double().cuda(), steps, o.eps, (o.a, o.b, o.c), t)[-1].double()  # noqa: E731
    want, plain = xs(torch.float64), xs(torch.float32)
    error, norm = float((c.O[0].double() - want).norm()), float(want.norm())
    assert error <= 8 * float((plain - want).norm()) + torch.finfo(torch.bfloat16).eps / 2 * norm, (error / norm, float((plain - want).norm()) / norm)


@pytest.mark.gpu
def test_the_workspace_is_enough_for_any_options():
    """The query knows the matrices, not the options: the most that any number of steps takes"""
    c = Case(2, "bf16", [(200, 300), (64, 640)])
    for o in (options(steps=1), options(steps=64, ns=CUBIC), options(steps=7)):
        c.run(o)  # (with exactly what the query says)
        torch.cuda.synchronize()
        assert all(x.isfinite().all() for x in c.O)
    need = hip.lib().cavs_ortho_update_workspace(c.code, 2, c.descs())
    for steps in (1, 64):
        with pytest.raises(hip.CavsError, match="workspace of"):
            hip.call("cavs_ortho_update", c.code, 2, c.descs(), options(steps=steps), hip.ptr(c.ws), need - 1, torch.cuda.current_stream().cuda_stream)
