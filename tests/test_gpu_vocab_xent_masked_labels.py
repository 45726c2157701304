"""Rows of cavs_vocab_xent* whose label names a masked class (a bias of -infinity): their loss is infinite and nothing comes of them, neither in
their row of d X nor in the masked class's of d W and d b, whatever is in that row of W."""
import copy

import pytest

from test_gpu_vocab_xent import Case, _device  # noqa: F401

torch = pytest.importorskip("torch")

INF = float("inf")


def _case(type_, n, H, C, weights, masked=5):
    c = Case(n + H + C, type_, n, H, C, ignored=0.2 if n > 8 else 0.0, masked=masked, weights=weights, pad=(1, 3, 2, 1))
    at = torch.arange(n, device="cuda")
    gone = (at % 3 == 0) & (c.labels >= 0) & (c.labels < C)
    c.labels = torch.where(gone, (C - 1 - at % masked).float(), c.labels)
    c.W[C - masked:, ::2] = float("nan")
    c.W[C - masked:, 1::2] = -INF
    if weights:  # (nothing comes of such a row's weight either)
        c.dloss = torch.where(gone & (at % 2 == 0), torch.full_like(c.dloss, INF), c.dloss)
    return c, gone


def _check(c, gone, o, keys):
    """As rows without a class, but for their loss and lse"""
    rest = copy.copy(c)
    rest.labels = torch.where(gone, torch.full_like(c.labels, -1.0), c.labels)
    if c.dloss is not None:
        rest.dloss = torch.where(gone, torch.zeros_like(c.dloss), c.dloss)
    want, err = rest.want()
    torch.cuda.synchronize()
    assert gone.any()
    has = (c.labels >= 0) & (c.labels < c.C)
    for k in keys:
        got = (o[k][:, :c.H] if k in ("dX", "dW") else o[k]).double()
        w, e = want[k], err[k]
        if k == "loss":
            assert (got[gone] == INF).all()
            got, w, e = got[~gone], w[~gone], e[~gone]
        elif k == "lse":  # (a row without a class may hold anything)
            got, w, e = got[has], w[has], e[has]
        assert ((got - w).abs() <= e).all(), k
    if "dX" in keys:
        assert (o["dX"][:, :c.H][gone] == 0).all() and (o["dW"][c.C - 5:, :c.H] == 0).all() and (o["db"][c.C - 5:] == 0).all()


# few tokens with z kept; packed, up to 64 tokens (bf16: weights beside d) and more; large tiles; W in two orders; several pieces
SHAPES = [(1, 1030, 300), (20, 1025, 3000), (64, 40, 33001), (5, 96, 300), (64, 130, 500), (70, 130, 500), (300, 61, 301), (700, 200, 20011), (2100, 515, 900),
          (1100, 40, 50003)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n,H,C", SHAPES)
def test_gradients(type_, weights, n, H, C):
    c, gone = _case(type_, n, H, C, weights)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    _check(c, gone, o, ("loss", "lse", "dX", "dW", "db"))
    h = c.outputs()
    h["lse"].copy_(o["lse"])
    ws.fill_(0xff)
    c.call("cavs_vocab_xent_bwd", h, ws, need)
    torch.cuda.synchronize()
    for k in ("dX", "dW", "db"):
        assert torch.equal(h[k], o[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", [(1, 64, 32), (40, 200, 777), (64, 130, 3001), (100, 64, 40003), (300, 130, 2000)])
def test_losses(type_, n, H, C):
    c, gone = _case(type_, n, H, C, False)
    o, (ws, need) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", o, ws, need)
    _check(c, gone, o, ("loss", "lse"))
