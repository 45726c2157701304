"""Forward passes of bf16 operands as they lie in the wide tiles, whose last rows and columns are no whole tiles: onto a residual in its own place, with rows' own numbers"""
import pytest

from test_gpu_linear import Case, torch


@pytest.mark.gpu
@pytest.mark.parametrize("n,K,N,act,p", [(8190, 136, 4088, "gelu", 0.1), (4090, 72, 8200, "none", 0.0)])
def test_many_tiles(n, K, N, act, p):
    c = Case("bf16", n, K, N, act, p, True, pads=(8, 16, 3, 1), ids=bool(p))
    want, err = c.forward()
    got = c.run(0)
    c.hold(got, want, err)
    R = c.R.clone()
    onto = c.run(0, out=dict(Y=c.R))["Y"]
    assert torch.equal(onto[:, :N], got["Y"][:, :N]) and bool(onto[:, N:].isnan().all()) and bool(R[:, N:].isnan().all())
