"""What dropout drops behind an activation takes no part in the gradients, whatever stands there (cavs_linear_bwd): Z or dY infinite or not a number in dropped places"""
import pytest

from test_gpu_linear import Case, hip, torch


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("act", list(hip.ACT))
@pytest.mark.parametrize("n,K,N", [(90, 64, 72), (300, 33, 130)])
def test_whatever_stands_in_dropped_places(type_, act, n, K, N):
    c = Case(type_, n, K, N, act, 0.3)
    want = c.run(1)
    c.hold(want, *c.backward())
    gone = ~c.keep
    for i, v in enumerate((float("nan"), float("inf"), -float("inf"))):
        for k in ("Z", "dY"):
            part = gone.clone()
            part[:, torch.arange(N, device="cuda") % 3 != i] = False
            getattr(c, k)[:, :N][part] = v
    got = c.run(1)
    assert all(torch.equal(got[k], want[k]) for k in want)
