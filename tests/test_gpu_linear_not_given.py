"""Operands that are not given, or not read, have no row stride to check (cavs_linear_*)"""
import pytest

from cavs_amd import hip
from test_gpu_linear import Case, _bwd, _fwd, torch


def test_no_strides_of_what_is_not_there():
    _fwd(n=0, X=None, ldx=0, W=None, ldw=0, Y=None, ldy=0, ws=None)
    _bwd(n=0, X=None, ldx=0, W=None, ldw=0, dY=None, lddy=0, dX=None, lddx=0, dW=None, lddw=0, db=None, ws=None)
    _bwd(X=None, ldx=0, W=None, ldw=0, dX=None, lddx=0, dW=None, lddw=0, db=None, ws=None)


@pytest.mark.parametrize("bad", [dict(ldx=7, dX=None), dict(ldw=7, dW=None), dict(ldx=7, db=None), dict(ldw=7, db=None)])
def test_strides_of_what_is_read(bad):
    with pytest.raises(hip.CavsError, match="row stride"):
        _bwd(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,K,N", [(40, 64, 72), (300, 33, 130)])
def test_gradients_of_what_is_given(type_, n, K, N):
    c = Case(type_, n, K, N, "silu", 0.2)
    want, err = c.backward()
    P, st, (ws, need) = hip.ptr, torch.cuda.current_stream().cuda_stream, c.workspace(1)
    for names, X, W in ((["db"], False, False), (["dX", "db"], False, True), (["dW", "db"], True, False), (["dX"], False, True), (["dW"], True, False)):
        out = {k: v for k, v in c.outputs(1).items() if k in names}
        at = lambda k: (P(out.get(k)), out[k].stride(0) if k in out else 0)  # noqa: E731
        print(f"[case] n={n} K={K} N={N} {names}", flush=True)
        hip.call("cavs_linear_bwd", c.code, *((P(c.X), K) if X else (None, 0)), *((P(c.W), K) if W else (None, 0)), P(c.Z), N, hip.ACT["silu"], c.mask, P(c.dY), N,
                 *at("dX"), *at("dW"), at("db")[0], n, K, N, P(ws), need, st)
        torch.cuda.synchronize()
        c.hold(out, want, err)
