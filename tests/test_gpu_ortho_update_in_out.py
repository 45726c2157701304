"""cavs_ortho_update_in_out: matrices stored [inputs, outputs], whose steps are sized by cols / rows."""
import math

import pytest

from cavs_amd import hip
from test_gpu_ortho_update import U, Case, _desc, _device, _steps, options  # noqa: F401

torch = pytest.importorskip("torch")


def test_refusals_name_the_call():
    d = (hip.OrthoDesc * 1)(_desc(rows=0))
    for name in ("cavs_ortho_update", "cavs_ortho_update_in_out"):
        with pytest.raises(hip.CavsError, match=name + ": matrix 0: unsupported shape"):
            hip.call(name, 0, 1, d, options(), 16, 1 << 40, None)
        hip.call(name, 0, 0, None, options(), None, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_the_step_alone_differs(type_):
    """The matrices of both calls are the same bits; the weights' step is sqrt(max(1, cols / rows)) or sqrt(max(1, rows / cols)) of them."""
    sizes = [(70, 130), (130, 70), (64, 64), (9, 1), (1, 7)]
    o = options()
    cs = {}
    for name in ("cavs_ortho_update", "cavs_ortho_update_in_out"):
        c = Case(3, type_, sizes, momentum=True, weights=True, pad=5)
        W0 = [w.clone() for w in c.W]
        d = c.descs()
        need = hip.lib().cavs_ortho_update_workspace(c.code, len(sizes), d)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        print(f"[case] {name} {type_} {sizes}", flush=True)
        hip.call(name, c.code, len(sizes), d, o, hip.ptr(ws), need, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        cs[name] = c
    for i, (rows, cols) in enumerate(sizes):
        a, b = (cs[n] for n in ("cavs_ortho_update", "cavs_ortho_update_in_out"))
        assert torch.equal(a.O[i], b.O[i]) and torch.equal(a.M[i], b.M[i])
        if rows == cols:
            assert torch.equal(a.W[i], b.W[i])
        # X out of the one call's weights gives the other's: each has its own two roundings of W and of the step
        W = W0[i][:, :cols].double()
        keep = (1 - o.lr * o.weight_decay) * W
        sa, sb = (o.lr * math.sqrt(max(1.0, r)) for r in (rows / cols, cols / rows))
        xa, xb = (keep - a.W[i][:, :cols].double()) / sa, (keep - b.W[i][:, :cols].double()) / sb
        # what W's last places leave of X: (2 U |W| + U |step|) / step, on either side
        off = sum(2 * U * (W.abs() + a.W[i][:, :cols].double().abs() + x.abs() * s) / s for x, s in ((xa, sa), (xb, sb)))
        assert ((xa - xb).abs() <= off).all(), (rows, cols)
        assert (a.W[i][:, cols:] == 5.0).all() and (b.W[i][:, cols:] == 5.0).all()
