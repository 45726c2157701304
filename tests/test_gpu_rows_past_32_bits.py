"""Dropout and norms of rows that lie more than 2^32 bytes behind the first"""
import pytest

import philox
from cavs_amd import hip
from test_gpu_norm_residual import Case, torch

LD = 1 << 24


def _apart(room, a, at):
    v = torch.as_strided(room, a.shape, (LD, 1), at)
    v.copy_(a)
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_norms(type_):
    n, w = 150, 130
    c = Case(type_, n, w, "rms", "layer", "rows")
    room = torch.zeros((n - 1) * LD + 4096, dtype=c.t, device="cuda")
    for i, k in enumerate(("y", "r", "s", "ds", "dx", "gate_rows")):
        setattr(c, k, _apart(room, getattr(c, k), 256 * i))
    c.pad = LD - w
    want, err = c.forward()
    out = {k: torch.as_strided(room, (n, w), (LD, 1), at) for k, at in (("s", 2048), ("x", 2304))}
    st = torch.cuda.current_stream().cuda_stream
    hip.call("cavs_norm_residual_fwd", c.code, c.desc(), hip.ptr(out["s"]), LD, hip.ptr(out["x"]), LD, st)
    torch.cuda.synchronize()
    for k in out:
        assert bool(((out[k].double() - want[k]).abs() <= err[k]).all()), k
    want, err = c.backward()
    got = {k: torch.as_strided(room, (n, w), (LD, 1), at) for k, at in (("dy", 2048), ("dr", 2304), ("dgate_rows", 2560))}
    got.update({k: torch.empty(w, device="cuda") for k in ("dpre_w", "dpre_b", "dpost_w", "dpost_b")})
    c.run_backward(c.names(), out=got)
    for k in got:
        assert bool(((got[k].double() - want[k]).abs() <= err[k] + 2.0 ** -126).all()), k


@pytest.mark.gpu
@pytest.mark.parametrize("type_,t", [(hip.F32, torch.float32), (hip.BF16, torch.bfloat16)])
def test_dropout(type_, t):
    n, w, p, seed, step = 150, 133, 0.4, 5, 6
    room = torch.zeros((n - 1) * LD + 1024, dtype=t, device="cuda")
    x, r = (_apart(room, torch.randn(n, w, device="cuda").to(t), at) for at in (0, 256))
    y = torch.as_strided(room, (n, w), (LD, 1), 512)
    mask = hip.DropoutMask(p, seed, step, None, None)
    hip.call("cavs_dropout", type_, hip.ptr(y), LD, hip.ptr(x), LD, hip.ptr(r), LD, n, w, mask, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    keep = torch.from_numpy(philox.kept(n, w, p, seed, step)).cuda()
    kept = torch.where(keep, x.double() * philox.factor(p), torch.zeros((), dtype=torch.float64, device="cuda"))
    want, u = r.double() + kept, 2.0 ** -24
    half = 0.0 if t == torch.float32 else torch.finfo(t).eps / 2
    assert bool(((y.double() - want).abs() <= 2 * u * kept.abs() + (u + half) * want.abs() + half * 2 * u * kept.abs()).all())
