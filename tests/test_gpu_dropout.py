"""Dropout from a counter-based generator (cavs_dropout) against the generator in numpy.

Bounds, u = 2^-24: the factor and its product are rounded once each, 2 u |x f|, the sum once more, u |y|, and the result to its type,
finfo.eps / 2 |y|.  What is dropped is r, bit for bit.
"""
import numpy as np
import pytest

import philox
from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}
SEED = 0x0123456789ABCDEF


# ------------------------------------------------------------------ the generator
@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
])
def test_generator_known_answers(counter, key, want):
    """vectors of seven rounds that its authors publish with it"""
    assert tuple(int(v) for v in philox.philox4x32(counter, key)) == want


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9])
def test_share_that_is_kept(p):
    """2^18 draws: the share is within five deviations of its own"""
    q = 1 - philox.threshold(p) / 65536
    share = philox.kept(512, 512, p, SEED, 3).mean()
    assert abs(share - q) <= 5 * (q * (1 - q) / 2 ** 18) ** 0.5


# ------------------------------------------------------------------ refusals: nothing is launched
def _call(**kw):
    a = dict(type=0, y=16, ldy=8, x=16, ldx=8, r=None, ldr=0, n=4, w=8, p=0.5)
    a.update(kw)
    hip.call("cavs_dropout", *[a[k] for k in ("type", "y", "ldy", "x", "ldx", "r", "ldr", "n", "w")], hip.DropoutMask(a["p"], 1, 2, None, None), None)


@pytest.mark.parametrize("bad,match", [
    (dict(type=2), "neither"), (dict(type=-1), "neither"), (dict(n=-1), "bad shape"), (dict(w=0), "bad shape"), (dict(ldy=7), "row stride"),
    (dict(ldx=7), "row stride"), (dict(r=16, ldr=7), "row stride"), (dict(y=None), "null pointer"), (dict(x=None), "null pointer"), (dict(p=1.0), "not in"),
    (dict(p=-0.1), "not in"), (dict(p=float("nan")), "not in"), (dict(p=float("inf")), "not in"),
])
def test_refusals(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        _call(**bad)


def test_refusals_of_null_structs_and_no_rows():
    with pytest.raises(hip.CavsError, match="null pointer"):
        hip.call("cavs_dropout", 0, 16, 8, 16, 8, None, 0, 4, 8, None, None)
    with pytest.raises(hip.CavsError, match="null pointer"):
        hip.call("cavs_dropout_advance", None, 1, None)
    _call(n=0, x=None, y=None)


# ------------------------------------------------------------------ on the GPU
def _rows(a, t, pad, fill=float("nan")):
    s = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=t, device="cuda")
    s[:, :a.shape[1]] = a.to(t)
    return s


def _run(code, y, x, r, n, w, mask):
    print(f"[case] type={code} n={n} w={w} p={mask.p}", flush=True)
    hip.call("cavs_dropout", code, hip.ptr(y), y.stride(0), hip.ptr(x), x.stride(0), hip.ptr(r), r.stride(0) if r is not None else 0, n, w, mask,
             torch.cuda.current_stream().cuda_stream)


def _hold(y, x, r, keep, p, t, w):
    """y [n, w + pad] against the definition; what is between its rows is as it was"""
    keep = torch.from_numpy(keep).cuda()
    xf, rf = x[:, :w].double(), r[:, :w].double() if r is not None else torch.zeros(x.shape[0], w, dtype=torch.float64, device="cuda")
    got = y[:, :w].double()
    want = torch.where(keep, xf * philox.factor(p), torch.zeros_like(xf)) + rf
    assert torch.equal(got[~keep], rf[~keep])
    d, v = got[keep], want[keep]
    tol = 2 * U * (v - rf[keep]).abs() + (U + (0 if t == torch.float32 else torch.finfo(t).eps / 2)) * v.abs()
    assert bool(((d - v).abs() <= tol).all()), float(((d - v).abs() - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,w,p,residual,ids,pads", [
    (1, 1, 0.5, False, False, (0, 0, 0)), (1, 8, 0.3, True, False, (0, 0, 0)), (3, 7, 0.5, True, True, (1, 2, 3)), (5, 9, 0.1, False, True, (0, 5, 0)),
    (320, 128, 0.5, False, True, (0, 0, 0)), (257, 515, 0.2, True, True, (0, 0, 0)), (63, 2050, 0.9, True, False, (3, 1, 6)), (2, 20001, 0.25, False, False, (7, 0, 0)),
    (40000, 3, 0.5, True, True, (0, 0, 1)), (1030, 1024, 0.0, True, False, (0, 8, 0)), (129, 64, 0.99999, False, False, (0, 0, 0)),
])
def test_against_the_generator(type_, n, w, p, residual, ids, pads):
    code, t = TYPES[type_]
    g = torch.Generator(device="cuda").manual_seed(n + w)
    x, r = (_rows(torch.randn(n, w, generator=g, device="cuda"), t, pad) for pad in pads[:2])
    r = r if residual else None
    y = _rows(torch.full((n, w), 7.0, device="cuda"), t, pads[2], 5.0)
    rows = np.random.default_rng(n).integers(-2 ** 31, 2 ** 31, n).astype(np.int32) if ids else None
    dev = torch.from_numpy(rows).cuda() if ids else None
    step = (1 << 40) + 17
    _run(code, y, x, r, n, w, hip.DropoutMask(p, SEED, step, None, hip.ptr(dev)))
    torch.cuda.synchronize()
    _hold(y, x, r, philox.kept(n, w, p, SEED, step, rows), p, t, w)
    assert bool((y[:, w:] == 5.0).all())


@pytest.mark.gpu
def test_what_is_dropped_may_be_anything():
    n, w = 64, 80
    keep = torch.from_numpy(philox.kept(n, w, 0.5, SEED, 0)).cuda()
    x = torch.where(keep, torch.ones(n, w, device="cuda"), torch.full((n, w), float("nan"), device="cuda"))
    x[0] = torch.where(keep[0], x[0], torch.full_like(x[0], float("inf")))
    y = torch.empty_like(x)
    _run(hip.F32, y, x, None, n, w, hip.DropoutMask(0.5, SEED, 0, None, None))
    torch.cuda.synchronize()
    assert torch.equal(y, 2 * keep.float())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_in_place_onto_x_and_onto_r(type_):
    code, t = TYPES[type_]
    n, w = 37, 203
    x, r = (torch.randn(n, w, device="cuda").to(t) for _ in range(2))
    mask = hip.DropoutMask(0.4, SEED, 9, None, None)
    y = torch.empty_like(x)
    _run(code, y, x, r, n, w, mask)
    a, b = x.clone(), r.clone()
    _run(code, a, a, r, n, w, mask)
    _run(code, b, x, b, n, w, mask)
    torch.cuda.synchronize()
    assert torch.equal(a, y) and torch.equal(b, y)


@pytest.mark.gpu
def test_the_gradient_is_the_same_call():
    """<drop(x), v> = <x, drop(v)>: exact products by powers of two, so the sums are equal"""
    n, w = 33, 77
    x, v = (torch.randint(-64, 64, (n, w), device="cuda").float() for _ in range(2))
    mask = hip.DropoutMask(0.5, SEED, 4, None, None)
    y, d = torch.empty_like(x), torch.empty_like(x)
    _run(hip.F32, y, x, None, n, w, mask)
    _run(hip.F32, d, v, None, n, w, mask)
    torch.cuda.synchronize()
    assert float((y.double() * v.double()).sum()) == float((x.double() * d.double()).sum())


@pytest.mark.gpu
def test_a_captured_call_draws_anew():
    """the step's word is read as the call runs: every replay is held to its own step, with other work of the stream between them"""
    n, w, p = 50, 130, 0.3
    x = torch.randn(n, w, device="cuda")
    y = torch.empty_like(x)
    word = torch.tensor([(1 << 32) - 2], dtype=torch.int64, device="cuda")
    mask = hip.DropoutMask(p, SEED, 5, hip.ptr(word), None)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            hip.call("cavs_dropout_advance", hip.ptr(word), 1, side.cuda_stream)
            hip.call("cavs_dropout", hip.F32, hip.ptr(y), w, hip.ptr(x), w, None, 0, n, w, mask, side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(1, 5):
        y.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        _hold(y, x, None, philox.kept(n, w, p, SEED, 5 + (1 << 32) - 2 + i), p, torch.float32, w)
        x.mul_(-1.0)


@pytest.mark.gpu
def test_rows_past_32_bits():
    """a matrix of more than 2^32 bytes and elements' offsets above 2^31: its last rows, and no others behind them"""
    w, n = 16384, (1 << 31) // 16384 + 70
    x = torch.ones(n, w, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(n + 1, w, dtype=torch.bfloat16, device="cuda")
    _run(hip.BF16, y, x, None, n, w, hip.DropoutMask(0.5, SEED, 1, None, None))
    torch.cuda.synchronize()
    rows = [0, 1, n // 2, n - 71, n - 2, n - 1]
    keep = philox.kept(len(rows), w, 0.5, SEED, 1, rows)
    assert torch.equal(y[rows].float(), 2 * torch.from_numpy(keep).cuda().float())
    assert not bool(y[n].any())
