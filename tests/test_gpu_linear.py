"""Products with bias, activation, dropout and residual in their epilogue, and their gradients (cavs_linear_*), against their definition in 64 bits.

Bounds are computed for every element, in units u = 2^-24 (half a step of a float).
  z       a product of K terms is added up 16 terms a rounding, its pieces once more: (K / 16 + 40) u sum |x| |w|; u |z| for the bias
  act     the error of z times the largest slope (1.13), and of the function 8 u |act(z)|; of gelu, whose tail moves with its argument's rounding, 4 u z^2 phi(z)
          besides
  y       dropout's factor 2 u, the sum u |y|
  slope   16 u (1 + |z|); D = drop(dY) slope: |drop(dY)| times that, 3 u |D|
  dX, dW  D's error, and in bf16 its rounding eps / 2 |D|, through the product, which has z's own bound
  db      D's error summed, and a rounding a term of a chain: (n / 256 + 40) u sum |D|
and each result half a step of its type, finfo.eps / 2, besides.
"""
import math

import numpy as np
import pytest

import philox
from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}
SEED, STEP = 0xFEDCBA9876543210, 77


# ------------------------------------------------------------------ refusals: nothing is launched
def _fwd(**kw):
    a = dict(type=0, X=16, ldx=8, W=16, ldw=8, b=None, act=0, mask=None, R=None, ldr=0, Z=None, ldz=0, Y=16, ldy=12, n=4, K=8, N=12, ws=16, bytes=1 << 40)
    a.update(kw)
    hip.call("cavs_linear_fwd", *a.values(), None)


def _bwd(**kw):
    a = dict(type=0, X=16, ldx=8, W=16, ldw=8, Z=None, ldz=0, act=0, mask=None, dY=16, lddy=12, dX=16, lddx=8, dW=16, lddw=8, db=16, n=4, K=8, N=12, ws=16,
             bytes=1 << 40)
    a.update(kw)
    hip.call("cavs_linear_bwd", *a.values(), None)


_MASKS = [hip.DropoutMask(p, 1, 1, None, None) for p in (1.0, -1.0, float("nan"))]
BOTH = [
    (dict(type=2), "neither"), (dict(n=-1), "bad shape"), (dict(K=0), "bad shape"), (dict(N=0), "bad shape"), (dict(n=(1 << 20) + 1), "unsupported shape"),
    (dict(K=(1 << 16) + 1), "unsupported shape"), (dict(N=(1 << 20) + 1), "unsupported shape"), (dict(n=1 << 20, N=(1 << 16) + 1), "unsupported shape"),
    (dict(act=-1), "unknown activation"), (dict(act=6), "unknown activation"), (dict(ldx=7), "row stride"), (dict(ldw=7), "row stride"), (dict(X=None), "null pointer"),
    (dict(W=None), "null pointer"), (dict(ws=None), "workspace of"), (dict(bytes=1), "workspace of"), (dict(ws=24), "16-byte aligned"),
] + [(dict(mask=m), "not in") for m in _MASKS]


@pytest.mark.parametrize("bad,match", BOTH + [(dict(ldy=11), "row stride"), (dict(R=16, ldr=11), "row stride"), (dict(Z=16, ldz=11), "row stride"),
                                              (dict(Y=None), "null pointer")])
def test_refusals_forward(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        _fwd(**bad)


@pytest.mark.parametrize("bad,match", BOTH + [(dict(lddy=11), "row stride"), (dict(act=1, Z=16, ldz=11), "row stride"), (dict(lddx=7), "row stride"),
                                              (dict(lddw=7), "row stride"), (dict(dY=None), "null pointer"), (dict(act=1, ldz=12), "null pointer")])
def test_refusals_backward(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        _bwd(**bad)


def test_shapes_that_are_refused_have_no_workspace():
    ws = hip.lib().cavs_linear_workspace
    assert ws(2, 4, 8, 12, 0) == 0 and ws(0, 0, 8, 12, 0) == 0 and ws(0, 4, 0, 12, 1) == 0 and ws(0, 4, 8, 0, 1) == 0
    assert ws(0, (1 << 20) + 1, 8, 12, 0) == 0 and ws(1, 4, (1 << 16) + 1, 12, 0) == 0 and ws(1, 1 << 20, 8, (1 << 16) + 1, 0) == 0


def test_calls_that_launch_nothing():
    _fwd(n=0, X=None, Y=None, ws=None)
    _bwd(dX=None, dW=None, db=None, ws=None)
    _bwd(n=0, dW=None, db=None, dY=None, X=None, ws=None)


# ------------------------------------------------------------------ the definition
def act64(z, act):
    """act(z) and its slope"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "tanh":
        return z.tanh(), 1 - z.tanh().square()
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    g = torch.sigmoid(z)
    return (g, g * (1 - g)) if act == "sigmoid" else (z * g, g * (1 + z * (1 - g)))


def act_error(z, act):
    e = 8 * U * act64(z, act)[0].abs()
    return e + 4 * U * z * z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi) if act == "gelu" else e


class Case:
    def __init__(self, type_, n, K, N, act="none", p=0.0, residual=False, bias=True, pads=(0, 0, 0, 0), ids=False, spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(n + 3 * K + 7 * N)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.code, self.t = TYPES[type_]
        self.n, self.K, self.N, self.act, self.p, self.pads = n, K, N, act, p, pads
        self.X, self.W = self.rows(normal(n, K), pads[0]), self.rows(normal(N, K) * spread / math.sqrt(K), pads[1])
        self.b = 0.5 * normal(N) if bias else None
        self.R = self.rows(normal(n, N), pads[2]) if residual else None
        self.Z, self.dY = self.rows(1.3 * normal(n, N), pads[2]), self.rows(1e-2 * normal(n, N), pads[3])
        self.ids = torch.randint(-2 ** 31, 2 ** 31, (n,), generator=g, device="cuda").int() if ids else None
        self.mask = hip.DropoutMask(p, SEED, STEP, None, hip.ptr(self.ids)) if p else None
        keep = philox.kept(n, N, p, SEED, STEP, None if self.ids is None else self.ids.cpu().numpy()) if p else np.ones((n, N), bool)
        self.keep = torch.from_numpy(keep).cuda()

    def rows(self, a, pad, fill=float("nan")):
        s = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=self.t, device="cuda")
        s[:, :a.shape[1]] = a.to(self.t)
        return s

    def eps(self):
        return 0.0 if self.t == torch.float32 else torch.finfo(self.t).eps / 2

    def dropped(self, v):
        return torch.where(self.keep, v * (philox.factor(self.p) if self.p else 1.0), torch.zeros_like(v))

    def forward(self):
        X, W, N = self.X[:, :self.K].double(), self.W[:, :self.K].double(), self.N
        z = X @ W.t() + (self.b.double() if self.b is not None else 0.0)
        ez = (self.K / 16 + 40) * U * (X.abs() @ W.abs().t()) + U * z.abs()
        a, ea = act64(z, self.act)[0], 1.13 * ez + act_error(z, self.act)
        y, ey = self.dropped(a), self.dropped(ea) + 2 * U * self.dropped(a).abs()
        if self.R is not None:
            y = y + self.R[:, :N].double()
            ey = ey + U * y.abs()
        return dict(Y=y, Z=z), dict(Y=ey + self.eps() * y.abs(), Z=ez + self.eps() * z.abs())

    def backward(self):
        X, W, N = self.X[:, :self.K].double(), self.W[:, :self.K].double(), self.N
        g, z = self.dropped(self.dY[:, :N].double()), self.Z[:, :N].double()
        D = g * act64(z, self.act)[1]
        eD = g.abs() * (16 * U * (1 + z.abs()) if self.act not in ("none", "relu") else 0.0) + 3 * U * D.abs()
        eP = eD + self.eps() * D.abs()
        dX, dW, db = D @ W, D.t() @ X, D.sum(0)
        e = dict(dX=eP @ W.abs() + (N / 16 + 40) * U * (D.abs() @ W.abs()) + self.eps() * dX.abs(),
                 dW=eP.t() @ X.abs() + (self.n / 16 + 40) * U * (D.abs().t() @ X.abs()) + self.eps() * dW.abs(),
                 db=eD.sum(0) + (self.n / 256 + 40) * U * D.abs().sum(0))
        return dict(dX=dX, dW=dW, db=db), e

    def workspace(self, back):
        need = hip.lib().cavs_linear_workspace(self.code, self.n, self.K, self.N, back)
        return torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda"), need  # (what is left in it is NaN)

    def outputs(self, back):
        f = lambda r, c, pad: self.rows(torch.full((r, c), 7.0, device="cuda"), pad, 5.0)  # noqa: E731
        n, K, N, p = self.n, self.K, self.N, self.pads
        return dict(dX=f(n, K, p[3]), dW=f(N, K, p[2]), db=torch.full((N,), 7.0, device="cuda")) if back else dict(Y=f(n, N, p[3]), Z=f(n, N, p[0]))

    def run(self, back, names=None, st=None, out=None, ws=None, x=None):
        out = {k: v for k, v in self.outputs(back).items() if names is None or k in names} if out is None else out
        ws, need = self.workspace(back) if ws is None else ws
        P, ld = (lambda k: hip.ptr(out.get(k))), (lambda k: out[k].stride(0) if k in out else 0)  # noqa: E731
        X = self.X if x is None else x
        stream = torch.cuda.current_stream().cuda_stream if st is None else st
        print(f"[case] back={back} type={self.code} n={self.n} K={self.K} N={self.N} {self.act} p={self.p} pads={self.pads} {sorted(out)}", flush=True)
        if back:
            hip.call("cavs_linear_bwd", self.code, hip.ptr(X), X.stride(0), hip.ptr(self.W), self.W.stride(0), hip.ptr(self.Z) if self.act != "none" else None,
                     self.Z.stride(0), hip.ACT[self.act], self.mask, hip.ptr(self.dY), self.dY.stride(0), P("dX"), ld("dX"), P("dW"), ld("dW"), P("db"), self.n,
                     self.K, self.N, hip.ptr(ws), need, stream)
        else:
            hip.call("cavs_linear_fwd", self.code, hip.ptr(X), X.stride(0), hip.ptr(self.W), self.W.stride(0), hip.ptr(self.b), hip.ACT[self.act], self.mask,
                     hip.ptr(self.R), self.R.stride(0) if self.R is not None else 0, P("Z"), ld("Z"), P("Y"), ld("Y"), self.n, self.K, self.N, hip.ptr(ws), need,
                     stream)
        if st is None:
            torch.cuda.synchronize()
            assert bool((ws[need:] == 0xff).all())
        return out

    def hold(self, got, want, err):
        for k, v in got.items():
            w = want[k].shape[-1]
            d = (v[..., :w].double() - want[k]).abs()
            assert bool((d <= err[k] + 2.0 ** -120).all()), (k, float((d - err[k]).max()), float((d / (err[k] + 1e-300)).max()))
            if v.dim() == 2:
                assert bool((v[:, w:] == 5.0).all()), k

    def check(self, fwd=True, back=True):
        if fwd:
            self.hold(self.run(0), *self.forward())
        if back:
            self.hold(self.run(1), *self.backward())


SHAPES = [
    (1, 1, 1), (1, 7, 5), (2, 8, 8), (1, 2048, 300), (1, 300, 2048), (3, 33, 17), (16, 512, 512), (17, 130, 260), (31, 64, 1000), (33, 1000, 40), (64, 256, 256),
    (65, 264, 136), (100, 72, 515), (128, 128, 128), (129, 127, 130), (257, 96, 64), (300, 777, 157), (511, 40, 513), (1000, 320, 256), (2050, 64, 33), (40, 3000, 24),
    (5, 24, 4000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,K,N", SHAPES)
def test_sizes(type_, n, K, N):
    Case(type_, n, K, N, "tanh", 0.25, True).check()
    Case(type_, n, K, N, bias=False).check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,K,N", [(3, 40, 24), (70, 129, 75), (200, 256, 264)])
@pytest.mark.parametrize("pads", [(1, 0, 3, 0), (0, 5, 0, 7), (8, 16, 8, 16), (2, 4, 6, 2)])
def test_row_strides(type_, n, K, N, pads):
    """what is between rows is not a number and not touched; rows off 16 bytes"""
    Case(type_, n, K, N, "silu", 0.3, True, pads=pads, ids=True).check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("act", list(hip.ACT))
@pytest.mark.parametrize("n,spread", [(1, 1.0), (24, 4.0), (140, 1.0)])
def test_activations(type_, act, n, spread):
    Case(type_, n, 160, 200, act, 0.0, True, spread=spread).check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_operands_off_their_alignment(type_):
    """X and W one element behind a 16-byte boundary, strides in whole 16 bytes"""
    c = Case(type_, 150, 128, 144, "relu", 0.1, True, pads=(8, 8, 8, 8))
    for k in ("X", "W", "dY", "Z"):
        v = getattr(c, k)
        room = torch.full((v.numel() + 1,), float("nan"), dtype=c.t, device="cuda")
        moved = room[1:].view(v.shape)
        moved.copy_(v)
        setattr(c, k, moved)
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_what_is_not_wanted(type_, n):
    c = Case(type_, n, 200, 136, "gelu", 0.2, True)
    want, err = c.forward()
    c.hold(c.run(0, ["Y"]), want, err)
    want, err = c.backward()
    for names in (["dX"], ["dW"], ["db"], ["dX", "db"], ["dW", "dX"]):
        c.hold(c.run(1, names), want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 300])
def test_y_onto_its_residual(type_, n):
    c = Case(type_, n, 256, 200, "silu", 0.2, True)
    want = c.run(0, ["Y"])["Y"]
    assert torch.equal(c.run(0, out=dict(Y=c.R))["Y"], want)


@pytest.mark.gpu
def test_no_rows():
    dW, db = torch.full((12, 9), 7.0, device="cuda"), torch.full((12,), 7.0, device="cuda")
    _bwd(n=0, dY=None, X=None, W=None, dX=None, dW=hip.ptr(dW), lddw=9, db=hip.ptr(db), ws=None)
    torch.cuda.synchronize()
    assert not bool(dW[:, :8].any()) and bool((dW[:, 8] == 7.0).all()) and not bool(db.any())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 90, 600])
def test_what_is_not_a_number_keeps_to_its_rows(type_, n):
    """a NaN in a row of X reaches its row of Y and all of dW's column; one in a row of W its column of Y and all of dX's column"""
    c = Case(type_, n, 264, 136, "relu", 0.0, False)
    want, back = c.run(0), c.run(1)
    c.X[1, 5], c.W[7, 9] = float("nan"), float("inf")
    got, gotb = c.run(0), c.run(1)
    rows = torch.arange(n, device="cuda") != 1
    cols = torch.arange(136, device="cuda") != 7
    for k in ("Y", "Z"):
        assert torch.equal(got[k][rows][:, cols], want[k][rows][:, cols]), k
        assert bool(got[k][1].isnan().all()), k
    ks = torch.arange(264, device="cuda")
    assert torch.equal(gotb["dW"][:, ks != 5], back["dW"][:, ks != 5])
    assert torch.equal(gotb["dX"][:, ks != 9], back["dX"][:, ks != 9])
    assert torch.equal(gotb["db"], back["db"])


@pytest.mark.gpu
def test_rows_whose_gradient_is_zero():
    c = Case("bf16", 300, 128, 256, "gelu", 0.1)
    c.dY[::3] = 0
    c.check(fwd=False)
    assert not bool(c.run(1)["dX"][::3].any())


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(hip.ACT))
def test_the_gradient_against_differences(act):
    """<Y, V> along a direction of X, W and b together: central differences of step h are off by h^2 / 6 of the third derivative (of these functions below 2, times
    the direction's third power through z, whose size along it is about 2) and by the values' roundings over h.  relu: its kinks are crossed by the share
    of z that lies within h of 0, each by at most its own step"""
    n, K, N, h = 20, 48, 40, 2.0 ** -6
    c = Case("f32", n, K, N, act, 0.3, True)
    V, dX, dW, db = torch.randn(n, N, device="cuda"), torch.randn(n, K, device="cuda"), torch.randn(N, K, device="cuda") / K ** 0.5, torch.randn(N, device="cuda")

    def value(shift):
        k = Case("f32", n, K, N, act, 0.3, True)
        k.X, k.W, k.b = c.X + shift * dX, c.W + shift * dW, c.b + shift * db
        return float((k.run(0)["Y"].double() * V.double()).sum())

    base = c.run(0)
    c.Z, c.dY = base["Z"], V
    g = c.run(1)
    terms = [(g["dX"].double() * dX.double()), (g["dW"].double() * dW.double()), (g["db"].double() * db.double())]
    slope, size = sum(float(t.sum()) for t in terms), sum(float(t.abs().sum()) for t in terms)
    magnitude = float((base["Y"].double() * V.double()).abs().sum())
    zdir = dX.double() @ c.W.double().t() + c.X.double() @ dW.double().t() + db.double()
    third = float((V.double().abs() * (1.5 * zdir.abs() ** 3 + 4 * zdir.abs() * (dX.double() @ dW.double().t()).abs() + (dX.double() @ dW.double().t()).abs())).sum())
    tol = h * h * third + 64 * U / h * magnitude + 1e-5 * size
    if act == "relu":
        z = base["Z"].double()
        near = z.abs() <= 2 * h * zdir.abs()
        tol += float((2 * V.double().abs() * zdir.abs() * near).sum())
    assert abs((value(h) - value(-h)) / (2 * h) - slope) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,K,N", [("f32", 200, 512, 200), ("bf16", 257, 512, 384), ("bf16", 8, 1024, 512), ("f32", 5, 700, 129)])
def test_results_are_the_same_on_every_call_and_stream(type_, n, K, N):
    """two streams with a workspace each, and a captured call replayed beside eager work, every replay against the eager result"""
    c, e = (Case(type_, n, K, N, "silu", 0.2, True) for _ in range(2))
    want, back = c.run(0), c.run(1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [(k.outputs(0), k.outputs(1), k.workspace(0), k.workspace(1)) for k in (c, e)]
    torch.cuda.synchronize()
    for _ in range(4):
        for k, st, (o0, o1, w0, w1) in zip((c, e), streams, outs):
            k.run(0, st=st.cuda_stream, out=o0, ws=w0)
            k.run(1, st=st.cuda_stream, out=o1, ws=w1)
    torch.cuda.synchronize()
    for o0, o1, _, _ in outs:
        assert all(torch.equal(o0[k], want[k]) for k in want) and all(torch.equal(o1[k], back[k]) for k in back)
    graph = torch.cuda.CUDAGraph()
    o0, o1, w0, w1 = outs[0]
    with torch.cuda.graph(graph, stream=streams[0]):
        c.run(0, st=streams[0].cuda_stream, out=o0, ws=w0)
        c.run(1, st=streams[0].cuda_stream, out=o1, ws=w1)
    for _ in range(3):
        c.X.mul_(-0.5), c.dY.mul_(2.0)
        eager, eagerb = c.run(0), c.run(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o0[k], eager[k]) for k in eager) and all(torch.equal(o1[k], eagerb[k]) for k in eagerb)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_operands_past_32_bits(type_):
    """rows further apart than 2^32 bytes reach: the last rows of X, W and Y, all of whose offsets are above 2^31 elements"""
    code, t = TYPES[type_]
    n, K, N, ld = 150, 64, 130, 1 << 24
    room = torch.zeros((n - 1) * ld + 3 * 256, dtype=t, device="cuda")
    c = Case(type_, n, K, N, "none", 0.0, False)
    X, W, Y = (torch.as_strided(room, (r, w), (ld, 1), off) for r, w, off in ((n, K, 0), (N, K, 256), (n, N, 512)))
    X.copy_(c.X), W.copy_(c.W)
    ws, need = c.workspace(0)
    hip.call("cavs_linear_fwd", code, hip.ptr(X), ld, hip.ptr(W), ld, hip.ptr(c.b), 0, None, None, 0, None, 0, hip.ptr(Y), ld, n, K, N, hip.ptr(ws), need,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want, err = c.forward()
    assert bool(((Y.double() - want["Y"]).abs() <= err["Y"]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,K,N,act", [("bf16", 4104, 2056, 4096, "gelu"), ("bf16", 2048, 1024, 4096, "none"), ("bf16", 8200, 520, 2056, "silu"),
                                             ("f32", 7001, 513, 2041, "relu"), ("f32", 1200, 512, 2048, "none"), ("f32", 300, 2041, 4100, "tanh")])
def test_gradients_of_many_tiles(type_, n, K, N, act):
    """Both products in a launch, in stretches and whole, either the longer; each by itself the same"""
    c = Case(type_, n, K, N, act, 0.1)
    both = c.run(1)
    c.hold(both, *c.backward())
    for k in both:
        assert torch.equal(c.run(1, names={k})[k], both[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,K,N", [(1 << 20, 8, 8), (1 << 20, 3, 1), (8, 8, 1 << 20), (3, 1 << 16, 5)])
def test_the_longest_sides(type_, n, K, N):
    Case(type_, n, K, N, "silu").check()


# ------------------------------------------------------------------ a block, as it is used
@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,F", [("f32", 37, 96, 200), ("bf16", 150, 128, 512), ("bf16", 1, 128, 512)])
def test_a_block_of_them(type_, n, H, F):
    """x = norm(h); u = drop(silu(x W1^T + b1)); y = h + drop(u W2^T + b2), and all gradients, against autograd in 64 bits.  What is rounded between the
    operators (x, u, Z, d u, d x, D) to the type is off by eps / 2 of it each time; a result that is a sum over many such terms is held to 8 such roundings of its
    largest size"""
    code, t = TYPES[type_]
    g = torch.Generator(device="cuda").manual_seed(n)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    h, dy = normal(n, H).to(t), normal(n, H).to(t)
    W1, W2 = (normal(F, H) / H ** 0.5).to(t), (normal(H, F) / F ** 0.5).to(t)
    b1, b2, wn = 0.1 * normal(F), 0.1 * normal(H), 1 + 0.1 * normal(H)
    p, st, P, lib = 0.2, torch.cuda.current_stream().cuda_stream, hip.ptr, hip.lib()
    m1, m2 = hip.DropoutMask(p, 1, STEP, None, None), hip.DropoutMask(p, 2, STEP, None, None)
    new = lambda *s: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    need = max(lib.cavs_linear_workspace(code, n, H, F, 1), lib.cavs_linear_workspace(code, n, F, H, 1), lib.cavs_linear_workspace(code, n, H, F, 0),
               lib.cavs_linear_workspace(code, n, F, H, 0), lib.cavs_norm_residual_workspace(n, H))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    x, u, z, y = new(n, H), new(n, F), new(n, F), new(n, H)
    desc = hip.NormDesc(n, H, P(h), H, None, 0, None, 0, None, 1.0, 0, None, None, hip.NORM_RMS, P(wn), None, 1e-5)
    hip.call("cavs_norm_residual_fwd", code, desc, None, 0, P(x), H, st)
    hip.call("cavs_linear_fwd", code, P(x), H, P(W1), H, P(b1), hip.ACT["silu"], m1, None, 0, P(z), F, P(u), F, n, H, F, P(ws), need, st)
    hip.call("cavs_linear_fwd", code, P(u), F, P(W2), F, P(b2), 0, m2, P(h), H, None, 0, P(y), H, n, F, H, P(ws), need, st)
    du, dx, dh, dW1, dW2 = new(n, F), new(n, H), new(n, H), new(F, H), new(H, F)
    db1, db2, dwn = (torch.empty(k, device="cuda") for k in (F, H, H))
    hip.call("cavs_linear_bwd", code, P(u), F, P(W2), F, None, 0, 0, m2, P(dy), H, P(du), F, P(dW2), F, P(db2), n, F, H, P(ws), need, st)
    hip.call("cavs_linear_bwd", code, P(x), H, P(W1), H, P(z), F, hip.ACT["silu"], m1, P(du), F, P(dx), H, P(dW1), H, P(db1), n, H, F, P(ws), need, st)
    grads = hip.NormGrads(None, 0, P(dh), H, None, 0, None, None, None, P(dwn), None)
    hip.call("cavs_norm_residual_bwd", code, desc, P(h), H, P(dy), H, P(dx), H, grads, P(ws), need, st)
    torch.cuda.synchronize()

    leaves = [v.double().requires_grad_() for v in (h, W1, b1, W2, b2, wn)]
    H64, A, a, B, b, w = leaves
    drop = lambda v, seed: v * torch.from_numpy(philox.kept(n, v.shape[1], p, seed, STEP)).cuda() * philox.factor(p)  # noqa: E731
    X = H64 * (H64.square().mean(1, keepdim=True) + float(torch.tensor(1e-5))).rsqrt() * w
    Z = X @ A.t() + a
    Y = H64 + drop(drop(Z * torch.sigmoid(Z), 1) @ B.t() + b, 2)
    want = torch.autograd.grad(Y, leaves, dy.double())
    eps = max(torch.finfo(t).eps / 2, 16 * U)
    for name, got, exact in [("y", y, Y.detach())] + list(zip(("dh", "dW1", "db1", "dW2", "db2", "dwn"), (dh, dW1, db1, dW2, db2, dwn), want)):
        off = float((got.double() - exact).abs().max() / exact.abs().max())
        assert off <= 8 * eps, (name, off)
