"""Norms after and before a block with its gate and residual scale (cavs_norm_residual_*) against their definition in 64 bits.

Bounds are computed for every element, in units u = 2^-24 (half a step of a float).  Sums of a row are in 64 bits, so a row's mean (as two floats) is exact here
and 1 / deviation has its own rounding u.
  v^      two differences and a product: 3 u |v^|, and with the deviation's 4 u
  norm    v^ w + b: 6 u |v^ w| + 2 u |b|;  in what goes into it with an error e (s, not yet rounded): |w| rstd (e + mean e + |v^| rms e) besides
  s       r + scale gate z: z's error times |scale gate|, 3 u of that product, u |s|
  D       ds + rstd ((h - h1) - v^ h2), h = dx w: 8 u rstd (|h| + mean|h| + |v^| (mean|h v^| + |h2|)), 2 u (|D| + |ds|)
  dz, dgate   scale, gate or z, D: their errors times the others', 4 u of the product
  dy      as D's second part, of dz with its error e: rstd |w| (e + mean e + |v^| rms e) besides
  sums    their terms' errors, and a rounding a term of a workgroup's chain and of the chains' sum: at most (n / 256 + 96) u sum |term|
and each result half a step of its type, finfo.eps / 2, besides.
"""
import itertools

import pytest

from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}
KINDS = ["none", "rms", "layer"]


# ------------------------------------------------------------------ refusals: nothing is launched
def _desc(**kw):
    a = dict(n=4, w=8, y=16, ldy=8, r=None, ldr=0, gate_rows=None, ldg=0, gate=None, scale=1.0, post=0, post_w=None, post_b=None, pre=1, pre_w=None, pre_b=None,
             eps=1e-5)
    a.update(kw)
    return hip.NormDesc(*[a[k] for k, _ in hip.NormDesc._fields_])


def _grads(**kw):
    a = dict(dy=16, lddy=8, dr=16, lddr=8, dgate_rows=None, lddg=0, dgate=None, dpost_w=None, dpost_b=None, dpre_w=None, dpre_b=None)
    a.update(kw)
    return hip.NormGrads(*[a[k] for k, _ in hip.NormGrads._fields_])


BAD = [
    (dict(n=-1), "bad shape"), (dict(w=0), "bad shape"), (dict(w=16385, ldy=16385), "unsupported shape"), (dict(n=1 << 22), "unsupported shape"),
    (dict(post=3), "unknown norm"), (dict(pre=-1), "unknown norm"), (dict(ldy=7), "row stride"), (dict(r=16, ldr=7), "row stride"),
    (dict(gate_rows=16, ldg=7), "row stride"), (dict(gate=16, gate_rows=16, ldg=8), "not both"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
]


@pytest.mark.parametrize("bad,match", BAD + [(dict(y=None), "null pointer")])
def test_refusals_forward(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        hip.call("cavs_norm_residual_fwd", 0, _desc(**bad), 16, 1 << 15, 16, 1 << 15, None)


@pytest.mark.parametrize("bad,match", BAD)
def test_refusals_backward(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        hip.call("cavs_norm_residual_bwd", 0, _desc(**bad), 16, 1 << 15, 16, 1 << 15, 16, 1 << 15, _grads(lddy=1 << 15, lddr=1 << 15), 16, 1 << 40, None)


def test_refusals_of_results():
    fwd = lambda *a: hip.call("cavs_norm_residual_fwd", *a, None)  # noqa: E731
    for args, match in [((2, _desc(), 16, 8, 16, 8), "neither"), ((0, None, 16, 8, 16, 8), "null pointer"), ((0, _desc(), None, 0, None, 0), "neither s nor x"),
                        ((0, _desc(), 16, 7, 16, 8), "row stride"), ((0, _desc(), 16, 8, 16, 7), "row stride")]:
        with pytest.raises(hip.CavsError, match=match):
            fwd(*args)


@pytest.mark.parametrize("desc,given,grads,ws,match", [
    ({}, (16, 16, 16), None, (16, 1 << 40), "null pointer"), ({}, (None, 16, 16), {}, (16, 1 << 40), "null pointer"), ({}, (16, None, None), {}, (16, 1 << 40), "neither ds nor dx"),
    (dict(y=None, gate=16), (16, 16, 16), dict(dgate=16), (16, 1 << 40), "null pointer"), (dict(y=None, post=1), (16, 16, 16), {}, (16, 1 << 40), "null pointer"),
    ({}, (16, 16, 16), dict(dpost_w=16), (16, 1 << 40), "a norm that is not there"), (dict(pre=0), (16, 16, 16), dict(dpre_b=16), (16, 1 << 40), "a norm that is not there"),
    ({}, (16, 16, 16), dict(dgate=16), (16, 1 << 40), "a gate that is not there"), ({}, (16, 16, 16), dict(dgate_rows=16, lddg=8), (16, 1 << 40), "a gate that is not there"),
    ({}, (16, 16, 16), dict(lddr=7), (16, 1 << 40), "row stride"),
])
def test_refusals_of_what_the_gradients_need(desc, given, grads, ws, match):
    s, ds, dx = given
    with pytest.raises(hip.CavsError, match=match):
        hip.call("cavs_norm_residual_bwd", 0, _desc(**desc), s, 8, ds, 8, dx, 8, _grads(**grads) if grads is not None else None, *ws, None)


def test_shapes_that_are_refused_have_no_workspace():
    ws = hip.lib().cavs_norm_residual_workspace
    assert ws(0, 8) == 0 and ws(4, 0) == 0 and ws(4, 16385) == 0 and ws(1 << 22, 8) == 0


# ------------------------------------------------------------------ the definition
def _rows(a, t, pad, fill=float("nan")):
    s = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=t, device="cuda")
    s[:, :a.shape[1]] = a.to(t)
    return s


class Case:
    def __init__(self, type_, n, w, post, pre, gate, bias=True, weights=True, residual=True, offset=0.0, size=1.0, pad=0, scale=0.7, eps=1e-5):
        g = torch.Generator(device="cuda").manual_seed(1000 * n + w)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.code, self.t = TYPES[type_]
        self.n, self.w, self.post, self.pre, self.gate_kind, self.pad, self.scale, self.eps = n, w, post, pre, gate, pad, scale, eps
        rows = lambda a: _rows(a, self.t, pad)  # noqa: E731
        self.y = rows(size * (normal(n, w) + offset))
        self.r = rows(size * 2 * normal(n, w)) if residual else None
        self.s = rows(size * (2 * normal(n, w) + offset))
        self.ds, self.dx = rows(1e-2 * normal(n, w)), rows(1e-2 * normal(n, w))
        self.gate = 1 + 0.3 * normal(w) if gate == "column" else None
        self.gate_rows = rows(torch.sigmoid(normal(n, w))) if gate == "rows" else None
        have = lambda on, v: v if on else None  # noqa: E731
        self.post_w, self.post_b = have(post != "none" and weights, 1 + 0.3 * normal(w)), have(post != "none" and bias, 0.3 * normal(w))
        self.pre_w, self.pre_b = have(pre != "none" and weights, 1 + 0.3 * normal(w)), have(pre != "none" and bias, 0.3 * normal(w))

    def desc(self, y=True):
        P, ld = hip.ptr, self.w + self.pad
        return hip.NormDesc(self.n, self.w, P(self.y) if y else None, ld, P(self.r), ld, P(self.gate_rows), ld, P(self.gate), self.scale, KINDS.index(self.post),
                            P(self.post_w), P(self.post_b), KINDS.index(self.pre), P(self.pre_w), P(self.pre_b), self.eps)

    def d(self, name):
        v = getattr(self, name)
        return None if v is None else v[..., :self.w].double()

    def hat(self, v, kind):
        if kind == "layer":
            v = v - v.mean(1, keepdim=True)
        rstd = ((v * v).mean(1, keepdim=True) + float(torch.tensor(self.eps))).rsqrt()
        return v * rstd, rstd

    def norm(self, v, kind, w, b, e):
        """norm(v) and its error where v has the error e"""
        if kind == "none":
            return v, e
        h, rstd = self.hat(v, kind)
        w = torch.ones_like(v[0]) if w is None else w
        o = h * w
        err = 6 * U * o.abs() + w.abs() * rstd * (e + e.mean(1, keepdim=True) + h.abs() * e.square().mean(1, keepdim=True).sqrt()) * (1 + 1e-3)
        return (o, err + U * o.abs()) if b is None else (o + b, err + 2 * U * b.abs() + U * (o + b).abs())

    def factor(self):
        scale = float(torch.tensor(self.scale, dtype=torch.float32))
        g = self.gate.double() if self.gate is not None else self.d("gate_rows")
        return torch.full((1, 1), scale, dtype=torch.float64, device="cuda") if g is None else scale * g

    def eps_t(self):
        return 0.0 if self.t == torch.float32 else torch.finfo(self.t).eps / 2

    def forward(self):
        d = self.d
        y = d("y")
        z, ez = self.norm(y, self.post, d("post_w"), d("post_b"), torch.zeros_like(y))
        f = self.factor()
        s = f * z + (d("r") if self.r is not None else 0.0)
        es = f.abs() * ez + 3 * U * (f * z).abs() + U * s.abs()
        x, ex = self.norm(s, self.pre, d("pre_w"), d("pre_b"), es)
        return dict(s=s, x=x), dict(s=es + self.eps_t() * s.abs(), x=ex + self.eps_t() * x.abs())

    def norm_bwd(self, g, eg, v, kind, w):
        """the gradient of v from that of norm(v), which has the error eg; and v^"""
        h = g * w
        eh = eg * w.abs() + U * h.abs()
        hat, rstd = self.hat(v, kind)
        m = lambda t: t.mean(1, keepdim=True)  # noqa: E731
        h1, h2 = (m(h) if kind == "layer" else 0.0), m(h * hat)
        o = rstd * (h - h1 - hat * h2)
        e = rstd * (eh + m(eh) + hat.abs() * m(eh * hat.abs())) + 8 * U * rstd * (h.abs() + m(h.abs()) + hat.abs() * (m((h * hat).abs()) + h2.abs()))
        return o, e, hat

    def backward(self, ds=True, dx=True):
        d = self.d
        out, err = {}, {}
        one = torch.ones(self.w, dtype=torch.float64, device="cuda")
        zero = torch.zeros(self.n, self.w, dtype=torch.float64, device="cuda")
        D, eD = (d("ds"), zero) if ds else (zero, zero)
        chain = (self.n / 256 + 96) * U

        def total(name, term, eterm):
            out[name], err[name] = term.sum(0), eterm.sum(0) + chain * term.abs().sum(0)

        if dx and self.pre == "none":
            D = D + d("dx")
        elif dx:
            o, e, hat = self.norm_bwd(d("dx"), zero, d("s"), self.pre, d("pre_w") if self.pre_w is not None else one)
            D, eD = D + o, e
            total("dpre_w", d("dx") * hat, 5 * U * (d("dx") * hat).abs())
            total("dpre_b", d("dx"), zero)
        eD = eD + 2 * U * (D.abs() + (d("ds").abs() if ds else 0.0))
        out["dr"], err["dr"] = D, eD
        y = d("y")
        z, ez = self.norm(y, self.post, d("post_w"), d("post_b"), zero)
        scale, f = float(torch.tensor(self.scale, dtype=torch.float32)), self.factor()
        dgate = scale * D * z
        egate = abs(scale) * (eD * z.abs() + ez * D.abs()) + 4 * U * dgate.abs()
        if self.gate_kind == "rows":
            out["dgate_rows"], err["dgate_rows"] = dgate, egate
        if self.gate_kind == "column":
            total("dgate", dgate, egate)
        dz = f * D
        edz = f.abs() * eD + 4 * U * dz.abs()
        if self.post == "none":
            out["dy"], err["dy"] = dz, edz
        else:
            w = d("post_w") if self.post_w is not None else one
            out["dy"], err["dy"], hat = self.norm_bwd(dz, edz, y, self.post, w)
            total("dpost_w", dz * hat, edz * hat.abs() + 5 * U * (dz * hat).abs())
            total("dpost_b", dz, edz)
        for k in ("dr", "dy", "dgate_rows"):
            if k in out:
                err[k] = err[k] + self.eps_t() * out[k].abs()
        return out, err

    def run_forward(self, s=True, x=True):
        out = {k: _rows(torch.full((self.n, self.w), 7.0, device="cuda"), self.t, self.pad, 5.0) for k, on in (("s", s), ("x", x)) if on}
        ld = self.w + self.pad
        print(f"[case] fwd type={self.code} n={self.n} w={self.w} {self.post} {self.pre} {self.gate_kind}", flush=True)
        hip.call("cavs_norm_residual_fwd", self.code, self.desc(), hip.ptr(out.get("s")), ld, hip.ptr(out.get("x")), ld, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out

    def results(self, names):
        out = {}
        for k in names:
            out[k] = _rows(torch.full((self.n, self.w), 7.0, device="cuda"), self.t, self.pad, 5.0) if k in ("dy", "dr", "dgate_rows") else torch.full(
                (self.w,), 7.0, device="cuda")
        return out

    def names(self, ds=True, dx=True):
        o = ["dy", "dr"] + (["dgate_rows"] if self.gate_kind == "rows" else []) + (["dgate"] if self.gate_kind == "column" else [])
        return o + (["dpre_w", "dpre_b"] if self.pre != "none" and dx else []) + (["dpost_w", "dpost_b"] if self.post != "none" else [])

    def run_backward(self, names, ds=True, dx=True, y=True, st=None, out=None, ws=None):
        out = self.results(names) if out is None else out
        need = hip.lib().cavs_norm_residual_workspace(self.n, self.w)
        ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda") if ws is None else ws
        P, ld = (lambda k: hip.ptr(out.get(k))), self.w + self.pad  # noqa: E731
        g = hip.NormGrads(P("dy"), ld, P("dr"), ld, P("dgate_rows"), ld, P("dgate"), P("dpost_w"), P("dpost_b"), P("dpre_w"), P("dpre_b"))
        print(f"[case] bwd type={self.code} n={self.n} w={self.w} {self.post} {self.pre} {self.gate_kind} {names}", flush=True)
        hip.call("cavs_norm_residual_bwd", self.code, self.desc(y), hip.ptr(self.s), ld, hip.ptr(self.ds) if ds else None, ld, hip.ptr(self.dx) if dx else None, ld, g,
                 hip.ptr(ws), need, st if st is not None else torch.cuda.current_stream().cuda_stream)
        if st is None:
            torch.cuda.synchronize()
            assert bool((ws[need:] == 0xff).all())
        return out

    def hold(self, got, want, err, names=None):
        for k in names or got:
            v = got[k][..., :self.w].double()
            worst = ((v - want[k]).abs() - err[k]).max()
            assert bool(((v - want[k]).abs() <= err[k] + 2.0 ** -126).all()), (k, float(worst))
            if got[k].dim() == 2:
                assert bool((got[k][:, self.w:] == 5.0).all()), k


SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 130), (33, 128), (17, 255), (9, 512), (70, 513), (35, 1001), (6, 2048), (4, 4100), (3, 8191), (2, 16384), (3000, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,w", SHAPES)
def test_sizes(type_, n, w):
    """every width's way of holding a row, both directions, norms of both kinds on both sides"""
    for post, pre, gate in [("rms", "layer", "rows"), ("none", "rms", "column"), ("layer", "none", "none")]:
        c = Case(type_, n, w, post, pre, gate, pad=3 if w < 600 else 0)
        c.hold(c.run_forward(), *c.forward())
        c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre,gate", list(itertools.product(KINDS, KINDS, ["none", "column", "rows"])))
def test_kinds(post, pre, gate):
    c = Case("f32", 29, 300, post, pre, gate)
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())
    c = Case("bf16", 29, 304, post, pre, gate, bias=False, weights=False, residual=False)
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 5000])
def test_many_rows(n):
    c = Case("f32", n, 520, "rms", "layer", "column")
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_the_most_rows(type_):
    c = Case(type_, (1 << 22) - 1, 12, "rms", "layer", "rows")
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("size,offset", [(1e18, 0.0), (1e-12, 0.0), (1.0, 3000.0), (1e25, 0.0)])
def test_values_far_from_one_and_from_zero(size, offset):
    """squares beyond a float's range; means thousands of deviations from 0; deviations far below sqrt(eps)"""
    c = Case("f32", 11, 777, "layer", "layer", "none", residual=False, offset=offset, size=size, scale=1.0)
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
def test_rows_of_zeros_and_one_value():
    c = Case("f32", 4, 65, "rms", "layer", "none", residual=False)
    c.y.zero_(), c.s.fill_(3.0)
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
def test_what_is_not_wanted_and_not_given():
    c = Case("f32", 40, 200, "rms", "layer", "column")
    want, err = c.forward()
    for k in ("s", "x"):
        c.hold(c.run_forward(s=k == "s", x=k == "x"), want, err)
    want, err = c.backward()
    for k in c.names():
        c.hold(c.run_backward([k]), want, err)
    c.hold(c.run_backward(["dr"], y=False), want, err)
    for given in (dict(ds=False), dict(dx=False)):
        want, err = c.backward(**given)
        c.hold(c.run_backward(c.names(**given), **given), want, err)
    got = c.run_backward(["dpre_w", "dpre_b", "dr"], dx=False)  # nothing comes through the norm
    assert not bool(got["dpre_w"].any()) and not bool(got["dpre_b"].any()) and torch.equal(got["dr"], c.ds)


@pytest.mark.gpu
def test_a_norm_alone():
    """y, pre, scale 1; backward from s = y, ds null: dr is the gradient of y"""
    c = Case("bf16", 21, 640, "none", "rms", "none", residual=False, scale=1.0)
    c.s = c.y
    want, err = c.forward()
    c.hold(c.run_forward(s=False), want, err)
    want, err = c.backward(ds=False)
    c.hold(c.run_backward(["dr", "dpre_w", "dpre_b"], ds=False, y=False), want, err)


@pytest.mark.gpu
def test_no_rows():
    out = [torch.full((8,), 7.0, device="cuda") for _ in range(5)]
    P = hip.ptr
    hip.call("cavs_norm_residual_fwd", 0, _desc(n=0, y=None), 16, 8, 16, 8, None)
    hip.call("cavs_norm_residual_bwd", 0, _desc(n=0, post=1, gate=16), None, 8, None, 8, None, 8,
             _grads(dgate=P(out[0]), dpost_w=P(out[1]), dpost_b=P(out[2]), dpre_w=P(out[3]), dpre_b=P(out[4])), None, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert not any(bool(o.any()) for o in out)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_in_place(type_):
    c = Case(type_, 30, 260, "rms", "layer", "rows")
    want = c.run_forward()
    back = c.run_backward(c.names())
    st, ld = torch.cuda.current_stream().cuda_stream, c.w
    for s_in, x_in in (("r", "y"), ("y", "gate_rows"), ("gate_rows", "r")):
        a = Case(type_, 30, 260, "rms", "layer", "rows")
        s, x = getattr(a, s_in), getattr(a, x_in)
        hip.call("cavs_norm_residual_fwd", a.code, a.desc(), hip.ptr(s), ld, hip.ptr(x), ld, st)
        torch.cuda.synchronize()
        assert torch.equal(s, want["s"]) and torch.equal(x, want["x"])
    for dr_in in ("ds", "dx", "s"):
        a = Case(type_, 30, 260, "rms", "layer", "rows")
        out = a.results(a.names())
        out.update(dr=getattr(a, dr_in), dy=a.y, dgate_rows=a.gate_rows)
        a.run_backward(a.names(), out=out)
        assert all(torch.equal(out[k], back[k]) for k in back)


@pytest.mark.gpu
def test_a_row_that_is_not_a_number_keeps_to_itself():
    c = Case("f32", 12, 100, "layer", "rms", "rows")
    clean, back = c.run_forward(), c.run_backward(["dy", "dr", "dgate_rows"])
    c.y[5, 7], c.s[5, 3] = float("inf"), float("nan")
    got, gotb = c.run_forward(), c.run_backward(["dy", "dr", "dgate_rows"])
    others = [i for i in range(12) if i != 5]
    for a, b in ((clean, got), (back, gotb)):
        for k in a:
            assert torch.equal(a[k][others], b[k][others]), k
            assert bool(b[k][5].isnan().all()), k


@pytest.mark.gpu
def test_the_gradient_against_differences():
    """<x(y, r), a> + <s(y, r), c> along a direction: central differences of step h differ from the slope by h^2 / 6 of the third derivative, which for rows of about
    unit deviation is some tens of the direction's own size over sqrt(w) terms, and by the roundings of the two values: 2^-24 times the sum of magnitudes, over h"""
    n, w, h = 6, 96, 2.0 ** -7
    c = Case("f32", n, w, "rms", "layer", "column")
    a, b, dirs = (torch.randn(n, w, device="cuda") for _ in range(3))

    def value(shift):
        k = Case("f32", n, w, "rms", "layer", "column")
        k.y, k.r = c.y + shift * dirs, c.r + shift * dirs
        o = k.run_forward()
        return float((o["x"].double() * a.double()).sum() + (o["s"].double() * b.double()).sum())

    s = c.run_forward()["s"]
    c.s, c.dx, c.ds = s, a, b
    g = c.run_backward(["dy", "dr"])
    slope = float(((g["dy"].double() + g["dr"].double()) * dirs.double()).sum())
    size = float((g["dy"].double().abs() * dirs.double().abs()).sum() + (g["dr"].double().abs() * dirs.double().abs()).sum())
    assert abs((value(h) - value(-h)) / (2 * h) - slope) <= (50 * h * h + 8 * U / h) * size


@pytest.mark.gpu
def test_two_streams_and_a_captured_call():
    """calls on two streams with a workspace each; a captured one replayed beside eager work, every replay against the eager result"""
    c, e = Case("f32", 900, 300, "rms", "rms", "column"), Case("bf16", 333, 1024, "layer", "rms", "rows")
    want, wante = c.run_backward(c.names()), e.run_backward(e.names())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    spaces = [torch.empty(hip.lib().cavs_norm_residual_workspace(k.n, k.w), dtype=torch.uint8, device="cuda") for k in (c, e)]
    outs = [c.results(c.names()), e.results(e.names())]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, st, ws, o in zip((c, e), streams, spaces, outs):
            k.run_backward(k.names(), st=st.cuda_stream, ws=ws, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0][k], want[k]) for k in want) and all(torch.equal(outs[1][k], wante[k]) for k in wante)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        c.run_backward(c.names(), st=streams[0].cuda_stream, ws=spaces[0], out=outs[0])
    for _ in range(3):
        for o in outs[0].values():
            o.fill_(1.0)
        c.dx.mul_(-2.0)
        eager = c.run_backward(c.names())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0][k], eager[k]) for k in eager)
