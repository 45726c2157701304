"""The softmax loss over a large vocabulary without logits in memory (cavs_vocab_xent*) against its definition in 64 bits.

Every element is held to a bound that is computed for it, in units u = 2^-24 (half a step of a float):
  z      a product of K terms is added up 16 terms a rounding, the pieces of both sums once more: (K / 16 + 8) u sum |x| |w|, and u |z| for the bias
  lse    the largest error of its row's z, the roundings of the logarithm and of the sum (tiles' sums, in pairs): 16 u, and u |lse|
  p      relative: both of these errors in the exponent, the exponent's own rounding 2 u |z - lse|, the exponential's 4 u
  d      |g| (p's error + u), and where gradients are bf16 half a step of that, 2^-9... of the value: finfo.eps / 2
  sums   each term's error, and a rounding for every sixteen terms of the sum of their magnitudes, two more for stretches and pieces
  gradients   half a step of their type
"""
import copy

import numpy as np
import pytest

from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}


# ------------------------------------------------------------------ refusals: nothing is launched
def _args(**kw):
    a = dict(type=0, X=16, ldx=8, W=16, ldw=8, b=None, labels=16, dloss=None, scale=1.0, loss=16, lse=16, dX=16, lddx=8, dW=16, lddw=8, db=16, n=4, H=8, C=8,
             ws=16, bytes=1 << 40)
    a.update(kw)
    return [a[k] for k in ("type", "X", "ldx", "W", "ldw", "b", "labels", "dloss", "scale", "loss", "lse", "dX", "lddx", "dW", "lddw", "db", "n", "H", "C", "ws",
                           "bytes")] + [None]


@pytest.mark.parametrize("bad,match", [
    (dict(type=2), "neither"), (dict(type=-1), "neither"), (dict(n=-1), "bad shape"), (dict(H=0), "bad shape"), (dict(C=0), "bad shape"),
    (dict(ldx=7), "row stride"), (dict(ldw=7), "row stride"), (dict(lddx=7), "row stride"), (dict(lddw=0), "row stride"),
    (dict(X=None), "null pointer"), (dict(W=None), "null pointer"), (dict(labels=None), "null pointer"),
    (dict(H=(1 << 16) + 1, ldx=1 << 17, ldw=1 << 17, lddx=1 << 17, lddw=1 << 17), "unsupported shape"), (dict(n=(1 << 20) + 1), "unsupported shape"),
    (dict(C=(1 << 23) + 1), "unsupported shape"),
])
def test_refusals(bad, match):
    with pytest.raises(hip.CavsError, match=match):
        hip.call("cavs_vocab_xent", *_args(**bad))


def test_refusals_of_the_halves():
    with pytest.raises(hip.CavsError, match="neither loss nor lse"):
        hip.call("cavs_vocab_xent_fwd", 0, 16, 8, 16, 8, None, 16, None, None, 4, 8, 8, 16, 1 << 40, None)
    with pytest.raises(hip.CavsError, match="null pointer"):
        hip.call("cavs_vocab_xent_bwd", 0, 16, 8, 16, 8, None, 16, None, None, 1.0, 16, 8, 16, 8, 16, 4, 8, 8, 16, 1 << 40, None)


def test_shapes_that_are_refused_have_no_workspace():
    ws = hip.lib().cavs_vocab_xent_workspace
    assert ws(2, 4, 8, 8, 1) == 0 and ws(0, 0, 8, 8, 1) == 0 and ws(0, 4, 0, 8, 0) == 0 and ws(0, 4, 8, 0, 0) == 0
    assert ws(0, (1 << 20) + 1, 8, 8, 0) == 0 and ws(1, 4, (1 << 16) + 1, 8, 0) == 0 and ws(1, 4, 8, (1 << 23) + 1, 0) == 0


# ------------------------------------------------------------------ the definition
class Case:
    def __init__(self, seed, type_, n, H, C, ignored=0.0, masked=0, weights=False, bias=True, pad=(0, 0, 0, 0), lean=4.0, top=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
        self.code, t = TYPES[type_]
        self.t, self.n, self.H, self.C, self.pad = t, n, H, C, pad
        W = normal(C, H) / max(1.0, H ** 0.5) * top
        self.labels = torch.floor(uniform(n) * (C - masked)).clamp_(max=C - masked - 1)
        X = normal(n, H) + lean * uniform(n, 1) * W[self.labels.long()]
        if ignored:
            out = torch.tensor([-1.0, -7.5, float(C), float(C) + 0.5, float("nan"), -float("inf"), float("inf"), 3e9], device="cuda")
            self.labels = torch.where(uniform(n) < ignored, out[torch.arange(n, device="cuda") % len(out)], self.labels)
        self.b = normal(C) if bias else None
        if masked:
            self.b[C - masked:] = -float("inf")
        self.dloss = normal(n) if weights else None
        self.scale = 1.0 / n
        self.X, self.W = self._strided(X, pad[0]), self._strided(W, pad[1])

    def _strided(self, a, pad, fill=float("nan")):
        """a [r, c] of the case's type, rows `pad` further apart, what is between them not a number"""
        s = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=self.t, device="cuda")
        s[:, :a.shape[1]] = a.to(self.t)
        return s

    def want(self):
        H, C = self.H, self.C
        X, W = self.X[:, :H].double(), self.W[:, :H].double()
        has = (self.labels >= 0) & (self.labels < C)
        X = torch.where(has[:, None], X, X.nan_to_num(0.0, 0.0, 0.0))
        b = self.b.double() if self.b is not None else torch.zeros(C, dtype=torch.float64, device="cuda")
        off = b == -float("inf")
        W = torch.where(off[:, None], torch.zeros_like(W), W)
        z = X @ W.t() + b
        ez = (H / 16 + 8) * U * (X.abs() @ W.abs().t()) + U * torch.where(off, torch.zeros_like(z), z.abs())
        lse = torch.logsumexp(z, 1)
        at = torch.where(has, self.labels, torch.zeros_like(self.labels)).long()
        rows = torch.arange(self.n, device="cuda")
        none = lse == -float("inf")
        loss = torch.where(has, torch.where(none, torch.full_like(lse, float("inf")), lse - z[rows, at]), torch.zeros_like(lse))
        elog = ez.max(1).values + 16 * U + U * lse.abs()
        lse_safe = torch.where(none, torch.zeros_like(lse), lse)
        g = torch.where(has & ~none, self.scale * (self.dloss.double() if self.dloss is not None else torch.ones(self.n, dtype=torch.float64, device="cuda")),
                        torch.zeros(self.n, dtype=torch.float64, device="cuda"))
        p = torch.exp(z - lse_safe[:, None])
        far = torch.where(off, torch.zeros_like(z), (z - lse_safe[:, None]).abs())
        rel = torch.expm1(ez + elog[:, None]) + 2 * U * far + 4 * U
        d = p.clone()
        d[rows, at] -= 1
        d *= g[:, None]
        eps = torch.finfo(self.t).eps / 2
        # (below 2^-126 nothing is promised: parts and results of that size may be lost)
        ed = g.abs()[:, None] * (p * rel + U) * (p > 0) + 2.0 ** -126
        ed += 4 * U * d.abs()
        edr = ed + (eps * d.abs() if self.t != torch.float32 else 0.0)
        dX, dW, db = d @ W, d.t() @ X, d.sum(0)
        e = dict(lse=elog, loss=elog + ez[rows, at] + U * loss.abs())
        e["dX"] = edr @ W.abs() + (C / 16 + 64) * U * (d.abs() @ W.abs()) + eps * dX.abs() + 2.0 ** -126
        e["dW"] = edr.t() @ X.abs() + (self.n / 16 + 64) * U * (d.abs().t() @ X.abs()) + eps * dW.abs() + 2.0 ** -126
        e["db"] = ed.sum(0) + (self.n / 16 + 16) * U * d.abs().sum(0)
        return dict(loss=loss, lse=lse, dX=dX, dW=dW, db=db), e

    def outputs(self):
        pad = self.pad
        f = lambda *s: torch.full(s, 7.0, device="cuda")  # noqa: E731
        return dict(loss=f(self.n), lse=f(self.n), db=f(self.C), dX=self._strided(torch.full((self.n, self.H), 7.0, device="cuda"), pad[2], 5.0),
                    dW=self._strided(torch.full((self.C, self.H), 7.0, device="cuda"), pad[3], 5.0))

    def workspace(self, grads):
        need = hip.lib().cavs_vocab_xent_workspace(self.code, self.n, self.H, self.C, grads)
        assert need > 0
        return torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda"), need  # (what is left in it is NaN)

    def call(self, name, o, ws, need, skip=()):
        print(f"[case] {name} type={self.code} n={self.n} H={self.H} C={self.C} pad={self.pad} skip={skip}", flush=True)
        P = lambda k: None if k in skip else hip.ptr(o[k])  # noqa: E731
        st = torch.cuda.current_stream().cuda_stream
        X, W = (hip.ptr(self.X), self.X.stride(0)), (hip.ptr(self.W), self.W.stride(0))
        b, lab, dl = hip.ptr(self.b), hip.ptr(self.labels), hip.ptr(self.dloss)
        tail = (self.n, self.H, self.C, hip.ptr(ws), need, st)
        grads = (P("dX"), o["dX"].stride(0), P("dW"), o["dW"].stride(0), P("db"))
        if name == "cavs_vocab_xent_fwd":
            hip.call(name, self.code, *X, *W, b, lab, P("loss"), P("lse"), *tail)
        elif name == "cavs_vocab_xent_bwd":
            hip.call(name, self.code, *X, *W, b, lab, hip.ptr(o["lse"]), dl, self.scale, *grads, *tail)
        else:
            hip.call(name, self.code, *X, *W, b, lab, dl, self.scale, P("loss"), P("lse"), *grads, *tail)

    def check(self, o, keys=("loss", "lse", "dX", "dW", "db")):
        want, err = self.want()
        torch.cuda.synchronize()
        has = (self.labels >= 0) & (self.labels < self.C)
        for k in keys:
            got = o[k][:, :self.H] if k in ("dX", "dW") else o[k]
            if k in ("dX", "dW"):
                assert (o[k][:, self.H:] == 5.0).all(), f"{k}: written between its rows"
            got, w, e = got.double(), want[k], err[k]
            if k == "lse":  # (of a row without a class that holds NaN it is not looked at)
                got, w, e = got[has], w[has], e[has]
            same = (got == w) | ((got - w).abs() <= e)
            assert same.all(), f"{k}: {int((~same).sum())} of {same.numel()} outside; worst {float(((got - w).abs() / e).nan_to_num(9e9).max()):.3g} times the bound"


@pytest.fixture(autouse=True)
def _device(request):
    if request.node.get_closest_marker("gpu"):
        assert torch.cuda.is_available(), "these tests need the MI355X"
        hip.call("cavs_init", 0)
    yield
    if request.node.get_closest_marker("gpu"):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()


SHAPES = [(1, 64, 256), (1, 1, 1), (2, 5, 3), (3, 33, 64), (17, 64, 65), (64, 128, 63), (65, 100, 257), (130, 300, 1000), (33, 16, 2048), (257, 72, 129),
          (320, 128, 1000), (5, 700, 5001), (1000, 31, 700), (257, 1, 1), (260, 5, 3), (300, 33, 64), (511, 64, 257), (1025, 700, 130), (100, 66, 4097),
          (129, 190, 3000), (250, 64, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", SHAPES)
def test_against_the_definition(type_, n, H, C):
    c = Case(n * 1000 + H + C, type_, n, H, C)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", [(700, 200, 20011), (2300, 512, 4100), (1500, 1030, 9000)])
def test_large_tiles(type_, n, H, C):
    c = Case(n + H, type_, n, H, C, ignored=0.2, masked=11, weights=True)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("f32", 1, 300, 33001), ("f32", 31, 530, 33000), ("f32", 33, 217, 40003), ("f32", 64, 96, 90001), ("bf16", 1, 1025, 33003),
                                         ("bf16", 32, 300, 60001), ("bf16", 40, 700, 35001), ("bf16", 64, 131, 130003)])
def test_few_tokens_and_a_large_vocabulary(type_, n, H, C):
    """W read where it lies: with rows without a class, masked classes whose rows hold no numbers, and rows of W and X further apart than H"""
    c = Case(n + H + C, type_, n, H, C, ignored=0.3 if n > 1 else 0.0, masked=5, weights=True, pad=(1, 3, 2, 1))
    gone = ~((c.labels >= 0) & (c.labels < C))
    c.X[gone, ::2] = float("nan")
    c.W[C - 5:, ::2] = float("inf")
    c.W[C - 5:, 1::2] = float("nan")
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    first = {k: v.clone() for k, v in o.items()}
    ws.fill_(0xff)
    c.call("cavs_vocab_xent", o, ws, need)
    torch.cuda.synchronize()
    for k, v in o.items():  # (lse of a row without a class that holds NaN is NaN)
        assert torch.equal(first[k][..., :H].nan_to_num(9.0) if k in ("dX", "dW") else first[k].nan_to_num(9.0), v[..., :H].nan_to_num(9.0) if k in ("dX", "dW")
                           else v.nan_to_num(9.0)), k


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("f32", 65, 100, 40003), ("f32", 200, 515, 17000), ("bf16", 70, 259, 30001), ("bf16", 129, 1030, 17000), ("bf16", 256, 64, 100001)])
def test_scores_of_more_tokens_and_a_large_vocabulary(type_, n, H, C):
    c = Case(n + H + C, type_, n, H, C, ignored=0.3, masked=5, pad=(1, 3, 0, 0))
    c.W[C - 5:, ::2] = float("nan")
    o, (ws, need) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", o, ws, need)
    c.check(o, ("loss", "lse"))


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("f32", 1100, 40, 50003), ("bf16", 3000, 72, 60001), ("f32", 60, 24, 400003), ("bf16", 50, 12, 1500001)])
def test_several_pieces(type_, n, H, C):
    c = Case(n + H, type_, n, H, C, weights=True)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [(0, 8, 0, 8), (1, 3, 5, 2), (64, 64, 64, 64)])
@pytest.mark.parametrize("n,H,C", [(1, 128, 300), (67, 128, 300), (67, 61, 300), (300, 61, 300), (300, 128, 301)])
def test_strides_rows_without_a_class_masked_classes(type_, pad, n, H, C):
    c = Case(5, type_, n, H, C, ignored=0.4, masked=7, weights=True, pad=pad)
    gone = ~((c.labels >= 0) & (c.labels < C))
    c.X[gone, ::3] = float("nan")
    c.X[gone, 1::3] = float("inf")
    c.W[C - 7:, ::2] = float("nan")
    c.W[C - 7:, 1::2] = -float("inf")
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    assert (o["dX"][:, :H][gone] == 0).all() and (o["dW"][:, :H][C - 7:] == 0).all() and (o["db"][C - 7:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 90, 300])
def test_every_class_masked_or_no_row_with_a_class(type_, n):
    c = Case(6, type_, n, 64, 70)
    c.b[:] = -float("inf")
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    torch.cuda.synchronize()
    assert (o["loss"] == float("inf")).all() and (o["lse"] == -float("inf")).all()
    assert all((o[k][:, :64] == 0).all() for k in ("dX", "dW")) and (o["db"] == 0).all()
    c = Case(7, type_, n, 64, 70)
    c.labels[:] = -1
    o = c.outputs()
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    assert (o["loss"] == 0).all() and all((o[k][:, :64] == 0).all() for k in ("dX", "dW")) and (o["db"] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_no_rows(type_):
    c = Case(8, type_, 1, 40, 90, pad=(0, 0, 3, 3))
    o = c.outputs()
    c.n = 0
    c.call("cavs_vocab_xent", o, None, 0)
    torch.cuda.synchronize()
    assert (o["dW"][:, :40] == 0).all() and (o["db"] == 0).all() and (o["dW"][:, 40:] == 5).all() and (o["loss"] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", [(1, 64, 500), (40, 64, 500), (130, 64, 500), (300, 130, 2000)])
def test_the_halves_are_the_whole(type_, n, H, C):
    """Forward, and backward from its lse, give the whole call's bits; what is not asked for changes nothing else."""
    c = Case(9, type_, n, H, C, ignored=0.2, masked=3, weights=True)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    h, (w0, need0) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", h, w0, need0)
    c.check(h, ("loss", "lse"))
    h2 = c.outputs()
    h2["lse"].copy_(o["lse"])
    ws.fill_(0xff)
    c.call("cavs_vocab_xent_bwd", h2, ws, need)
    torch.cuda.synchronize()
    for k in ("dX", "dW", "db"):
        assert torch.equal(h2[k], o[k]), k
    for skip in (("dX",), ("dW",), ("db",), ("dX", "dW"), ("loss", "lse", "dW", "db"), ("dX", "dW", "db")):
        s = c.outputs()
        ws.fill_(0xff)
        c.call("cavs_vocab_xent", s, ws, need, skip)
        torch.cuda.synchronize()
        for k in ("loss", "lse", "dX", "dW", "db"):
            assert (s[k] == 7.0).all() if k in skip else torch.equal(s[k], o[k]), (skip, k)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_logits_far_apart(type_):
    """Probabilities of one and of next to nothing, logits of hundreds: no overflow, and losses that are small differences of large numbers."""
    c = Case(10, type_, 100, 96, 3001, lean=0.0, top=30.0, bias=False)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_gradients_are_the_differences_of_the_loss(type_):
    """sum_r dloss_r loss_r moves as d X, d W and d b say (central differences in 64 bits of the definition along a direction)."""
    c = Case(11, type_, 24, 48, 130, weights=True, ignored=0.2)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    torch.cuda.synchronize()
    has = (c.labels >= 0) & (c.labels < c.C)
    X, W, b, w = c.X.double(), c.W.double(), c.b.double(), torch.where(has, c.dloss.double() * c.scale, torch.zeros(c.n, device="cuda").double())
    at = torch.where(has, c.labels, torch.zeros_like(c.labels)).long()
    total = lambda X, W, b: (w * torch.nn.functional.cross_entropy(X @ W.t() + b, at, reduction="none")).sum()  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(3)
    for which, k in enumerate(("dX", "dW", "db")):
        v = [torch.zeros_like(t) for t in (X, W, b)]
        v[which] = torch.randn(v[which].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        slope = (total(X + h * v[0], W + h * v[1], b + h * v[2]) - total(X - h * v[0], W - h * v[1], b - h * v[2])) / (2 * h)
        got = (o[k].double() * v[which]).sum()
        size = (o[k].double().abs() * v[which].abs()).sum()
        # half a step of d and of the gradient each; the differences' own h^2 term is below 1e-6 here
        assert abs(got - slope) <= size * (torch.finfo(c.t).eps + 1e-5), (k, float(got), float(slope))


@pytest.mark.gpu
def test_a_workspace_that_is_too_small_or_crooked_is_refused():
    c = Case(12, "f32", 50, 64, 300)
    o, (ws, need) = c.outputs(), c.workspace(1)
    with pytest.raises(hip.CavsError, match="workspace of"):
        c.call("cavs_vocab_xent", o, ws, need - 1)
    with pytest.raises(hip.CavsError, match="workspace of"):
        c.call("cavs_vocab_xent", o, None, need)
    with pytest.raises(hip.CavsError, match="aligned"):
        c.call("cavs_vocab_xent", o, ws[4:], need)
    torch.cuda.synchronize()
    assert (o["loss"] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("f32", 70, 100, 900), ("bf16", 1, 128, 900), ("bf16", 600, 128, 9000)])
def test_the_same_bits_every_time_captured_and_on_another_stream(type_, n, H, C):
    c = Case(13, type_, n, H, C, weights=True)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    torch.cuda.synchronize()
    first = {k: v.clone() for k, v in o.items()}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.call("cavs_vocab_xent", o, ws, need)
    s.synchronize()
    assert all(torch.equal(o[k], first[k]) for k in o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.call("cavs_vocab_xent", o, ws, need)
    X0 = c.X.clone()
    for turn in range(4):
        c.X.copy_(X0 * (1 if turn != 2 else 0.5))
        for v in o.values():
            v.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.clone() for k, v in o.items()}
        c.call("cavs_vocab_xent", o, ws, need)  # eager work of the same program between the replays
        torch.cuda.synchronize()
        for k in ("loss", "lse", "db"):
            assert torch.equal(got[k], o[k]), (turn, k)
        for k in ("dX", "dW"):
            assert torch.equal(got[k][:, :H], o[k][:, :H]), (turn, k)
        if turn != 2:
            assert torch.equal(got["dW"], first["dW"])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [(0, 0, 0, 0), (3, 1, 0, 0), (0, 7, 0, 0)])
@pytest.mark.parametrize("n,H,C", [(1, 1, 1), (1, 64, 32), (1, 1024, 5000), (2, 300, 33), (5, 31, 1000), (32, 65, 40000), (33, 200, 777), (64, 130, 3001), (65, 63, 4096),
                                   (96, 283, 1500), (100, 512, 9000), (129, 100, 2000), (200, 33, 300), (256, 96, 5000), (257, 96, 5000)])
def test_scores(type_, pad, n, H, C):
    c = Case(n + H + C, type_, n, H, C, ignored=0.2 if n > 1 else 0.0, masked=min(3, C - 1), pad=pad)
    o, (ws, need) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", o, ws, need)
    c.check(o, ("loss", "lse"))
    torch.cuda.synchronize()
    assert (o["dX"][:, :H] == 7).all() and (o["db"] == 7).all()


# ------------------------------------------------------------------ few tokens with long rows or many classes, whose z is kept between the passes
@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", [(1, 1030, 33), (2, 1100, 1), (20, 1025, 3000), (32, 1024, 64), (33, 1500, 8100), (64, 40, 33001), (64, 2050, 6001)])
def test_gradients_of_few_tokens(type_, n, H, C):
    c = Case(n + H + C, type_, n, H, C, ignored=0.3 if n > 2 else 0.0, masked=min(3, C - 1), weights=True, pad=(3, 1, 2, 5))
    gone = ~((c.labels >= 0) & (c.labels < C))
    c.X[gone, ::2] = float("nan")
    if C > 3:
        c.W[C - 3:, ::2] = float("nan")
        c.W[C - 3:, 1::2] = -float("inf")
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    assert (o["dX"][:, :H][gone] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,H,C", [(1, 1030, 300), (20, 1025, 3000), (64, 40, 33001)])
def test_the_halves_of_few_tokens(type_, n, H, C):
    test_the_halves_are_the_whole(type_, n, H, C)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("f32", 9, 1026, 900), ("bf16", 50, 32, 40000)])
def test_few_tokens_captured_and_on_another_stream(type_, n, H, C):
    test_the_same_bits_every_time_captured_and_on_another_stream(type_, n, H, C)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,H,C", [("bf16", 5, 1024, 131201), ("f32", 33, 1024, 65700), ("f32", 2, 1027, 65700), ("f32", 3, 8, 1500003)])
def test_few_tokens_and_gradients_larger_than_a_cache(type_, n, H, C):
    """dW of more than 256 MB, in whole lines and not, with rows that follow it left as they were; and classes in several pieces"""
    c = Case(n + C, type_, n, H, C, masked=2)
    o, (ws, need) = c.outputs(), c.workspace(1)
    behind = torch.full((C + 1, H), 7.0, dtype=c.t, device="cuda")
    o["dW"] = behind[:C]
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    assert (behind[C] == 7).all()


# ------------------------------------------------------------------ rows so far apart that offsets pass 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("type_,n,C,pad", [("bf16", 5, 70001, 32700), ("bf16", 100, 70001, 32700), ("bf16", 300, 70001, 32700), ("f32", 64, 35001, 32700),
                                           ("f32", 300, 35001, 32700)])
def test_rows_of_a_table_far_apart(type_, n, C, pad):
    """W and dW of more than 2^32 bytes, few columns of them the matrix's: with and without gradients"""
    H = 61
    c = Case(n + C, type_, n, H, C, ignored=0.2, masked=3, pad=(7, pad, 9, pad))
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    h, (w0, need0) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", h, w0, need0)
    c.check(h, ("loss", "lse"))


@pytest.mark.gpu
def test_a_million_rows():
    """d of a piece of more than 2^32 bytes.  The definition row block by row block; a block's bounds on sums over rows are its share of all rows'."""
    c = Case(77, "f32", 1000003, 32, 1030, ignored=0.1, masked=2)
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    total, bound, step = {}, {}, 125001
    for r in range(0, c.n, step):
        part = copy.copy(c)
        part.X, part.labels = c.X[r:r + step], c.labels[r:r + step]
        part.n = part.X.shape[0]
        want, err = part.want()
        for k in ("loss", "lse", "dX"):
            got, w, e = (v if k == "loss" else v[(part.labels >= 0) & (part.labels < c.C)] for v in (o[k][r:r + step].double(), want[k], err[k]))
            assert ((got - w).abs() <= e).all(), (k, r)
        for k in ("dW", "db"):
            total[k] = total.get(k, 0.0) + want[k]
            bound[k] = bound.get(k, 0.0) + err[k] * (c.n / part.n)
    for k in ("dW", "db"):
        assert ((o[k].double() - total[k]).abs() <= bound[k]).all(), k


@pytest.mark.gpu
def test_recorded_calls_that_share_a_workspace():
    """Two recorded calls, one large and one of few tokens, replayed in turn through one workspace with eager work between"""
    cs = [Case(31, "f32", 500, 70, 900, weights=True), Case(32, "bf16", 20, 1040, 3000, weights=True), Case(33, "bf16", 900, 130, 2000)]
    outs, need = [c.outputs() for c in cs], max(c.workspace(1)[1] for c in cs)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    graphs, first = [], []
    for c, o in zip(cs, outs):
        c.call("cavs_vocab_xent", o, ws, need)
        torch.cuda.synchronize()
        first.append({k: v.clone() for k, v in o.items()})
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.call("cavs_vocab_xent", o, ws, need)
        graphs.append(g)
    for turn in range(3):
        for o in outs:
            for v in o.values():
                v.fill_(3.0)
        for g in graphs if turn != 1 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for o, f in zip(outs, first):
            assert all(torch.equal(o[k], f[k]) for k in o), turn
        cs[turn].call("cavs_vocab_xent", outs[turn], ws, need)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("n,H,C", [(2001, 513, 40), (2050, 600, 3001), (2100, 515, 9000), (2300, 1030, 300)])
def test_many_tokens_and_long_rows(n, H, C):
    """W packed in two orders: with gradients alone, all at once and in halves; masked classes whose rows hold no numbers"""
    c = Case(n + C, "bf16", n, H, C, ignored=0.2, masked=3, weights=True, pad=(1, 3, 2, 0))
    c.W[C - 3:, ::2] = float("nan")
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    h = c.outputs()
    h["lse"].copy_(o["lse"])
    ws.fill_(0xff)
    c.call("cavs_vocab_xent_bwd", h, ws, need)
    torch.cuda.synchronize()
    assert all(torch.equal(h[k], o[k]) for k in ("dX", "dW", "db"))


@pytest.mark.gpu
@pytest.mark.parametrize("n,H,C", [(1, 96, 300), (1, 1100, 2000), (20, 1500, 3000), (40, 130, 500), (64, 64, 40000)])
def test_weights_of_few_tokens_are_not_rounded(n, H, C):
    """bf16, a weight that bf16 would round by all but half a step: rows of dX are the weight times those without one, to the rounding of both results (2 eps,
    and eps^2); so is dW of one token, but for the 2^-16 that two parts leave of the weighted row."""
    c = Case(n + H, "bf16", n, H, C, weights=False)
    one, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", one, ws, need)
    w = 1.0 + 2.0 ** -8 * 0.99
    c.dloss = torch.full((n,), w, device="cuda")
    o = c.outputs()
    c.call("cavs_vocab_xent", o, ws, need)
    c.check(o)
    eps = torch.finfo(torch.bfloat16).eps / 2
    for k in ("dX", "dW")[:2 if n == 1 else 1]:
        got, want = o[k].double(), w * one[k].double()
        assert ((got - want).abs() <= ((1 + eps) / (1 - eps) - 1 + (n == 1) * 2.0 ** -15) * want.abs() + 2.0 ** -126).all(), k
