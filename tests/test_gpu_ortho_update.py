"""Momentum orthogonalised by Newton-Schulz products (cavs_ortho_update) against its definition in 64 bits.

The 2-norm of X's error is held to a bound computed from the definition's own steps.  With X_s after s steps and u = 2^-24 (2^-17 where two
parts are used), a step's map moves an error by at most 4 (its slope is below 3.9 for singular values up to 1.2), step s makes an error of
at most u k |X_s|, k = 14 (8 + sqrt(K / 16)): a product of K terms is rounded once for every 16 and the roundings are as good as
independent, and a + |b| |A| + |c| |A|^2 is below 14; the first one is u |X_0|, from the division.  Results in bf16: half a step more.
fp32 results are also held to three times the error of the same formulas in fp32, which are rounded as often.
"""
import ctypes
import math

import pytest

from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
NS = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}
f32 = lambda v: ctypes.c_float(v).value  # noqa: E731


def options(steps=5, nesterov=1, eps=1e-7, momentum=0.95, lr=0.02, decay=0.01, ns=NS, guard=None):
    return hip.OrthoOptions(steps, nesterov, *ns, eps, momentum, lr, decay, guard)


# ------------------------------------------------------------------ refusals: nothing is launched
def _desc(**kw):
    a = dict(rows=4, cols=4, G=16, ldg=4, M=None, ldm=0, W=None, ldw=0, O=16, ldo=4)
    a.update(kw)
    return hip.OrthoDesc(*[a[k] for k in ("rows", "cols", "G", "ldg", "M", "ldm", "W", "ldw", "O", "ldo")])


@pytest.mark.parametrize("bad,match", [
    (dict(rows=0), "unsupported shape"), (dict(cols=-3), "unsupported shape"), (dict(rows=(1 << 16) + 1), "unsupported shape"), (dict(G=None), "null pointer"),
    (dict(O=None), "neither O nor W"), (dict(ldg=3), "row stride"), (dict(ldo=3), "row stride"), (dict(M=16, ldm=3), "row stride"),
    (dict(W=16, ldw=3), "row stride"),
])
def test_refusals_of_a_matrix(bad, match):
    d = (hip.OrthoDesc * 2)(_desc(), _desc(**bad))
    with pytest.raises(hip.CavsError, match=match):
        hip.call("cavs_ortho_update", 0, 2, d, options(), 16, 1 << 40, None)


def test_refusals_of_a_call():
    d = (hip.OrthoDesc * 1)(_desc())
    for args, match in (((2, 1, d, options()), "neither"), ((0, -1, d, options()), "bad count"), ((0, 1, None, options()), "null pointer"),
                        ((0, 1, d, None), "null pointer"), ((0, 1, d, options(steps=0)), "steps"), ((0, 1, d, options(steps=65)), "steps"),
                        ((0, 1, d, options(eps=-1.0)), "eps"), ((0, 1, d, options(eps=float("nan"))), "eps")):
        with pytest.raises(hip.CavsError, match=match):
            hip.call("cavs_ortho_update", *args, 16, 1 << 40, None)
    hip.call("cavs_ortho_update", 0, 0, None, options(), None, 0, None)  # no matrices: nothing to do
    ws = hip.lib().cavs_ortho_update_workspace
    assert ws(0, 0, None) == 0 and ws(5, 1, d) == 0 and ws(0, 1, (hip.OrthoDesc * 1)(_desc(cols=0))) == 0 and ws(0, 1, None) == 0


# ------------------------------------------------------------------ the definition
def _steps(u, steps, eps, ns, dtype):
    """X_0 .. X_steps of the definition"""
    a, b, c = (f32(v) for v in ns)
    u = u.to(dtype)
    x = u / (u.double().square().sum().sqrt().to(dtype) + f32(eps))
    flat = x.shape[0] <= x.shape[1]
    x = x if flat else x.t().contiguous()
    out = [x]
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * (A @ A)) @ x
        out.append(x)
    return [x if flat else x.t() for x in out]


class Case:
    def __init__(self, seed, type_, sizes, momentum=False, weights=False, orthogonal=True, pad=0, scale=1e-3, rank=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.code, self.t = TYPES[type_]
        self.sizes, self.pad = sizes, pad
        self.G, self.M, self.W, self.O = [], [], [], []
        for rows, cols in sizes:
            v = normal(rows, cols) if rank is None else normal(rows, rank) @ normal(rank, cols)
            self.G.append(self._strided(v * scale, self.t))
            self.M.append(self._strided(2 * scale * normal(rows, cols), torch.float32) if momentum else None)
            self.W.append(self._strided(normal(rows, cols) / math.sqrt(cols), torch.float32) if weights else None)
            self.O.append(self._strided(torch.full((rows, cols), 7.0, device="cuda"), self.t) if orthogonal else None)

    def _strided(self, a, t):
        s = torch.full((a.shape[0], a.shape[1] + self.pad), 5.0, dtype=t, device="cuda")
        s[:, :a.shape[1]] = a.to(t)
        return s

    def descs(self):
        d = (hip.OrthoDesc * len(self.sizes))()
        ld = lambda t: t.stride(0) if t is not None else 0  # noqa: E731
        for i, (rows, cols) in enumerate(self.sizes):
            G, M, W, O = self.G[i], self.M[i], self.W[i], self.O[i]
            d[i] = hip.OrthoDesc(rows, cols, hip.ptr(G), ld(G), hip.ptr(M), ld(M), hip.ptr(W), ld(W), hip.ptr(O), ld(O))
        return d

    def run(self, o, ws=None):
        d = self.descs()
        need = hip.lib().cavs_ortho_update_workspace(self.code, len(self.sizes), d)
        assert need > 0
        if ws is None:
            ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
        print(f"[case] cavs_ortho_update type={self.code} sizes={self.sizes[:4]} x{len(self.sizes)} pad={self.pad} steps={o.steps}", flush=True)
        hip.call("cavs_ortho_update", self.code, len(self.sizes), d, o, hip.ptr(ws), need, torch.cuda.current_stream().cuda_stream)
        self.ws = ws

    def state(self):
        return [t.clone() for t in self.M + self.W + self.O if t is not None]

    def check(self, o, before, fp32_too=True):
        """before: copies of (M, W) as they were"""
        torch.cuda.synchronize()
        mu, lr, decay = o.momentum, o.lr, o.weight_decay
        two = self.t == torch.bfloat16 and all(w is None for w in self.W)
        for i, (rows, cols) in enumerate(self.sizes):
            G = self.G[i][:, :cols].double() if self.O[i] is None or self.O[i].data_ptr() != self.G[i].data_ptr() else self.G0[i][:, :cols].double()
            U_ = G
            if self.M[i] is not None:
                M0 = before[0][i][:, :cols].double()
                M1 = mu * M0 + G
                got = self.M[i][:, :cols].double()
                assert ((got - M1).abs() <= U * M1.abs() + 2.0 ** -149).all()
                U_ = G + mu * got if o.nesterov else got  # (of what is stored; its rounding is the product's below)
            xs = _steps(U_, o.steps, o.eps, (o.a, o.b, o.c), torch.float64)
            K = max(rows, cols)
            k = 14 * (8 + math.sqrt(K / 16))
            u = 2.0 ** -17 if two else U
            norm = [float(x.norm()) for x in xs]
            bound = u * (4.0 ** o.steps * 2 * norm[0] + sum(4.0 ** (o.steps - s) * k * norm[s] for s in range(1, o.steps + 1)))
            x = xs[-1]
            error = bound
            if self.O[i] is not None:
                got = self.O[i][:, :cols].double()
                error = float((got - x).norm())
                rounded = torch.finfo(self.t).eps / 2 * norm[-1]
                assert error <= bound + rounded, (i, rows, cols, error, bound, rounded)
                if two:  # what two parts leave off, grown 485-fold, is no more than one more rounding to bf16
                    assert error <= 2 * rounded + 1e-30, (i, rows, cols, error, rounded)
                if self.t == torch.float32 and fp32_too:
                    plain = float((_steps(U_, o.steps, o.eps, (o.a, o.b, o.c), torch.float32)[-1].double() - x).norm())
                    assert error <= 3 * plain + 8 * U * norm[-1], (i, rows, cols, error, plain)
            if self.W[i] is not None:
                W0 = before[1][i][:, :cols].double()
                s = lr * math.sqrt(max(1.0, rows / cols))
                want = (1 - lr * decay) * W0 - s * x
                # the factor and s are rounded, and the result
                off = (self.W[i][:, :cols].double() - want).norm()
                assert off <= s * bound + 3 * U * (W0.norm() + s * norm[-1]), (i, float(off))
            for t in (self.M[i], self.W[i], self.O[i]):
                assert t is None or (t[:, cols:] == 5.0).all(), "written between the rows"

    def go(self, o, **kw):
        before = [[None if t is None else t.clone() for t in v] for v in (self.M, self.W)]
        self.run(o)
        self.check(o, before, **kw)


@pytest.fixture(autouse=True)
def _device(request):
    if request.node.get_closest_marker("gpu"):
        assert torch.cuda.is_available(), "these tests need the MI355X"
        hip.call("cavs_init", 0)
    yield
    if request.node.get_closest_marker("gpu"):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()


SIZES = [(1, 1), (1, 7), (9, 1), (2, 3), (16, 16), (33, 20), (64, 64), (65, 63), (63, 130), (128, 512), (129, 64), (300, 512), (517, 200), (37, 2003), (1500, 41)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES)
def test_one_matrix(type_, size):
    Case(size[0] * 31 + size[1], type_, [size]).go(options(), fp32_too=min(size) > 1)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_many_matrices_of_all_sizes(type_):
    """More than one launch takes, and with that every size beside every other."""
    Case(1, type_, SIZES + SIZES[::-1], momentum=True, weights=True, pad=3).go(options(), fp32_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[(1024, 1024)] * 4, [(1030, 2500), (900, 700)], [(4000, 1100)], [(100, 20000)]])
def test_large(type_, sizes):
    Case(2, type_, sizes).go(options())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("nesterov", [0, 1])
@pytest.mark.parametrize("momentum,weights,orthogonal", [(True, True, True), (True, True, False), (False, True, False), (True, False, True), (False, True, True)])
def test_momentum_and_weights(type_, nesterov, momentum, weights, orthogonal):
    Case(3, type_, [(70, 130), (130, 70), (64, 64)], momentum, weights, orthogonal, pad=5).go(options(nesterov=nesterov), fp32_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("steps,ns", [(1, NS), (2, NS), (6, NS), (5, (1.5, -0.5, 0.0)), (5, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(type_, steps, ns):
    Case(4, type_, [(96, 160), (50, 20)]).go(options(steps=steps, ns=ns))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1.0, 1e20, 1e36])
def test_the_size_of_a_gradient_does_not_matter(scale):
    Case(5, "f32", [(80, 100)], scale=scale).go(options(eps=0.0), fp32_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("rank", [1, 3])
def test_few_directions(type_, rank):
    """Of a gradient of low rank everything but a few directions is rounding, its own and the products'; both grow."""
    Case(6, type_, [(96, 128), (200, 64)], rank=rank).go(options(), fp32_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_nothing_and_no_numbers(type_):
    c = Case(7, type_, [(40, 70), (70, 40), (20, 20)], weights=True)
    c.G[0][:] = 0
    c.G[1][3, 5] = float("nan")
    c.G[2][3, 5] = float("inf")
    W0 = [w.clone() for w in c.W]
    o = options()
    c.run(o)
    torch.cuda.synchronize()
    assert (c.O[0] == 0).all()
    assert ((c.W[0].double() - (1 - o.lr * o.weight_decay) * W0[0].double()).abs() <= 2 * U * W0[0].abs().double()).all()
    assert c.O[1].isnan().all() and c.O[2].isnan().all() and c.W[1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-7])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_no_gradient_and_no_momentum(type_, eps):
    """U = 0 has no norm to divide by: X is 0, momentum and weights only decay."""
    c = Case(9, type_, [(40, 70), (1, 1), (70, 40)], momentum=True, weights=True)
    for i in (0, 1):
        c.G[i][:] = 0
        c.M[i][:] = 0
    W0 = [w.clone() for w in c.W]
    o = options(eps=eps)
    c.run(o)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert (c.O[i] == 0).all() and (c.M[i] == 0).all()
        assert ((c.W[i].double() - (1 - o.lr * o.weight_decay) * W0[i].double()).abs() <= 2 * U * W0[i].abs().double()).all()
    assert c.O[2].isfinite().all() and (c.O[2] != 0).any() and c.W[2].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_in_place_of_the_gradient(type_):
    c = Case(8, type_, [(90, 130), (130, 90)])
    c.G0 = [g.clone() for g in c.G]
    c.O = c.G
    c.go(options())


@pytest.mark.gpu
def test_blocks_of_one_matrix():
    """Four gates' columns of one weight matrix, each a matrix by itself; the columns between them stay as they are."""
    g = torch.Generator(device="cuda").manual_seed(9)
    E, H, ld = 60, 96, 4 * 96 + 10
    G, W = torch.randn(E, ld, generator=g, device="cuda"), torch.randn(E, ld, generator=g, device="cuda")
    M = torch.zeros(E, ld, device="cuda")
    W0 = W.clone()
    d = (hip.OrthoDesc * 4)()
    for k in range(4):
        at = 4 * k * H
        d[k] = hip.OrthoDesc(E, H, G.data_ptr() + at, ld, M.data_ptr() + at, ld, W.data_ptr() + at, ld, None, 0)
    need = hip.lib().cavs_ortho_update_workspace(0, 4, d)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    o = options(nesterov=0)
    hip.call("cavs_ortho_update", 0, 4, d, o, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(W[:, 4 * H:], W0[:, 4 * H:]) and (M[:, 4 * H:] == 0).all()
    for k in range(4):
        part = slice(k * H, k * H + H)
        x = _steps(G[:, part].double(), 5, o.eps, NS, torch.float64)[-1]
        want = (1 - o.lr * o.weight_decay) * W0[:, part].double() - o.lr * x
        assert (W[:, part].double() - want).norm() <= 1e-5 * want.norm()  # (W's rounding 2^-24, X's error 1e-5 of lr X at most: see above)


@pytest.mark.gpu
def test_a_guard_that_is_up_holds_everything_back():
    c = Case(10, "f32", [(64, 80), (30, 500)], momentum=True, weights=True)
    before = c.state()
    word = torch.ones(1, dtype=torch.int32, device="cuda")
    o = options(guard=word.data_ptr())
    c.run(o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, c.state()))
    word.zero_()
    c.go(o, fp32_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,sizes", [("f32", [(128, 512), (37, 5003), (300, 70)]), ("bf16", [(1024, 1024), (20, 3000)])])
def test_the_same_bits_every_time_captured_and_on_another_stream(type_, sizes):
    c = Case(11, type_, sizes, momentum=True, weights=type_ == "f32")
    start = [None if t is None else t.clone() for t in c.M + c.W]

    def reset():
        for t, s in zip(c.M + c.W, start):
            if t is not None:
                t.copy_(s)

    o = options()
    c.run(o)
    torch.cuda.synchronize()
    first = c.state()
    reset()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.run(o, c.ws)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, c.state()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(o, c.ws)
    for _ in range(4):
        reset()
        for t in c.O:
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, c.state()))
        reset()
        c.run(o, c.ws)  # eager work of the same program between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, c.state()))


@pytest.mark.gpu
def test_a_workspace_that_is_too_small_or_crooked_is_refused():
    c = Case(12, "f32", [(64, 64)])
    d = c.descs()
    need = hip.lib().cavs_ortho_update_workspace(0, 1, d)
    ws = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    for at, room, match in ((ws.data_ptr(), need - 1, "workspace of"), (None, need, "workspace of"), (ws.data_ptr() + 8, need, "aligned")):
        with pytest.raises(hip.CavsError, match=match):
            hip.call("cavs_ortho_update", 0, 1, d, options(), at, room, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (c.O[0] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_,sizes", [("f32", [(9000, 40), (50, 60)]), ("bf16", [(17000, 30)])])
def test_rows_far_apart(type_, sizes):
    """Columns of tables of more than 2^32 bytes: gradients, momentum, weights and results"""
    Case(21, type_, sizes, momentum=True, weights=True, pad=131000).go(options())


@pytest.mark.gpu
def test_recorded_calls_that_share_a_workspace():
    """Two recorded updates replayed in turn through one workspace, the stretches' counters among what they share"""
    cs = [Case(41, "f32", [(128, 512), (128, 512)], momentum=True, weights=True), Case(42, "bf16", [(300, 512), (64, 40)])]
    o = options()
    need = max(hip.lib().cavs_ortho_update_workspace(c.code, len(c.sizes), c.descs()) for c in cs)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    start = [c.state() for c in cs]

    def reset():
        for c, s in zip(cs, start):
            for t, v in zip([t for t in c.M + c.W + c.O if t is not None], s):
                t.copy_(v)

    def call(c):
        hip.call("cavs_ortho_update", c.code, len(c.sizes), c.descs(), o, hip.ptr(ws), need, torch.cuda.current_stream().cuda_stream)

    want = []
    for c in cs:
        call(c)
        torch.cuda.synchronize()
        want.append(c.state())
    graphs = []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c)
        graphs.append(g)
    for turn in range(3):
        reset()
        for g in graphs if turn != 1 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for c, w in zip(cs, want):
            assert all(torch.equal(a, b) for a, b in zip(c.state(), w)), turn
        reset()
        call(cs[turn % 2])
        torch.cuda.synchronize()
