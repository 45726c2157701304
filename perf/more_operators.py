"""Operators of the residual block between a model's states and its head, as their users call them through `cavs_amd.hip`:

  dropout  r + x with elements dropped by a counter-based generator, whose mask is never stored (`cavs_dropout`); the
           gradient is the same call on d y
  norm     norms after and before a block with its gate and residual scale: s = r + scale gate norm(y), x = norm(s)
           (`cavs_norm_residual_fwd`), and the gradients of all of it (`cavs_norm_residual_bwd`)
  linear   R + dropout(act(X W^T + b)) in one product (`cavs_linear_fwd`), and the gradients of X, W and b (`cavs_linear_bwd`)

Types are those of the rows and matrices; biases, the norms' weights, a gate of one value a column, and their gradients are fp32 throughout.
"""
import math

import torch

own = False

# Defaults of every field, so that a case names what is particular to it.
# dropout: p; residual: is added; ids: rows are numbered by the vertex they belong to, not by their place
# norm:    back: gradients; post, pre: the norm of what comes out of the block, of what goes on from the sum (none, rms, layer); bias: of the norms;
#          gate: none, column (one value a column), rows (a matrix)
# linear:  back: gradients; act; p: of a dropout behind the activation; residual: is added; empty: share of the rows whose gradient is zero
_DROPOUT = dict(op="dropout", dtype="f32", n=1024, w=512, p=0.1, residual=False, ids=False)
_NORM = dict(op="norm", dtype="f32", back=False, n=1024, w=512, post="none", pre="rms", bias=False, gate="none", residual=True)
_LINEAR = dict(op="linear", dtype="f32", back=False, n=1024, K=512, N=512, act="none", p=0.0, residual=False, empty=0.0)

_EPS = 1e-5
_ACTS = ["none", "relu", "tanh", "sigmoid", "silu", "gelu"]
_KINDS = ["none", "rms", "layer"]


def listed():
    return [
        # the small chain LSTM of the benchmark (16 sequences of 20 tokens): latency
        dict(_DROPOUT, name="dropout_small_lm", n=320, w=128, p=0.5, ids=True),
        # the benchmark's word-level language model (H = 512, about 7000 tokens of 128 sequences), rows by vertex, odd width
        dict(_DROPOUT, name="dropout_lm_odd", n=7331, w=515, p=0.2, ids=True),
        # a wide model's block output onto its residual stream: the largest
        dict(_DROPOUT, name="dropout_residual_large", dtype="bf16", n=16384, w=4096, residual=True),
        # one token of a wide model: latency
        dict(_NORM, name="norm_token", dtype="bf16", n=1, w=4096, gate="column"),
        # the word-level language model, layer norm before the next block
        dict(_NORM, name="norm_lm", n=7088, w=512, pre="layer", bias=True),
        # its gradients with norms on both sides and a gate of its own rows, odd sizes
        dict(_NORM, name="norm_odd_train", back=True, n=2371, w=1001, post="rms", pre="layer", bias=True, gate="rows"),
        # a wide model's training step: norms on both sides, a learned scale of each column
        dict(_NORM, name="norm_large_train", dtype="bf16", back=True, n=16384, w=4096, post="rms", pre="rms", gate="column"),
        # one token through the widening half of a block: one pass over the weights
        dict(_LINEAR, name="linear_token", dtype="bf16", n=1, K=2048, N=8192, act="silu"),
        # a few sentences scored in fp32, sizes that are no multiple of anything
        dict(_LINEAR, name="linear_sentences", n=157, K=300, N=777, act="tanh", residual=True),
        # the word-level language model's block (512 to 2048) in training, dropout behind the activation
        dict(_LINEAR, name="linear_lm_train", back=True, n=7088, K=512, N=2048, act="relu", p=0.2),
        # a mid-sized model's gradients in bf16, a padded batch
        dict(_LINEAR, name="linear_mid_train", dtype="bf16", back=True, n=4096, K=2048, N=8192, act="gelu", p=0.1, empty=0.25),
        # the narrowing half of a wide block onto the residual stream: the largest
        dict(_LINEAR, name="linear_large", dtype="bf16", n=8192, K=8192, N=4096, p=0.1, residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Half of the users take a multiple of 64, the others any size."""
    v = _log_int(rng, lo, hi)
    return min(hi, max(64, 64 * int(round(v / 64)))) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["dropout", "norm", "linear", "linear"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        t = rng.choice(["f32", "bf16"])
        if op == "dropout":
            c = dict(_DROPOUT, dtype=t, n=_log_int(rng, 1, 65536), w=_size(rng, 32, 8192), p=round(rng.uniform(0.02, 0.6), 3),
                     residual=rng.random() < 0.5, ids=rng.random() < 0.5)
        elif op == "norm":
            c = dict(_NORM, dtype=t, back=rng.random() < 0.5, n=_log_int(rng, 1, 32768), w=_size(rng, 32, 8192), post=rng.choice(_KINDS),
                     pre=rng.choice(_KINDS[1:]), bias=rng.random() < 0.5, gate=rng.choice(["none", "column", "rows"]), residual=rng.random() < 0.8)
        else:
            c = dict(_LINEAR, dtype=t, back=rng.random() < 0.5, n=_log_int(rng, 1, 16384), K=_size(rng, 32, 8192), N=_size(rng, 32, 16384),
                     act=rng.choice(_ACTS), p=rng.choice([0.0, 0.0, 0.1, 0.35]))
            if c["back"]:
                c["empty"] = rng.choice([0.0, 0.0, 0.25])
            else:
                c["residual"] = rng.random() < 0.5
        if _cost(c) <= most:
            return c


# --------------------------------------------------------------------------- what a program has in hand
def _dtype(case):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[case["dtype"]]


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (lambda *shape: torch.randn(*shape, generator=g, device="cuda"), lambda *shape: torch.rand(*shape, generator=g, device="cuda"),
            lambda n: torch.randperm(n, generator=g, device="cuda").int())


def _inputs(case, seed):
    normal, uniform, order = _random(seed)
    t, n = _dtype(case), case["n"]
    d = {"seed": (0x9E3779B97F4A7C15 * (seed + 1)) & (2 ** 64 - 1), "step": 3 * seed + 5}
    if case["op"] == "dropout":
        d["x"] = normal(n, case["w"]).to(t)
        d["r"] = (2 * normal(n, case["w"])).to(t) if case["residual"] else None
        d["ids"] = order(n) if case["ids"] else None
    elif case["op"] == "norm":
        w = case["w"]
        # a residual stream: its rows differ in size, a few of its columns are much larger than the others
        stream = lambda: normal(n, w).mul_(0.5 + 2 * uniform(n, 1)).mul_(1 + 9 * (uniform(w) < 0.01).float()).to(t)  # noqa: E731
        d["y"] = normal(n, w).mul_(0.3 + uniform(n, 1)).to(t)
        d["gate"] = 0.5 + 0.2 * normal(w) if case["gate"] == "column" else None
        d["gate_rows"] = torch.sigmoid(normal(n, w)).to(t) if case["gate"] == "rows" else None
        for k in ("post", "pre"):
            d[k + "_w"] = 1 + 0.2 * normal(w) if case[k] != "none" else None
            d[k + "_b"] = 0.1 * normal(w) if case[k] != "none" and case["bias"] else None
        d["scale"] = 0.7
        if case["back"]:
            d["s"], d["dx"], d["ds"] = stream(), (1e-3 * normal(n, w)).to(t), (1e-3 * normal(n, w)).to(t)
        else:
            d["r"] = stream() if case["residual"] else None
    else:
        K, N = case["K"], case["N"]
        d["X"] = normal(n, K).to(t)
        d["W"] = (normal(N, K) / math.sqrt(K)).to(t)
        if case["back"]:
            d["Z"] = (1.1 * normal(n, N)).to(t) if case["act"] != "none" else None
            d["dY"] = normal(n, N).mul_(1e-3 * (0.2 + uniform(n, 1))).mul_((uniform(n, 1) >= case["empty"]).float()).to(t)
        else:
            d["b"] = 0.3 * normal(N)
            d["R"] = normal(n, N).to(t) if case["residual"] else None
    return d


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    from cavs_amd import hip

    P, n = hip.ptr, case["n"]
    s["hip"] = hip
    s["type"] = {"f32": hip.F32, "bf16": hip.BF16}[case["dtype"]]
    out = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")  # noqa: E731
    need = 0
    if case["op"] == "dropout":
        s["out"] = {"y": torch.empty_like(s["x"])}
        s["mask"] = hip.DropoutMask(case["p"], s["seed"], s["step"], None, P(s["ids"]))
    elif case["op"] == "norm":
        w, like = case["w"], s["y"]
        s["desc"] = hip.NormDesc(n, w, P(s["y"]), w, P(s.get("r")), w, P(s["gate_rows"]), w, P(s["gate"]), s["scale"], _KINDS.index(case["post"]),
                                 P(s["post_w"]), P(s["post_b"]), _KINDS.index(case["pre"]), P(s["pre_w"]), P(s["pre_b"]), _EPS)
        if case["back"]:
            o = s["out"] = {"dy": torch.empty_like(like), "dr": torch.empty_like(like)}
            if case["gate"] == "rows":
                o["dgate_rows"] = torch.empty_like(like)
            if case["gate"] == "column":
                o["dgate"] = out(w)
            for k in ("post_w", "post_b", "pre_w", "pre_b"):
                if s[k] is not None:
                    o["d" + k] = out(w)
            s["grads"] = hip.NormGrads(P(o["dy"]), w, P(o["dr"]), w, P(o.get("dgate_rows")), w, P(o.get("dgate")), P(o.get("dpost_w")),
                                       P(o.get("dpost_b")), P(o.get("dpre_w")), P(o.get("dpre_b")))
            need = hip.lib().cavs_norm_residual_workspace(n, w)
        else:
            s["out"] = {"s": torch.empty_like(like), "x": torch.empty_like(like)}
    else:
        K, N = case["K"], case["N"]
        s["act"] = _ACTS.index(case["act"])
        s["mask"] = hip.DropoutMask(case["p"], s["seed"], s["step"], None, None) if case["p"] else None
        need = hip.lib().cavs_linear_workspace(s["type"], n, K, N, int(case["back"]))
        if case["back"]:
            s["out"] = {"dX": torch.empty_like(s["X"]), "dW": torch.empty_like(s["W"]), "db": out(N)}
        else:  # training keeps Z for its gradients where there is an activation
            s["out"] = {"Y": torch.empty(n, N, dtype=_dtype(case), device="cuda")}
            if case["act"] != "none":
                s["out"]["Z"] = torch.empty_like(s["out"]["Y"])
    s["need"], s["workspace"] = need, torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if not own:
        return {"dropout": _plain_dropout, "norm": _plain_norm_bwd if c.get("back") else _plain_norm,
                "linear": _plain_linear_bwd if c.get("back") else _plain_linear}[c["op"]](s)
    hip, o, n = s["hip"], s["out"], c["n"]
    P, st = hip.ptr, torch.cuda.current_stream().cuda_stream
    if c["op"] == "dropout":
        w = c["w"]
        hip.call("cavs_dropout", s["type"], P(o["y"]), w, P(s["x"]), w, P(s["r"]), w, n, w, s["mask"], st)
    elif c["op"] == "norm":
        w = c["w"]
        if c["back"]:
            hip.call("cavs_norm_residual_bwd", s["type"], s["desc"], P(s["s"]), w, P(s["ds"]), w, P(s["dx"]), w, s["grads"], P(s["workspace"]), s["need"], st)
        else:
            hip.call("cavs_norm_residual_fwd", s["type"], s["desc"], P(o["s"]), w, P(o["x"]), w, st)
    else:
        K, N = c["K"], c["N"]
        if c["back"]:
            hip.call("cavs_linear_bwd", s["type"], P(s["X"]), K, P(s["W"]), K, P(s["Z"]), N, s["act"], s["mask"], P(s["dY"]), N, P(o["dX"]), K, P(o["dW"]), K,
                     P(o["db"]), n, K, N, P(s["workspace"]), s["need"], st)
        else:
            hip.call("cavs_linear_fwd", s["type"], P(s["X"]), K, P(s["W"]), K, P(s["b"]), s["act"], s["mask"], P(s["R"]), N, P(o.get("Z")), N, P(o["Y"]), N,
                     n, K, N, P(s["workspace"]), s["need"], st)
    return o


# --------------------------------------------------------------------------- the plain forms
_M32 = 0xFFFFFFFF


def _threshold(p):
    """p to the nearest multiple of 2^-16 (p is a float of the call)"""
    return min(65535, int(float(torch.tensor(p, dtype=torch.float32)) * 65536 + 0.5))


def _keep(n, w, p, seed, step, ids=None):
    """[n, w]: which elements stay.  Philox4x32 of seven rounds: the key is the seed, the counter (column / 8, row, step); its four words are eight
    draws of 16 bits, low halves first."""
    rows = torch.arange(n, device="cuda") if ids is None else ids.long()
    blocks = (w + 7) // 8
    c0 = torch.arange(blocks, device="cuda")[None, :].expand(n, blocks)
    c1 = rows[:, None].expand(n, blocks)
    c2, c3 = torch.full_like(c0, step & _M32), torch.full_like(c0, step >> 32 & _M32)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(7):  # (products of 64 bits wrap around: their bits are the unsigned ones)
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & _M32) ^ c1 ^ k0, b & _M32, (a >> 32 & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = k0 + 0x9E3779B9 & _M32, k1 + 0xBB67AE85 & _M32
    draws = torch.stack([v for c in (c0, c1, c2, c3) for v in (c & 0xFFFF, c >> 16)], 2)
    return draws.reshape(n, 8 * blocks)[:, :w] >= _threshold(p)


def _dropped(x, p, seed, step, ids=None):
    keep = _keep(x.shape[0], x.shape[1], p, seed, step, ids)
    return torch.where(keep, x * (65536.0 / (65536 - _threshold(p))), torch.zeros_like(x))


def _plain_dropout(s):
    y = _dropped(s["x"].float(), s["case"]["p"], s["seed"], s["step"], s["ids"])
    return {"y": (y if s["r"] is None else y + s["r"].float()).to(s["x"].dtype)}


def _normed(v, kind):
    """v without mean and scale, 1 / its deviation"""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS)
    return v * rstd, rstd


def _norm(v, kind, w, b):
    if kind == "none":
        return v
    v = _normed(v, kind)[0] * w
    return v if b is None else v + b


def _gate(s):
    g = s["gate"] if s["gate_rows"] is None else s["gate_rows"].float()
    return s["scale"] if g is None else s["scale"] * g


def _plain_norm(s):
    c, t = s["case"], s["y"].dtype
    total = _norm(s["y"].float(), c["post"], s["post_w"], s["post_b"]) * _gate(s)
    if s["r"] is not None:
        total = total + s["r"].float()
    return {"s": total.to(t), "x": _norm(total, c["pre"], s["pre_w"], s["pre_b"]).to(t)}


def _norm_bwd(d, v, kind, w):
    """d of v, of the weight and of the bias, from the d of norm(v)"""
    hat, rstd = _normed(v, kind)
    h = d * w
    dv = h - hat * (h * hat).mean(1, keepdim=True)
    if kind == "layer":
        dv = dv - h.mean(1, keepdim=True)
    return rstd * dv, (d * hat).sum(0), d.sum(0)


def _plain_norm_bwd(s):
    c, t, o = s["case"], s["y"].dtype, {}
    ds, dw, db = _norm_bwd(s["dx"].float(), s["s"].float(), c["pre"], s["pre_w"])
    total = s["ds"].float() + ds
    y = s["y"].float()
    z = _norm(y, c["post"], s["post_w"], s["post_b"])
    dgate = s["scale"] * z * total
    dz = _gate(s) * total
    o["dr"] = total.to(t)
    if c["post"] != "none":
        dy, dpw, dpb = _norm_bwd(dz, y, c["post"], s["post_w"])
        o.update(dy=dy.to(t), dpost_w=dpw)
        if s["post_b"] is not None:
            o["dpost_b"] = dpb
    else:
        o["dy"] = dz.to(t)
    if c["gate"] == "rows":
        o["dgate_rows"] = dgate.to(t)
    if c["gate"] == "column":
        o["dgate"] = dgate.sum(0)
    o["dpre_w"] = dw
    if s["pre_b"] is not None:
        o["dpre_b"] = db
    return o


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "tanh":
        return torch.tanh(z)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "tanh":
        return 1.0 - torch.tanh(z).square()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    g = 1.0 / (1.0 + torch.exp(-z))
    return g * (1.0 - g) if act == "sigmoid" else g * (1.0 + z * (1.0 - g))


def _plain_linear(s):
    c, t = s["case"], s["X"].dtype
    z = s["X"].float() @ s["W"].float().t() + s["b"]
    y = _act(z, c["act"])
    if c["p"]:
        y = _dropped(y, c["p"], s["seed"], s["step"])
    if s["R"] is not None:
        y = y + s["R"].float()
    o = {"Y": y.to(t)}
    if c["act"] != "none":
        o["Z"] = z.to(t)
    return o


def _plain_linear_bwd(s):
    c, t = s["case"], s["X"].dtype
    d = s["dY"].float()
    if c["p"]:
        d = _dropped(d, c["p"], s["seed"], s["step"])
    if c["act"] != "none":
        d = d * _slope(s["Z"].float(), c["act"])
    return {"dX": (d @ s["W"].float()).to(t), "dW": (d.t() @ s["X"].float()).to(t), "db": d.sum(0)}


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "dropout":
        x = d["x"].double() * _factors(case, d, case["w"], d["ids"])
        return {"y": x if d["r"] is None else d["r"].double() + x}
    if case["op"] == "norm":
        return _exact_norm_bwd(case, d) if case["back"] else _exact_norm(case, d)
    return _exact_linear_bwd(case, d) if case["back"] else _exact_linear(case, d)


def _factors(case, d, w, ids=None):
    """What dropout multiplies by: 0 or 1 / (share kept).  One word of a block at a time, products of 32 by 32 bits from halves."""
    def product(a, m):  # high and low word
        low, high = (a & 0xFFFF) * m, (a >> 16) * m
        mid = high + (low >> 16)
        return mid >> 16, (mid & 0xFFFF) << 16 | low & 0xFFFF

    n, t = case["n"], _threshold(case["p"])
    out = torch.empty(n, w, dtype=torch.float64, device="cuda")
    column, row = torch.arange(w, device="cuda"), torch.arange(n, device="cuda") if ids is None else ids.long()
    for r in range(0, n, max(1, (1 << 24) // w)):
        rows = row[r:r + max(1, (1 << 24) // w)]
        x = [torch.div(torch.arange(0, w, 8, device="cuda"), 8, rounding_mode="floor").expand(len(rows), -1), rows[:, None], d["step"] % 2 ** 32, d["step"] // 2 ** 32]
        x[1:] = [torch.zeros_like(x[0]) + v for v in x[1:]]
        key = [d["seed"] % 2 ** 32, d["seed"] // 2 ** 32]
        for _ in range(7):
            (h0, l0), (h1, l1) = product(x[0], 0xD2511F53), product(x[2], 0xCD9E8D57)
            x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        for j in range(8):
            mine = column[j::8]
            word = x[j // 2][:, :len(mine)]
            draw16 = torch.div(word, 65536, rounding_mode="floor") if j % 2 else torch.remainder(word, 65536)
            out[r:r + len(rows), j::8] = (draw16 >= t).double() * (65536 / (65536 - t))
    return out


def _exact_norm_of(v, kind, w, b):
    if kind == "none":
        return v
    n = v.shape[1]
    centre = v.sum(1, keepdim=True) / n if kind == "layer" else 0.0
    spread = ((v - centre) ** 2).sum(1, keepdim=True) / n
    out = (v - centre) * (spread + _eps64()).rsqrt() * w.double()
    return out if b is None else out + b.double()


def _eps64():
    return float(torch.tensor(_EPS, dtype=torch.float32))  # (arguments of the call: floats)


def _scale64(d):
    return float(torch.tensor(d["scale"], dtype=torch.float32))


def _gate64(d):
    g = d["gate"] if d["gate"] is not None else d["gate_rows"]
    return torch.ones((), dtype=torch.float64, device="cuda") if g is None else g.double()


def _exact_norm(case, d):
    total = _scale64(d) * _gate64(d) * _exact_norm_of(d["y"].double(), case["post"], d["post_w"], d["post_b"])
    if d["r"] is not None:
        total = total + d["r"].double()
    return {"s": total, "x": _exact_norm_of(total, case["pre"], d["pre_w"], d["pre_b"])}


def _exact_norm_bwd(case, d):
    """The forward definition, differentiated: of <norm(s), dx> by s, and of <scale gate norm(y), that + ds> by all it is made of."""
    leaf = lambda v: None if v is None else v.double().requires_grad_()  # noqa: E731
    rows = max(1, (1 << 25) // case["w"])  # (a stretch of rows at a time: sums over rows add up)
    whole = {}
    for r in range(0, case["n"], rows):
        at = slice(r, r + rows)
        v = {k: leaf(d[k]) for k in ("post_w", "post_b", "pre_w", "pre_b", "gate")}
        v.update(s=leaf(d["s"][at]), y=leaf(d["y"][at]), gate_rows=None if d["gate_rows"] is None else leaf(d["gate_rows"][at]))
        first = [k for k in ("s", "pre_w", "pre_b") if v[k] is not None]
        g1 = dict(zip(first, torch.autograd.grad(_exact_norm_of(v["s"], case["pre"], v["pre_w"], v["pre_b"]), [v[k] for k in first], d["dx"][at].double())))
        through = d["ds"][at].double() + g1["s"]
        z = _scale64(d) * _gate64(v) * _exact_norm_of(v["y"], case["post"], v["post_w"], v["post_b"])
        second = [k for k in ("y", "gate", "gate_rows", "post_w", "post_b") if v[k] is not None]
        g = dict(zip(second, torch.autograd.grad(z, [v[k] for k in second], through)))
        g.update(g1, r=through)
        del g["s"]
        for k, x in g.items():
            if k in ("y", "r", "gate_rows"):
                whole.setdefault("d" + k, []).append(x)
            else:
                whole["d" + k] = x + whole.get("d" + k, 0.0)
    return {k: torch.cat(x) if isinstance(x, list) else x for k, x in whole.items()}


def _exact_act(z, act):
    """act and its derivative"""
    one = torch.ones_like(z)
    if act == "none":
        return z, one
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "tanh":
        h = z.tanh()
        return h, one / z.cosh() ** 2
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    g = torch.sigmoid(z)
    return (g, g * torch.sigmoid(-z)) if act == "sigmoid" else (z * g, g + z * g * torch.sigmoid(-z))


def _exact_linear(case, d):
    z = torch.addmm(d["b"].double(), d["X"].double(), d["W"].double().t())
    y = _exact_act(z, case["act"])[0]
    if case["p"]:
        y = y * _factors(case, d, case["N"])
    if d["R"] is not None:
        y = y + d["R"].double()
    return {"Y": y, "Z": z} if case["act"] != "none" else {"Y": y}


def _exact_linear_bwd(case, d):
    g = d["dY"].double()
    if case["p"]:
        g = g * _factors(case, d, case["N"])
    if case["act"] != "none":
        g = g * _exact_act(d["Z"].double(), case["act"])[1]
    return {"dX": torch.mm(g, d["W"].double()), "dW": torch.mm(g.t(), d["X"].double()), "db": torch.mv(g.t(), torch.ones_like(g[:, 0]))}


# --------------------------------------------------------------------------- what a pass cannot do without
def _rows_moved(c):
    """matrices of n rows that a pass of dropout or norm reads and writes, each once"""
    if c["op"] == "dropout":
        return 3 if c["residual"] else 2
    if c["back"]:
        return 6 + (2 if c["gate"] == "rows" else 0)  # s, dx, ds, y; dr, dy
    return 3 + (1 if c["residual"] else 0) + (1 if c["gate"] == "rows" else 0)  # y; s, x


def _cost(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "linear":  # (fp32 takes the matrix pipe six times as long)
        return work(c)["flops"] * (6 if c["dtype"] == "f32" else 1)
    return size * _rows_moved(c) * c["n"] * c["w"]


def work(case):
    c, n = case, case["n"]
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "dropout":
        return {"bytes": float(size * _rows_moved(c) * n * c["w"] + (4 * n if c["ids"] else 0)), "flops": 2.0 * n * c["w"]}
    if c["op"] == "norm":
        vectors = sum((2 if c["bias"] else 1) for k in ("post", "pre") if c[k] != "none") + (c["gate"] == "column")
        return {"bytes": float(size * _rows_moved(c) * n * c["w"] + 4 * vectors * c["w"] * (2 if c["back"] else 1)),
                "flops": (24.0 if c["back"] else 10.0) * n * c["w"]}
    K, N = c["K"], c["N"]
    if c["back"]:  # X, W, dY (and Z); dX, dW
        b = size * (2 * n * K + 2 * N * K + n * N * (2 if c["act"] != "none" else 1)) + 4 * N
        return {"bytes": float(b), "flops": 4.0 * n * K * N}
    b = size * (n * K + N * K + n * N * (1 + (c["act"] != "none") + c["residual"])) + 4 * N
    return {"bytes": float(b), "flops": 2.0 * n * K * N}
