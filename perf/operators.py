"""Operators at the end of a language model's training step, as their users call them through `cavs_amd.hip`:

  xent    softmax cross entropy of X W^T + b over a large vocabulary, without logits in memory: the losses
          alone (`cavs_vocab_xent_fwd`: scoring), or with all gradients (`cavs_vocab_xent`: training)
  ortho   a weight matrix's momentum, orthogonalised by Newton-Schulz products, several matrices a call
          (`cavs_ortho_update`): the orthogonal matrix alone, or with the update of momentum and weights

Types are those of the operands and of what is returned in their place (X, W, d X, d W; the gradient and the
orthogonal matrix); losses, biases, momentum and updated weights are fp32 throughout.
"""
import math

import torch

own = False

# Defaults of every field, so that a case names what is particular to it.
# xent:  grads: with gradients; ignored: share of the rows without a class (padding of a batch); weights: rows carry a weight of their own
#        masked: so many of the last classes are padding of the table, shut off by a bias of -inf
# ortho: sizes "rows x cols, ..." of the matrices of a call; update: momentum and weights take part
_XENT = dict(op="xent", dtype="f32", grads=True, n=1024, H=512, C=10000, ignored=0.0, weights=False, masked=0)
_ORTHO = dict(op="ortho", dtype="f32", sizes="512x512", steps=5, update=False)

# Newton-Schulz coefficients that lift small singular values fast (they end between 0.7 and 1.2, not at 1)
_NS = (3.4445, -4.7750, 2.0315)
_EPS, _MU, _LR, _DECAY = 1e-7, 0.95, 0.02, 0.01


def listed():
    return [
        # one token's loss under a vocabulary of 32000: latency, and one pass over the weights
        dict(_XENT, name="score_token", dtype="bf16", grads=False, n=1, H=1024, C=32000),
        # a few sentences rescored in fp32, sizes that are no multiple of anything
        dict(_XENT, name="score_sentences", grads=False, n=157, H=300, C=21701),
        # the small chain LSTM of the benchmark (16 sequences of 20 tokens): the smallest training step
        dict(_XENT, name="small_lm_train", n=320, H=128, C=1000),
        # the benchmark's word-level language model (H = 512, 10000 classes, about 7000 tokens of 128 sequences)
        dict(_XENT, name="lm_train", n=7088, H=512, C=10000),
        # a padded batch in bf16: rows without a class, weighted rows, a table with padding classes, odd sizes
        dict(_XENT, name="padded_batch_train", dtype="bf16", n=2371, H=1000, C=25040, ignored=0.3, weights=True, masked=39),
        # a mid-sized language model in bf16
        dict(_XENT, name="mid_lm_train", dtype="bf16", n=4096, H=2048, C=50000),
        # the largest: a wide model over a vocabulary of 128000
        dict(_XENT, name="large_vocab_train", dtype="bf16", n=8192, H=4096, C=128000),
        # the benchmark's Tree-LSTM (E = 300, H = 512): eight matrices, momentum and weights with them
        dict(_ORTHO, name="treelstm_update", sizes="300x512,300x512,300x512,300x512,512x512,512x512,512x512,512x512", update=True),
        # a small LSTM's, latency
        dict(_ORTHO, name="small_lstm_update", sizes="128x512,128x512", update=True),
        # the benchmark's widest Tree-LSTM (E = H = 1024)
        dict(_ORTHO, name="wide_treelstm_update", sizes=",".join(["1024x1024"] * 8), update=True),
        # odd sizes, tall and flat, in one call
        dict(_ORTHO, name="odd_matrices", sizes="1023x517,37x5003,700x701,2000x1"),
        # a wide model's matrices in bf16: the largest
        dict(_ORTHO, name="large_bf16", dtype="bf16", sizes="4096x4096,8192x4096"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Half of the users take a multiple of 64, the others any size."""
    v = _log_int(rng, lo, hi)
    return min(hi, max(64, 64 * int(round(v / 64)))) if rng.random() < 0.5 else v


def draw(rng):
    xent_most, ortho_most = (max(_flops(c) for c in listed() if c["op"] == op) for op in ("xent", "ortho"))
    while True:
        if rng.random() < 0.5:
            c = dict(_XENT, dtype=rng.choice(["f32", "bf16"]), grads=rng.random() < 0.7, n=_log_int(rng, 1, 8192), H=_size(rng, 32, 4096),
                     C=_size(rng, 100, 128000), ignored=rng.choice([0.0, 0.0, 0.25]), weights=rng.random() < 0.3)
            c["masked"] = rng.choice([0, 0, rng.randint(1, 60)])
            # (fp32 takes the matrix pipe six times as long)
            if _flops(c) * (6 if c["dtype"] == "f32" else 1) <= xent_most:
                return c
        else:
            sizes = [(_size(rng, 16, 4096), _size(rng, 16, 8192)) for _ in range(rng.choice([1, 2, 4, 8]))]
            sizes = [s if rng.random() < 0.5 else s[::-1] for s in sizes]
            c = dict(_ORTHO, dtype=rng.choice(["f32", "bf16"]), sizes=",".join("%dx%d" % s for s in sizes), steps=rng.choice([5, 5, 6]))
            c["update"] = c["dtype"] == "f32" and rng.random() < 0.5
            if _flops(c) * (2 if c["dtype"] == "f32" else 1) <= ortho_most:
                return c


# --------------------------------------------------------------------------- what a program has in hand
def _dtype(case):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[case["dtype"]]


def _sizes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["sizes"].split(",")]


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device="cuda"), lambda *shape: torch.rand(*shape, generator=g, device="cuda")


def _inputs(case, seed):
    normal, uniform = _random(seed)
    t = _dtype(case)
    if case["op"] == "xent":
        n, H, C, used = case["n"], case["H"], case["C"], case["C"] - case["masked"]
        W = normal(C, H) / math.sqrt(H)
        labels = torch.floor(used ** uniform(n)).clamp_(max=used) - 1  # frequent words first, as vocabularies are ordered
        # states of a model that has learned something: they lean to their label's row, some much
        X = normal(n, H).mul_(1.5).add_(W[labels.long()] * (12 * uniform(n, 1)))
        b = 0.5 * normal(C)
        if case["masked"]:
            b[used:] = -math.inf
        if case["ignored"]:
            labels = torch.where(uniform(n) < case["ignored"], torch.full_like(labels, -1.0), labels)
        counted = 1.0 / n
        return dict(X=X.to(t), W=W.to(t), b=b, labels=labels, scale=counted, dloss=0.25 + uniform(n) if case["weights"] else None)
    G, M, W = [], [], []
    for rows, cols in _sizes(case):
        # a gradient is a sum over few strong directions and much noise
        r = max(1, min(rows, cols) // 8)
        g = normal(rows, r) @ normal(r, cols) / math.sqrt(r) + 0.3 * normal(rows, cols)
        G.append((1e-3 * g).to(t))
        M.append(2e-3 * normal(rows, cols) if case["update"] else None)
        W.append(normal(rows, cols) / math.sqrt(cols) if case["update"] else None)
    return dict(G=G, M=M, W=W)


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    from cavs_amd import hip

    s["hip"] = hip
    s["type"] = {"f32": hip.F32, "bf16": hip.BF16}[case["dtype"]]
    if case["op"] == "xent":
        n, H, C = case["n"], case["H"], case["C"]
        need = hip.lib().cavs_vocab_xent_workspace(s["type"], n, H, C, int(case["grads"]))
        out = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")  # noqa: E731
        s["loss"], s["lse"] = out(n), out(n)
        if case["grads"]:
            s["dX"], s["dW"], s["db"] = torch.empty_like(s["X"]), torch.empty_like(s["W"]), out(C)
    else:
        s["O"] = [torch.empty_like(g) for g in s["G"]]
        if case["update"]:
            s["M1"], s["W1"] = [torch.empty_like(m) for m in s["M"]], [torch.empty_like(w) for w in s["W"]]
        s["jobs"] = (hip.OrthoDesc * len(s["G"]))()
        for i, (rows, cols) in enumerate(_sizes(case)):
            m, w = (hip.ptr(s[k][i]) if case["update"] else None for k in ("M1", "W1"))
            s["jobs"][i] = hip.OrthoDesc(rows, cols, hip.ptr(s["G"][i]), cols, m, cols, w, cols, hip.ptr(s["O"][i]), cols)
        s["options"] = hip.OrthoOptions(case["steps"], 1, *_NS, _EPS, _MU, _LR, _DECAY)
        need = hip.lib().cavs_ortho_update_workspace(s["type"], len(s["G"]), s["jobs"])
    s["need"], s["workspace"] = need, torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    if s["case"]["op"] == "xent":
        return _run_xent(s) if own else _plain_xent(s)
    return _run_ortho(s) if own else _plain_ortho(s)


def _run_xent(s):
    hip, c = s["hip"], s["case"]
    P, n, H, C = hip.ptr, c["n"], c["H"], c["C"]
    st = torch.cuda.current_stream().cuda_stream
    if not c["grads"]:
        hip.call("cavs_vocab_xent_fwd", s["type"], P(s["X"]), H, P(s["W"]), H, P(s["b"]), P(s["labels"]), P(s["loss"]), P(s["lse"]), n, H, C,
                 P(s["workspace"]), s["need"], st)
        return {"loss": s["loss"], "lse": s["lse"]}
    hip.call("cavs_vocab_xent", s["type"], P(s["X"]), H, P(s["W"]), H, P(s["b"]), P(s["labels"]), P(s["dloss"]), s["scale"], P(s["loss"]),
             P(s["lse"]), P(s["dX"]), H, P(s["dW"]), H, P(s["db"]), n, H, C, P(s["workspace"]), s["need"], st)
    return {"loss": s["loss"], "lse": s["lse"], "dX": s["dX"], "dW": s["dW"], "db": s["db"]}


def _run_ortho(s):
    hip = s["hip"]
    if s["case"]["update"]:  # (the update is in place: a pass works on copies, so that it can be made again)
        torch._foreach_copy_(s["M1"] + s["W1"], s["M"] + s["W"])
    hip.call("cavs_ortho_update", s["type"], len(s["G"]), s["jobs"], s["options"], hip.ptr(s["workspace"]), s["need"],
             torch.cuda.current_stream().cuda_stream)
    return {"O": s["O"], "M": s["M1"], "W": s["W1"]} if s["case"]["update"] else {"O": s["O"]}


def _plain_xent(s):
    X, W, b, labels = s["X"].float(), s["W"].float(), s["b"], s["labels"]
    has = (labels >= 0) & (labels < W.shape[0])
    at = torch.where(has, labels, torch.zeros_like(labels)).long()[:, None]
    z = X @ W.t()
    z += b
    top = z.max(1, keepdim=True).values
    label = z.gather(1, at)
    z -= top
    z.exp_()
    total = z.sum(1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(has, (lse - label)[:, 0], torch.zeros_like(labels))
    out = {"loss": loss, "lse": lse[:, 0]}
    if s["case"]["grads"]:
        weight = has.float() * s["scale"] if s["dloss"] is None else has.float() * s["scale"] * s["dloss"]
        z *= 1.0 / total
        z.scatter_add_(1, at, torch.full_like(label, -1.0))
        z *= weight[:, None]
        out.update(dX=(z @ W).to(s["X"].dtype), dW=(z.t() @ X).to(s["W"].dtype), db=z.sum(0))
    return out


def _plain_ortho(s):
    c = s["case"]
    a, b, cc = _NS
    O, M1, W1 = [], [], []
    for G, M, W in zip(s["G"], s["M"], s["W"]):
        g = G.float()
        rows, cols = g.shape
        if c["update"]:
            M1.append(_MU * M + g)
            g = g + _MU * M1[-1]
        x = g.t() if rows > cols else g
        x = x / (x.square().sum().sqrt() + _EPS)
        for _ in range(c["steps"]):
            A = x @ x.t()
            x = a * x + (b * A + cc * (A @ A)) @ x
        x = x.t() if rows > cols else x
        if c["update"]:
            W1.append((1 - _LR * _DECAY) * W - _LR * math.sqrt(max(1.0, rows / cols)) * x)
        O.append(x.to(G.dtype).contiguous())
    return {"O": O, "M": M1, "W": W1} if c["update"] else {"O": O}


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    d = _inputs(case, seed)
    return _exact_xent(case, d) if case["op"] == "xent" else _exact_ortho(case, d)


def _exact_xent(case, d):
    """Rows a stretch at a time: p = exp(z - lse), d X = w (p W - W[label]), d W and d b from the same two terms."""
    n, H, C = case["n"], case["H"], case["C"]
    W, b = d["W"].double(), d["b"].double()
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    loss, lse, dX, dW, db = new(n), new(n), new(n, H), new(C, H) if case["grads"] else None, new(C)
    step = max(1, (1 << 28) // C)
    for r in range(0, n, step):
        x, lab = d["X"][r:r + step].double(), d["labels"][r:r + step].long()
        z = torch.addmm(b, x, W.t())
        on = (lab >= 0).double()
        at = lab.clamp(min=0)
        lse[r:r + step] = torch.logsumexp(z, 1)
        loss[r:r + step] = on * (lse[r:r + step] - z[torch.arange(len(lab), device="cuda"), at])
        if not case["grads"]:
            continue
        w = on * case_scale(d) * (1.0 if d["dloss"] is None else d["dloss"][r:r + step].double())
        p = torch.exp_(z.sub_(lse[r:r + step, None])).mul_(w[:, None])
        dX[r:r + step] = torch.mm(p, W).sub_(W[at] * w[:, None])
        dW += torch.mm(p.t(), x)
        dW.index_add_(0, at, x * -w[:, None])
        db += p.sum(0)
        db.index_add_(0, at, -w)
    out = {"loss": loss, "lse": lse}
    if case["grads"]:
        out.update(dX=dX, dW=dW, db=db)
    return out


def case_scale(d):
    return float(torch.tensor(d["scale"], dtype=torch.float32))  # (an argument of the call: a float)


def _exact_ortho(case, d):
    """Every factor is a polynomial of S = X0 X0^T, they commute: X = Y X0 with Y <- (a + b A + c A^2) Y, A = Y S Y."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    a, b, c, eps, mu, lr, decay = (f32(v) for v in (*_NS, _EPS, _MU, _LR, _DECAY))
    O, M1, W1 = [], [], []
    for G, M, W in zip(d["G"], d["M"], d["W"]):
        u = G.double()
        rows, cols = u.shape
        if case["update"]:
            M1.append(mu * M.double() + u)
            u = u + mu * M1[-1]
        flat = rows <= cols
        x0 = u / (torch.linalg.vector_norm(u) + eps)
        S = x0 @ x0.t() if flat else x0.t() @ x0
        one = torch.eye(len(S), dtype=torch.float64, device="cuda")
        Y = one
        for _ in range(case["steps"]):
            A = Y @ S @ Y
            A = 0.5 * (A + A.t())
            Y = (a * one + b * A + c * (A @ A)) @ Y
            Y = 0.5 * (Y + Y.t())
        x = Y @ x0 if flat else x0 @ Y
        if case["update"]:
            W1.append((1 - lr * decay) * W.double() - lr * math.sqrt(max(1.0, rows / cols)) * x)
        O.append(x)
    return {"O": O, "M": M1, "W": W1} if case["update"] else {"O": O}


# --------------------------------------------------------------------------- what a pass cannot do without
def _flops(case):
    if case["op"] == "xent":  # the logits; their gradients' two products
        return (6.0 if case["grads"] else 2.0) * case["n"] * case["H"] * case["C"]
    total = 0.0
    for s in _sizes(case):
        m, n = min(s), max(s)  # X X^T and A A are symmetric: half of each
        total += case["steps"] * (3.0 * m * m * n + 1.0 * m * m * m)
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "xent":
        n, H, C = case["n"], case["H"], case["C"]
        operands = size * (n * H + C * H)
        b = operands + 4 * C + 4 * n + 8 * n + (4 * n if case["weights"] else 0)
        if case["grads"]:
            b += operands + 4 * C
    else:
        b = sum(m * n * (2 * size + (16 if case["update"] else 0)) for m, n in _sizes(case))
    return {"bytes": float(b), "flops": _flops(case)}
