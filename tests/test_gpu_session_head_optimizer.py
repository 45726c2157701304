"""The session's head without logits (vocab_head) and its orthogonalised updates (optimizer="ortho"), alone and together, against the oracle
in double precision and against the definition of the update in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

from cavs_amd import hip, session
from test_oracle_models import small_workload
from tolerance import close

NS = (3.4445, -4.7750, 2.0315)


# ------------------------------------------------------------------ refusals: the configuration is looked at before the device
@pytest.mark.parametrize("field,value", [("vocab_head", 2), ("vocab_head", -1), ("optimizer", 2), ("optimizer", -1), ("ortho_lr", -1.0),
                                         ("ortho_momentum", 1.0), ("ortho_decay", -0.5), ("ortho_lr", float("nan"))])
def test_refusals(field, value):
    cfg = session._Config(model=0, loss=0, opt=2, V=10, E=4, H=8, C=20)
    setattr(cfg, field, value)
    h = C.c_void_p()
    assert session.lib().cavs_session_create(C.byref(cfg), C.byref(h)) == -1 and not h
    assert session.lib().cavs_session_error()


def test_a_head_without_logits_goes_with_the_softmax_loss():
    cfg = session._Config(model=2, loss=1, opt=2, H=8, vocab_head=1)
    h = C.c_void_p()
    assert session.lib().cavs_session_create(C.byref(cfg), C.byref(h)) == -1 and not h


# ------------------------------------------------------------------ on the device
def _names(model, use_bias=False):
    return {"treelstm": ("Emb", "W", "U", "Bv"), "lstm": ("Emb", "W", "Bv"), "treefc": ("W", "Bv") if use_bias else ("W",)}[model] + ("Wfc", "bfc")


def _open(w, **kw):
    extra = dict(act=1, use_bias=True, use_x=True) if w["model"] == "treefc" else {}
    s = session.Session(w["model"], H=w["H"], E=w["E"], V=w["V"], C_=w["C"], **extra, **kw)
    s.set_params({k: w["params"][k] for k in _names(w["model"], True)})
    return s


def _params(s, w):
    return {k: s.param(k, np.asarray(w["params"][k]).shape) for k in _names(w["model"], True)}


def _blocks(model, E, H):
    """(parameter, [(first element, rows, columns, row stride)])"""
    cols = lambda at, n, rows: [(at + k * H, rows, H, n * H) for k in range(n)]  # noqa: E731
    if model == "treelstm":
        return {"W": cols(0, 4, E), "U": cols(0, 3, H) + cols(3 * H * H, 1, H)}
    if model == "lstm":
        return {"W": cols(0, 4, H) + cols(4 * H * H, 4, H)}
    return {"W": cols(0, 1, H) + cols(H * H, 1, H)}


def _view(a, block):
    at, rows, n, ld = block
    return np.lib.stride_tricks.as_strided(a.reshape(-1)[at:], (rows, n), (ld * a.itemsize, a.itemsize))


def _orthogonal(u, steps=5):
    a, b, c = (float(np.float32(v)) for v in NS)
    x = u / (np.sqrt((u * u).sum()) + float(np.float32(1e-7)))
    flat = x.shape[0] <= x.shape[1]
    x = x if flat else x.T
    for _ in range(steps):
        A = x @ x.T
        x = a * x + (b * A + c * (A @ A)) @ x
    return x if flat else x.T


def _update(model, E, H, w, g, m, lr, mu=0.95, decay=0.0):
    """(weights, momentum) after one update, in 64 bits"""
    mu, lr, decay = (float(np.float32(v)) for v in (mu, lr, decay))
    w, m = {k: np.array(v, np.float64) for k, v in w.items()}, {k: np.array(v, np.float64) for k, v in m.items()}
    for name, blocks in _blocks(model, E, H).items():
        G = np.array(g["d" + name], np.float64)
        for b in blocks:
            W, M, g_ = _view(w[name], b), _view(m[name], b), _view(G, b)
            M[:] = mu * M + g_
            u = g_ + mu * M
            W[:] = (1 - lr * decay) * W - lr * math.sqrt(max(1.0, b[1] / b[2])) * _orthogonal(u)
    return w, m


@pytest.fixture
def _gpu():
    import torch

    assert torch.cuda.is_available(), "these tests need the MI355X"
    hip.call("cavs_init", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm", "treefc"])
@pytest.mark.parametrize("H,classes", [(12, 5), (12, 9), (32, 23), (40, 700), (64, 3000)])
@pytest.mark.parametrize("batching", [True, False])
def test_head_without_logits(_gpu, oracle, model, H, classes, batching):
    w = small_workload(model, 31 + H, H=H, C=classes)
    print(f"[case] model={model} N={w['N']} H={H} C={classes} batching={batching}", flush=True)
    extra = dict(act=1, use_bias=True, use_x=True) if model == "treefc" else {}
    want = oracle.model_step(model, w["graph"], w["x"], w["labels"], w["params"], H=w["H"], E=w["E"], V=w["V"], Cc=w["C"], batching=batching, precise=True, **extra)
    s = _open(w, vocab_head=True, opt=session.OPT_BATCHING if batching else 0)
    s.step(w["graph"], w["x"], w["labels"], backward=False)
    close(s.fetch("loss"), want["loss"], "loss, forward", scaled=False)
    s.step(w["graph"], w["x"], w["labels"], backward=True)
    close(s.fetch("loss"), want["loss"], "loss", scaled=False)
    close(s.fetch("dgraph_out"), want["dgraph_out"], "dgraph_out", scaled=False)
    grads = s.grads()
    for k, v in want["grads"].items():
        if k in grads:
            close(grads[k], v, k, scaled=False)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm"])
def test_vertices_without_a_label(_gpu, oracle, model):
    """A vertex labelled -1 has loss 0 and sends nothing: the gradients are those of the others, whose sum the oracle gives as the difference
    of two batches' that differ in those labels alone (it is linear in the d logits of each)."""
    w = small_workload(model, 5, H=32, C=40)
    labels = np.array(w["labels"])
    gone = np.arange(w["N"]) % 3 == 1
    labels[gone] = -1
    s = _open(w, vocab_head=True)
    s.step(w["graph"], w["x"], labels, backward=True)
    loss, go, dgo = s.fetch("loss"), s.fetch("graph_out").astype(np.float64), s.fetch("dgraph_out")
    grads = s.grads()
    s.close()
    z = go @ np.array(w["params"]["Wfc"], np.float64).T + w["params"]["bfc"]
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    at = np.maximum(labels, 0).astype(int)
    d = p.copy()
    d[np.arange(w["N"]), at] -= 1
    d[gone] = 0
    d /= w["N"]
    close(loss, np.where(gone, 0.0, -np.log(p[np.arange(w["N"]), at])), "loss", scaled=False)
    close(dgo, d @ np.array(w["params"]["Wfc"], np.float64), "dgraph_out", scaled=False)
    close(grads["dWfc"], d.T @ go, "dWfc", scaled=False)
    close(grads["dbfc"], d.sum(0), "dbfc", scaled=False)
    assert (loss[gone] == 0).all() and (dgo[gone] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm", "treefc"])
@pytest.mark.parametrize("H", [12, 32, 50, 64])
@pytest.mark.parametrize("kw", [dict(), dict(ortho_lr=0.05, ortho_momentum=0.8, ortho_decay=0.1), dict(ortho_momentum=-1.0)])
def test_updates(_gpu, model, H, kw):
    """Two updates, each from the gradients the session itself reports; everything that is no matrix moves by SGD."""
    w = small_workload(model, 7 + H, H=H, C=5)
    print(f"[case] model={model} N={w['N']} H={H} {kw}", flush=True)
    s = _open(w, optimizer="ortho", **kw)
    lr, mu = 0.02, max(kw.get("ortho_momentum", 0.95), 0.0)
    names = list(_blocks(model, w["E"], H))
    want_m = {k: np.zeros(np.asarray(w["params"][k]).shape) for k in names}
    for _ in range(2):
        before = _params(s, w)
        s.step(w["graph"], w["x"], w["labels"], backward=True, lr=lr)
        grads = s.grads()
        want_w, want_m = _update(model, w["E"], H, {k: before[k] for k in names}, grads, want_m, kw.get("ortho_lr") or lr, mu, kw.get("ortho_decay", 0.0))
        after = _params(s, w)
        for k in after:
            if k in names:
                # (X's entries are below 1; its error, 1e-5 of its norm at most, comes in times lr: what is left is the weights' rounding)
                close(after[k], want_w[k], k, scaled=False)
                assert np.abs(after[k] - before[k]).max() > 1e-4
                if mu > 0:
                    close(s.param(k + ".momentum", after[k].shape), want_m[k], k + ".momentum", scaled=False)
            else:
                close(after[k], before[k] - np.float32(lr) * grads["d" + k].reshape(before[k].shape), k, scaled=False)
    with pytest.raises(hip.CavsError, match="no gradient"):
        s.grad("W.momentum", want_m["W"].shape)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("model,H", [("treelstm", 50), ("lstm", 64)])
def test_a_training_run_goes_on_from_its_checkpoint(_gpu, model, H):
    """Head and updates together: three steps, and one step, all state read out, a new session, two steps, give the same bits; so do
    kept plans and recorded launches."""
    import torch

    w = small_workload(model, 77, H=H, C=50, B=8)
    kw = dict(vocab_head=True, optimizer="ortho", ortho_decay=0.01)
    x, labels = torch.from_numpy(w["x"]).cuda(), torch.from_numpy(w["labels"]).cuda()
    step = lambda s: s.step(w["graph"], x, labels, backward=True, lr=0.02)  # noqa: E731
    a = _open(w, **kw)
    for _ in range(3):
        step(a)
    want, loss = _params(a, w), a.fetch("loss")
    b = _open(w, **kw)
    step(b)
    state = _params(b, w)
    state.update({k + ".momentum": b.param(k + ".momentum", state[k].shape) for k in _blocks(model, w["E"], H)})
    c = _open(w, **kw)
    c.set_params(state)
    step(c)
    step(c)
    got = _params(c, w)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
    np.testing.assert_array_equal(c.fetch("loss"), loss)
    for more in (dict(plan_cache=4), dict(plan_cache=4, graph_replay=True), dict(schedule="device")):
        d = _open(w, **kw, **more)
        for _ in range(3):
            step(d)
        got = _params(d, w)
        for k in want:
            np.testing.assert_array_equal(got[k], want[k], err_msg=f"{k} {more}")
        for _ in range(4):
            step(d)
        a2 = _params(d, w)
        d.close()
        e = _open(w, **kw)
        for _ in range(7):
            step(e)
        got = _params(e, w)
        for k in got:
            np.testing.assert_array_equal(a2[k], got[k], err_msg=f"{k} {more}, seven steps")
        e.close()
    for s in (a, b, c):
        s.close()


@pytest.mark.gpu
def test_sessions_side_by_side(_gpu):
    """Two sessions on streams of their own, stepping in turn without waiting for each other, each with its own state and workspaces."""
    w = [small_workload("lstm", 3, H=32, C=30), small_workload("treelstm", 4, H=64, C=90)]
    kw = dict(vocab_head=True, optimizer="ortho")
    alone = []
    for v in w:
        s = _open(v, **kw)
        for _ in range(4):
            s.step(v["graph"], v["x"], v["labels"], backward=True, lr=0.02)
        alone.append(_params(s, v))
        s.close()
    both = [_open(v, **kw) for v in w]
    for _ in range(4):
        for s, v in zip(both, w):
            s.step(v["graph"], v["x"], v["labels"], backward=True, lr=0.02)
    for s, v, want in zip(both, w, alone):
        got = _params(s, v)
        for k in want:
            np.testing.assert_array_equal(got[k], want[k], err_msg=k)
        s.close()
