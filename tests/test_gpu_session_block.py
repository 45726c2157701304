"""Sessions with a residual block between the vertices and the head, norm, two products, activation, dropouts and residual: losses and all gradients against the 64-bit
model under the same masks, training runs recorded and not."""
import ctypes as C

import numpy as np
import pytest

import philox
import textbook
from cavs_amd import session
from test_gpu_session_head_optimizer import _gpu, _open, _params  # noqa: F401
from test_oracle_models import small_workload
from tolerance import close

P, SEED = 0.2, 77


@pytest.mark.parametrize("kw", [dict(block=-1), dict(block=65537), dict(block=8, loss=1), dict(block=8, H=16416), dict(block=8, block_act=6), dict(block_act=-1)])
def test_refusals(kw):
    cfg = session._Config(**dict(dict(model=2, loss=0, opt=2, V=10, E=4, H=8, C=20), **kw))
    h = C.c_void_p()
    assert session.lib().cavs_session_create(C.byref(cfg), C.byref(h)) == -1 and not h
    assert "block" in session.lib().cavs_session_error().decode()


def test_fields_behind_the_older_struct_are_not_read():
    lib = session.lib()
    at = session._Config.block.offset
    for field in "block", "block_act":
        cfg = session._Config(model=0, loss=0, opt=2, V=10, E=4, H=8, C=20, device=-5, **{field: -1})
        h = C.c_void_p()
        assert lib.cavs_session_create_sized(C.byref(cfg), C.c_size_t(at), C.byref(h)) < 0 and not h
        assert "block" not in lib.cavs_session_error().decode()


def _block_params(seed, H, F):
    r = np.random.default_rng(seed)
    f = lambda s, *n: (s * r.standard_normal(n)).astype(np.float32)  # noqa: E731
    return dict(gnorm=1 + f(0.2, H), Wup=f(0.3, F, H), bup=f(0.2, F), Wdown=f(0.3, H, F), bdown=f(0.2, H))


def _head(monkeypatch, act, step):
    """step None: nothing is dropped"""
    import torch

    acts = dict(none=lambda z: z, relu=torch.relu, tanh=torch.tanh, sigmoid=torch.sigmoid, silu=lambda z: z * torch.sigmoid(z),
                gelu=lambda z: 0.5 * z * torch.erfc(-z / 2 ** 0.5))

    def drop(v, place):
        if step is None:
            return v
        return v * torch.tensor(philox.kept(*v.shape, P, SEED + (place << 32), step) * philox.factor(P), dtype=v.dtype)

    def head(GO, p, labels, loss, parents):
        x = GO / torch.sqrt((GO * GO).mean(1, keepdim=True) + 1e-6) * p["gnorm"]
        a = drop(acts[act](x @ p["Wup"].T + p["bup"]), 1)
        y = GO + drop(a @ p["Wdown"].T + p["bdown"], 2)
        rows = torch.nn.functional.cross_entropy(y @ p["Wfc"].T + p["bfc"], torch.tensor(np.asarray(labels), dtype=torch.long), reduction="none")
        return rows, rows.mean()

    monkeypatch.setattr(textbook, "_head", head)


def _losses(got, want):
    """The head with logits gives -log of a probability in fp32, which is 0 where the loss is above 150 log 2 = 103.97: half of the least float is 2^-150"""
    none = want > 104
    assert np.isinf(got[none]).all()
    close(got[~none], want[~none], "loss", scaled=False)


MODELS = {"treelstm": dict(), "lstm": dict(), "treefc": dict(act=1, use_bias=True, use_x=True)}


@pytest.mark.gpu
@pytest.mark.parametrize("model,H,F,classes,act,p,kw", [
    ("treelstm", 32, 64, 5, "gelu", P, {}), ("treelstm", 20, 50, 40, "silu", P, {}), ("lstm", 32, 128, 40, "relu", P, dict(vocab_head=True)),
    ("lstm", 20, 7, 5, "tanh", 0.0, {}), ("treefc", 32, 1, 40, "sigmoid", P, {}), ("treefc", 12, 300, 5, "none", 0.0, {}),
    ("lstm", 32, 64, 9000, "gelu", P, {}), ("treelstm", 20, 33, 40, "gelu", P, dict(schedule="device")), ("lstm", 64, 96, 40, "gelu", P, dict(opt=0))])
def test_against_the_model(_gpu, monkeypatch, model, H, F, classes, act, p, kw):
    w = small_workload(model, 5, H=H, C=classes)
    params = dict(w["params"], **_block_params(3, H, F))
    s = _open(w, pairing="rowid", dropout=p, dropout_seed=SEED, block=F, block_act=act, **kw)
    s.set_params({k: params[k] for k in ("gnorm", "Wup", "bup", "Wdown", "bdown")})
    args = (model, w["graph"], w["x"], w["labels"], params, w["H"])
    for step in range(2):
        _head(monkeypatch, act, None)
        s.step(w["graph"], w["x"], w["labels"], backward=False)  # (drops nothing, and counts for nothing)
        _losses(s.fetch("loss"), textbook.per_sample(*args, **MODELS[model])["loss"])
        _head(monkeypatch, act, step if p else None)
        want = textbook.per_sample(*args, **MODELS[model])
        s.step(w["graph"], w["x"], w["labels"], backward=True)
        _losses(s.fetch("loss"), want["loss"])
        close(s.fetch("graph_out"), want["graph_out"], "graph_out", scaled=False)
        close(s.fetch("dgraph_out"), want["dgraph_out"], "dgraph_out", scaled=False)
        grads = s.grads()
        assert {"dgnorm", "dWup", "dbup", "dWdown", "dbdown"} <= set(grads)
        for k, v in want["grads"].items():
            if k in grads:
                close(grads[k], v, k, scaled=False)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm"])
def test_recorded_steps(_gpu, model):
    import torch

    w = small_workload(model, 11, H=20, C=40)
    block = _block_params(4, 20, 50)
    x, labels = torch.tensor(np.asarray(w["x"], np.float32), device="cuda"), torch.tensor(np.asarray(w["labels"], np.float32), device="cuda")
    got = []
    for kw in (dict(plan_cache=2), dict(plan_cache=2, graph_replay=True)):
        s = _open(w, dropout=P, dropout_seed=SEED, block=50, **kw)
        s.set_params(block)
        run = []
        for _ in range(8):
            s.step(w["graph"], x, labels, backward=True, lr=0.05)
            run.append(s.fetch("loss").copy())
        got.append((run, _params(s, w), {k: s.param(k, v.shape) for k, v in block.items()}))
        if "graph_replay" in kw:
            assert s.counter("graph_replays") >= 4
        s.close()
    assert np.array_equal(got[0][0], got[1][0])
    for i in 1, 2:
        assert all(np.array_equal(got[0][i][k], got[1][i][k]) for k in got[0][i])
    assert all(not np.array_equal(got[0][2][k], block[k]) for k in block)  # (all of them are trained)


@pytest.mark.gpu
def test_batches_of_growing_sizes_in_one_session(_gpu, monkeypatch):
    """Buffers grow with the batch, and nothing of a larger one is left in a smaller"""
    H, F = 20, 50
    s = None
    for B in (2, 9, 3, 14):
        w = small_workload("treelstm", 5, B=B, H=H, C=40)
        w0 = small_workload("treelstm", 5, B=2, H=H, C=40)
        params = dict(w0["params"], **_block_params(3, H, F))
        if s is None:
            s = _open(w0, pairing="rowid", block=F)
            s.set_params({k: params[k] for k in ("gnorm", "Wup", "bup", "Wdown", "bdown")})
        _head(monkeypatch, "gelu", None)
        want = textbook.per_sample("treelstm", w["graph"], w["x"], w["labels"], params, H)
        s.step(w["graph"], w["x"], w["labels"], backward=True)
        close(s.fetch("loss"), want["loss"], "loss", scaled=False)
        close(s.fetch("dgraph_out"), want["dgraph_out"], "dgraph_out", scaled=False)
        grads = s.grads()
        for k, v in want["grads"].items():
            if k in grads:
                close(grads[k], v, k, scaled=False)
    s.close()
