"""Sessions that drop a share of what the vertices push before their head: losses and all gradients against the 64-bit model under the same mask, over steps,
heads, schedules and recorded steps."""
import ctypes as C

import numpy as np
import pytest

import philox
import textbook
from cavs_amd import session
from test_gpu_session_head_optimizer import _gpu, _open, _params  # noqa: F401
from test_oracle_models import small_workload
from tolerance import close

P, SEED = 0.3, 4000000007


@pytest.mark.parametrize("kw", [dict(dropout=1.0), dict(dropout=-0.1), dict(dropout=float("nan")), dict(dropout=0.5, loss=1)])
def test_refusals(kw):
    cfg = session._Config(**dict(dict(model=2, loss=0, opt=2, V=10, E=4, H=8, C=20), **kw))
    h = C.c_void_p()
    assert session.lib().cavs_session_create(C.byref(cfg), C.byref(h)) == -1 and not h
    assert "dropout" in session.lib().cavs_session_error().decode()


def _masked_head(monkeypatch, step, p=P, seed=SEED):
    import torch

    def head(GO, params, labels, loss, parents):
        n, w = GO.shape
        mask = torch.tensor(philox.kept(n, w, p, seed, step) * philox.factor(p), dtype=GO.dtype)
        rows = torch.nn.functional.cross_entropy(GO * mask @ params["Wfc"].T + params["bfc"], torch.tensor(np.asarray(labels), dtype=torch.long), reduction="none")
        return rows, rows.mean()

    monkeypatch.setattr(textbook, "_head", head)


MODELS = {"treelstm": dict(), "lstm": dict(), "treefc": dict(act=1, use_bias=True, use_x=True)}


@pytest.mark.gpu
@pytest.mark.parametrize("model,H,classes,kw", [("treelstm", 32, 5, {}), ("treelstm", 20, 40, {}), ("lstm", 32, 40, dict(vocab_head=True)), ("lstm", 20, 5, {}),
                                                ("treefc", 32, 40, {}), ("treefc", 12, 5, {}), ("lstm", 32, 9000, {}), ("treelstm", 20, 40, dict(schedule="device")),
                                                ("lstm", 64, 40, dict(opt=0)), ("treelstm", 32, 40, dict(vocab_head=True, tail_rows=-1))])
def test_against_the_model_under_the_same_mask(_gpu, monkeypatch, model, H, classes, kw):
    w = small_workload(model, 5, H=H, C=classes)
    s = _open(w, pairing="rowid", dropout=P, dropout_seed=SEED, **kw)
    for step in range(3):
        s.step(w["graph"], w["x"], w["labels"], backward=False)  # (drops nothing, and counts for nothing)
        monkeypatch.undo()
        plain = textbook.per_sample(model, w["graph"], w["x"], w["labels"], w["params"], w["H"], **MODELS[model])
        close(s.fetch("loss"), plain["loss"], "loss without backward", scaled=False)
        _masked_head(monkeypatch, step)
        want = textbook.per_sample(model, w["graph"], w["x"], w["labels"], w["params"], w["H"], **MODELS[model])
        s.step(w["graph"], w["x"], w["labels"], backward=True)
        close(s.fetch("loss"), want["loss"], "loss", scaled=False)
        close(s.fetch("dgraph_out"), want["dgraph_out"], "dgraph_out", scaled=False)
        grads = s.grads()
        assert len(grads) >= 3
        for k, v in want["grads"].items():
            if k in grads:
                close(grads[k], v, k, scaled=False)
    s.close()


@pytest.mark.gpu
def test_no_dropout_is_the_session_of_before(_gpu):
    w = small_workload("treelstm", 9, H=32, C=40)
    got = []
    for kw in ({}, dict(dropout=0.0, dropout_seed=SEED)):
        s = _open(w, **kw)
        for _ in range(3):
            s.step(w["graph"], w["x"], w["labels"], backward=True, lr=0.1)
        got.append(_params(s, w))
        s.close()
    assert all(np.array_equal(got[0][k], got[1][k]) for k in got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm"])
def test_recorded_steps_draw_anew(_gpu, model):
    """A session whose steps are one recorded graph trains as one that enqueues every launch, mask after mask"""
    import torch

    w = small_workload(model, 11, H=32, C=40)
    x, labels = torch.tensor(np.asarray(w["x"], np.float32), device="cuda"), torch.tensor(np.asarray(w["labels"], np.float32), device="cuda")
    got, losses = [], []
    for kw in (dict(plan_cache=2), dict(plan_cache=2, graph_replay=True)):
        s = _open(w, dropout=P, dropout_seed=SEED, **kw)
        losses.append([])
        for _ in range(8):
            s.step(w["graph"], x, labels, backward=True, lr=0.05)
            losses[-1].append(s.fetch("loss").copy())
        got.append(_params(s, w))
        if "graph_replay" in kw:
            assert s.counter("graph_replays") >= 4
        s.close()
    assert np.array_equal(losses[0], losses[1])
    assert all(np.array_equal(got[0][k], got[1][k]) for k in got[0])
