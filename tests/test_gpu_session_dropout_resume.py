"""A training run with dropout goes on from its checkpoint with the masks it would have had: parameters and the number of steps are all of a session's state"""
import ctypes as C

import numpy as np
import pytest

from cavs_amd import session
from test_gpu_session_block import _block_params
from test_gpu_session_head_optimizer import _gpu, _open, _params  # noqa: F401
from test_oracle_models import small_workload


def test_null_sessions():
    n = C.c_ulonglong()
    assert session.lib().cavs_session_get_dropout_steps(None, C.byref(n)) < 0 and session.lib().cavs_session_set_dropout_steps(None, 3) < 0


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm"])
@pytest.mark.parametrize("more", [dict(), dict(block=24), dict(plan_cache=2, graph_replay=True), dict(vocab_head=True, block=24)])
def test_goes_on_from_a_checkpoint(_gpu, model, more):
    import torch

    w = small_workload(model, 13, H=32, C=40)
    block = _block_params(6, 32, 24) if "block" in more else {}
    x, labels = torch.from_numpy(w["x"]).cuda(), torch.from_numpy(np.asarray(w["labels"], np.float32)).cuda()

    def opened():
        s = _open(w, dropout=0.4, dropout_seed=9, **more)
        s.set_params(block)
        return s

    def state(s):
        return dict(_params(s, w), **{k: s.param(k, v.shape) for k, v in block.items()})

    def run(s, steps):
        losses = []
        for _ in range(steps):
            s.step(w["graph"], x, labels, backward=True, lr=0.05)
            losses.append(s.fetch("loss").copy())
        return losses

    a = opened()
    assert a.dropout_steps == 0
    a.step(w["graph"], x, labels, backward=False)
    assert a.dropout_steps == 0
    run(a, 3)
    saved, steps = state(a), a.dropout_steps
    assert steps == 3
    want, end = run(a, 5), state(a)
    b = opened()
    b.set_params(saved)
    b.dropout_steps = steps
    got = run(b, 5)
    assert np.array_equal(got, want) and b.dropout_steps == 8
    final = state(b)
    assert all(np.array_equal(final[k], end[k]) for k in end)
    # other steps, other masks: far ones too
    b.set_params(saved)
    b.dropout_steps = (1 << 40) + steps
    assert not np.array_equal(run(b, 1)[0], want[0]) and b.dropout_steps == (1 << 40) + steps + 1


@pytest.mark.gpu
def test_sessions_without_dropout_have_no_steps(_gpu):
    s = _open(small_workload("treelstm", 9, H=32, C=40), block=8)
    for go in (lambda: s.dropout_steps, lambda: setattr(s, "dropout_steps", 1)):
        with pytest.raises(RuntimeError, match="drops nothing"):
            go()
