"""What flows on from vertices without a label under the head without logits."""
import numpy as np
import pytest

import textbook
from cavs_amd import session
from test_gpu_session_head_optimizer import _gpu, _open  # noqa: F401
from test_oracle_models import small_workload
from tolerance import close


@pytest.mark.gpu
@pytest.mark.parametrize("model,kw", [("treelstm", dict()), ("lstm", dict()), ("treefc", dict(act=1, use_bias=True, use_x=True))])
@pytest.mark.parametrize("batching", [True, False])
def test_what_flows_on_from_vertices_without_a_label(_gpu, monkeypatch, model, kw, batching):
    """All gradients, the recurrent weights' and the embedding's among them, against the 64-bit model whose loss leaves those vertices out"""
    import torch

    def head(GO, P, labels, loss, parents):
        rows = torch.nn.functional.cross_entropy(GO @ P["Wfc"].T + P["bfc"], torch.tensor(np.asarray(labels), dtype=torch.long), reduction="none", ignore_index=-1)
        return rows, rows.sum() / len(rows)

    monkeypatch.setattr(textbook, "_head", head)
    w = small_workload(model, 5, H=32, C=40)
    labels = np.array(w["labels"])
    labels[np.arange(w["N"]) % 3 == 1] = -1
    want = textbook.per_sample(model, w["graph"], w["x"], labels, w["params"], w["H"], **kw)
    s = _open(w, vocab_head=True, pairing="rowid", opt=session.OPT_BATCHING if batching else 0)
    s.step(w["graph"], w["x"], labels, backward=True)
    close(s.fetch("loss"), want["loss"], "loss", scaled=False)
    close(s.fetch("dgraph_out"), want["dgraph_out"], "dgraph_out", scaled=False)
    grads = s.grads()
    s.close()
    assert len(grads) >= 4
    for k, v in want["grads"].items():
        if k in grads:
            close(grads[k], v, k, scaled=False)
