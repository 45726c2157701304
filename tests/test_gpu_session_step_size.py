"""The size of the session's orthogonalised updates goes by what a matrix does, not by how it is stored."""
import math

import numpy as np
import pytest

from test_gpu_session_head_optimizer import _blocks, _gpu, _open, _orthogonal, _params, _view  # noqa: F401
from test_oracle_models import small_workload
from tolerance import close


@pytest.mark.gpu
@pytest.mark.parametrize("E,H", [(10, 32), (40, 12), (96, 50), (33, 128)])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_a_step_is_sized_by_outputs_over_inputs(_gpu, E, H, decay):
    """sqrt(max(1, outputs / inputs)): a block of "W" takes a vertex's E inputs to H outputs (x W), one of "U" H to H, whichever way they are stored."""
    w = small_workload("treelstm", 17, H=H, E=E, C=5)
    print(f"[case] N={w['N']} E={E} H={H}", flush=True)
    lr, mu = 0.02, float(np.float32(0.95))
    s = _open(w, optimizer="ortho", ortho_decay=decay)
    before = _params(s, w)
    s.step(w["graph"], w["x"], w["labels"], backward=True, lr=lr)
    grads, after = s.grads(), _params(s, w)
    s.close()
    x, rows = np.asarray(before["Emb"]), np.asarray(before["W"])
    assert (x @ rows).shape[1] == 4 * H and rows.shape[0] == E  # what the factor is about: E in, H out a gate
    lr, decay = float(np.float32(lr)), float(np.float32(decay))
    for name, size in (("W", math.sqrt(max(1.0, H / E))), ("U", 1.0)):
        want, G = np.array(before[name], np.float64), np.array(grads["d" + name], np.float64)
        for b in _blocks("treelstm", E, H)[name]:
            g = _view(G, b)
            W = _view(want, b)
            W[:] = (1 - lr * decay) * W - lr * size * _orthogonal(g + mu * g)  # (the first step: the momentum is the gradient)
        close(after[name], want, name, scaled=False)
