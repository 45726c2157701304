"""What the session's head without logits counts."""
import pytest

from test_gpu_session_head_optimizer import _gpu, _open  # noqa: F401
from test_oracle_models import small_workload


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["treelstm", "lstm"])
def test_the_heads_products_are_counted_alike(_gpu, model):
    """Three products of N, C and H a training step and one a forward pass: what the head is asked for, with logits or without"""
    w = small_workload(model, 3, H=32, C=40)
    flops = {}
    for vocab in (False, True):
        s = _open(w, vocab_head=vocab)
        for backward in (False, True):
            s.step(w["graph"], w["x"], w["labels"], backward=backward)
            s.sync()
            flops[vocab, backward] = s.counter("gemm_flops")
        s.close()
    for backward in (False, True):
        assert flops[True, backward] == flops[False, backward], flops
