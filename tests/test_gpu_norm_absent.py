"""Weights of a norm that is not there (cavs_norm_residual_*): a descriptor may hold them, and neither pass reads them."""
import pytest

from test_gpu_norm_residual import Case, torch


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("post,pre", [("none", "none"), ("rms", "none"), ("layer", "none"), ("none", "rms"), ("none", "layer")])
@pytest.mark.parametrize("n,w", [(29, 304), (3, 5), (2, 9000)])
def test_absent_norms_have_no_weights(type_, post, pre, n, w):
    c = Case(type_, n, w, post, pre, "column")
    for k, kind in (("post", post), ("pre", pre)):
        if kind == "none":
            setattr(c, k + "_w", 3.0 * torch.randn(w, device="cuda")), setattr(c, k + "_b", 5.0 * torch.randn(w, device="cuda"))
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_nothing_comes_through_a_norm_without_dx(type_):
    """whatever its weights are"""
    c = Case(type_, 40, 200, "rms", "layer", "column")
    c.pre_w[7], c.pre_w[8] = float("inf"), float("nan")
    want, err = c.backward(dx=False)
    c.hold(c.run_backward(c.names(dx=False), dx=False), want, err)
