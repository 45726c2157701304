"""Norms of values near the type's largest (cavs_norm_residual_*): finite rows have finite results, with the bounds of any other row."""
import pytest

from test_gpu_norm_residual import Case, torch


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("w", [3, 9, 300, 2500])
def test_values_of_the_largest_size(type_, kind, w):
    """the largest value on one side of 0 and its negative on the other, few against many: a difference from the mean may be twice the largest value"""
    c = Case(type_, 6, w, kind, kind, "none", residual=False, scale=1.0, bias=False)
    most = torch.finfo(c.t).max
    for v in (c.y, c.s):
        v[:3], v[0, :], v[1, :], v[2, 1::2], v[2, ::2] = 0.0, -most, most, -most, most
        v[0, 0], v[1, w // 2] = most, -most
        v[3, :], v[3, w - 1] = 0.0, -most
    names = [k for k in c.names() if not k.endswith("_b")]
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(names), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("rms", "rms"), ("rms", "none")])
@pytest.mark.parametrize("w", [7, 300, 2048])
def test_gradients_whose_products_are_beyond_a_float(type_, post, pre, w):
    """values of 10^25 under gradients of 10^18: their products' sum is part of a row's, their gradient is a float"""
    c = Case(type_, 11, w, post, pre, "column", size=1e25)
    c.ds.mul_(1e20), c.dx.mul_(1e20)
    names = [k for k in c.names() if not k.endswith("_b")]
    if post == "none":
        names.remove("dgate")  # (10^25 times 10^18 is no float)
    c.hold(c.run_backward(names), *c.backward())


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [8192.0, -8000.0])
def test_means_thousands_of_deviations_from_zero(offset):
    """as far as sums of values and of their squares in 64 bits give a deviation a float's rounding"""
    c = Case("f32", 40, 777, "layer", "layer", "none", residual=False, offset=offset, scale=1.0)
    c.hold(c.run_forward(), *c.forward())
    c.hold(c.run_backward(c.names()), *c.backward())
