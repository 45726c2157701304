"""The bias's gradient alone (cavs_linear_bwd without dX and dW): of sizes whose plans differ with what is wanted, within the workspace that is asked for"""
import pytest

from test_gpu_linear import Case


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,K,N", [(1082, 105, 576), (2058, 833, 2816), (300, 1, 8), (1082, 104, 576), (1, 7, 8), (70, 13, 4096), (500, 9, 33)])
def test_alone(type_, n, K, N):
    c = Case(type_, n, K, N, "gelu", 0.1)
    c.hold(c.run(1, ["db"]), *c.backward())
