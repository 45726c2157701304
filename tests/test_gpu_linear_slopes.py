"""Slopes of saturated units (cavs_linear_bwd): far from 0 the slopes of sigmoid and tanh are small numbers with all their digits.

One row with dY = 1 and no other wanted result than db makes db the slope itself, in fp32 for either type.  In units u = 2^-24, relative to the slope, below which 2^-122
takes in what is no longer a normal float:
  fp32 sigmoid  g = 1 / (1 + e^|z|): 2 u of e, u of the sum, 5 u of the division; 1 - g, at least 1/2, 9 u; the product u: 20 u
  fp32 tanh     4 e / (1 + e)^2, e = e^-2|z|: 2 u of e, 8 u of the quotient, twice; two products: 24 u
  bf16          e from the instruction of x log2 e: 2 u |x| of the argument's rounding and of the constant's, 2 u; its reciprocal 2 u: (4 |z| + 16) u, tanh's x is
                2 |z|: (12 |z| + 16) u
"""
import pytest

from cavs_amd import hip

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (hip.F32, torch.float32), "bf16": (hip.BF16, torch.bfloat16)}


def _slopes(type_, act, z):
    code, t = TYPES[type_]
    z = z.to(t).cuda()
    N, K, P = z.numel(), 8, hip.ptr
    dY, W, db = torch.ones(N, dtype=t, device="cuda"), torch.zeros(N, K, dtype=t, device="cuda"), torch.empty(N, device="cuda")
    need = hip.lib().cavs_linear_workspace(code, 1, K, N, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    hip.call("cavs_linear_bwd", code, None, K, P(W), K, P(z), N, hip.ACT[act], None, P(dY), N, None, 0, None, 0, P(db), 1, K, N, P(ws), need,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return z.double(), db.double()


def _far():
    return torch.cat([torch.linspace(-100, 100, 4001), torch.linspace(-2, 2, 801), torch.tensor([0.0, -0.0, 17.0, -17.0])])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_sigmoid(type_):
    z, got = _slopes(type_, "sigmoid", _far())
    want = torch.sigmoid(z) * torch.sigmoid(-z)
    bound = 20 * U if type_ == "f32" else (4 * z.abs() + 16) * U
    assert bool(((got - want).abs() <= bound * want + 2.0 ** -122).all()), float(((got - want).abs() / want).max())



@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_tanh(type_):
    z, got = _slopes(type_, "tanh", _far())
    e = torch.exp(-2 * z.abs())
    want = 4 * e / (1 + e).square()
    bound = 24 * U if type_ == "f32" else (12 * z.abs() + 16) * U
    assert bool(((got - want).abs() <= bound * want + 2.0 ** -122).all()), float(((got - want).abs() / want).max())
