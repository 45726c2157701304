"""Slopes of saturated units (cavs_linear_bwd): far from 0 the slopes of sigmoid and tanh are small numbers with all their digits.

One row with dY = 1 and no other wanted result than db makes db the slope itself, in fp32 for either type.  In units u = 2^-24, relative to the slope, below which 2^-122
takes in what is no longer a normal float:
  fp32 sigmoid  g = 1 / (1 + e^|z|): 2 u of e, u of the sum, 5 u of the division; 1 - g, at least 1/2, 9 u; the product u: 20 u
  fp32 tanh     4 e / (1 + e)^2, e = e^-2|z|: 2 u of e, 8 u of the quotient, twice; two products: 24 u
  bf16          e from the instruction of x log2 e: 2 u |x| of the argument's rounding and of the constant's, 2 u; its reciprocal 2 u: (4 |z| + 16) u, tanh's x is
                2 |z|: (12 |z| + 16) u
silu and gelu, g (1 + z (1 - g)) and Phi + z phi, have a zero: relative to the sum of their terms' sizes, sigmoid's (and 16 u) for the first; for the second the bf16 form's
2^-19 and 2^-22 z^2, of fp32 the rounding of what goes into erfc and e^x, 2 z^2 u each, and 24 u
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


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_silu(type_):
    z, got = _slopes(type_, "silu", _far())
    g, size = torch.sigmoid(z), torch.sigmoid(z) * (1 + z.abs() * torch.sigmoid(-z))
    want = g * (1 + z * torch.sigmoid(-z))
    # (z (1 - g) of a g near 1: u of 1 times z, beside 1)
    bound = (36 + 2 * z.abs()) * U if type_ == "f32" else (8 * z.abs() + 32) * U
    assert bool(((got - want).abs() <= bound * size + 2.0 ** -115).all()), float(((got - want).abs() / size).max())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_gelu(type_):
    z, got = _slopes(type_, "gelu", _far())
    phi, pdf = 0.5 * torch.erfc(-z / 2 ** 0.5), torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    bound = (4 * z * z + 24) * U if type_ == "f32" else 2.0 ** -19 + 2.0 ** -22 * z * z
    size = phi + z.abs() * pdf
    assert bool(((got - (phi + z * pdf)).abs() <= bound * size + 2.0 ** -118).all()), float(((got - (phi + z * pdf)).abs() / size).max())
