"""cavs_vocab_xent* in fp32 with operands next to the largest float."""
import pytest

from test_gpu_vocab_xent import Case, _device  # noqa: F401

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["W", "X"])
@pytest.mark.parametrize("n,H,C", [(1, 96, 900), (20, 1030, 3000), (40, 96, 900), (100, 96, 900), (300, 130, 2000)])
def test_operands_next_to_the_largest_float(which, n, H, C):
    """fp32 values that bf16 would round to infinity, beside ones so small that their products are ordinary logits.  (Those are whole in bf16: parts below
    2^-126 would be lost.)"""
    c = Case(n + H, "f32", n, H, C)
    big, small = (c.W, c.X) if which == "W" else (c.X, c.W)
    g = torch.Generator(device="cuda").manual_seed(5)
    last = torch.finfo(torch.float32).max
    for k in (0, H // 2, H - 1):  # (of one sign: sums of them weighted with probabilities are floats too)
        u = torch.rand(big.shape[0], generator=g, device="cuda")
        big[:, k] = last * (1 - 2.0 ** -10 * (1 + 0.9 * u))  # (from last (1 - 2^-9) on bf16 rounds to infinity)
        small[:, k] = (2.0 ** -126 * (1 + 3 * torch.rand(small.shape[0], generator=g, device="cuda"))).bfloat16().float()
    assert big.isfinite().all() and big.bfloat16()[:, 0].isinf().all()
    o, (ws, need) = c.outputs(), c.workspace(0)
    c.call("cavs_vocab_xent_fwd", o, ws, need)
    c.check(o, ("loss", "lse"))
    o, (ws, need) = c.outputs(), c.workspace(1)
    c.call("cavs_vocab_xent", o, ws, need)
    # (rows of X add up in d W, before the scale: more than one of these are no float)
    c.check(o, ("loss", "lse", "dX", "dW", "db") if which == "W" or n == 1 else ("loss", "lse", "dX", "db"))
