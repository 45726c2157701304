"""bf16 products of operands as they lie whose rows are as far apart as that takes (2^22 elements, so that a tile's rows reach 2^31 bytes and its lines of k 2^29), and of
some a piece further apart, which are packed first"""
import pytest

from test_gpu_linear import Case, torch


@pytest.mark.gpu
@pytest.mark.parametrize("n,K,N,ld", [(300, 136, 264, 1 << 22), (300, 136, 264, (1 << 22) + 8), (129, 64, 128, 1 << 22), (4096, 64, 4096, 1 << 22)])
def test_rows_as_far_apart_as_tiles_take(n, K, N, ld):
    c = Case("bf16", n, K, N)
    rows, at = max(n, N), 0
    room = torch.empty(rows * ld, dtype=c.t, device="cuda")
    for k, height, width in (("X", n, K), ("W", N, K), ("dY", n, N)):
        v = torch.as_strided(room, (height, width), (ld, 1), at)
        v.copy_(getattr(c, k))
        setattr(c, k, v)
        at += (width + 71) // 64 * 64
    c.check()
