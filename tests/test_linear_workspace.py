"""cavs_linear_workspace covers whatever path a call takes: shapes, strides and alignments of every kind, every choice of results.  Without a device: a call that gets as far
as its first launch has found its plan inside the workspace (and would write to made-up addresses where there is a device)."""
import random

import pytest

from cavs_amd import hip

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="launches must fail")

FAR = 1 << 40  # (an address that only the refused launch sees)


def _shapes(seed, count):
    r = random.Random(seed)
    size = lambda most: max(1, round(2 ** r.uniform(0, most)) // r.choice([1, 8]) * r.choice([1, 8]))  # noqa: E731
    return [(size(13), size(12), size(13)) for _ in range(count)]


def _reaches_its_launch(name, *args):
    with pytest.raises(hip.CavsError) as e:
        hip.call(name, *args, None)
    assert "hipGetLastError" in str(e.value), (args, str(e.value))


KNOWN = [(1082, 105, 576), (2058, 833, 2816), (300, 1, 8), (70, 13, 4096), (1082, 104, 576)]


@pytest.mark.parametrize("type_", [hip.F32, hip.BF16])
@pytest.mark.parametrize("off", [0, 2, 8])
def test_gradients(type_, off):
    """(off: bytes of X and W behind 16, elements of stride beyond the width)"""
    off = 2 * off if type_ == hip.F32 else off
    for n, K, N in KNOWN + _shapes(off, 400):
        need = hip.lib().cavs_linear_workspace(type_, n, K, N, 1)
        for wanted in range(1, 8):
            dX, dW, db = (FAR if wanted >> i & 1 else None for i in range(3))
            _reaches_its_launch("cavs_linear_bwd", type_, FAR + off, K + off, FAR + off, K + off, FAR, N, wanted % 6, None, FAR, N, dX, K, dW, K, db, n, K, N, FAR, need)


@pytest.mark.parametrize("type_", [hip.F32, hip.BF16])
@pytest.mark.parametrize("off", [0, 2, 8])
def test_forward(type_, off):
    off = 2 * off if type_ == hip.F32 else off
    for n, K, N in KNOWN + _shapes(off + 1, 400):
        need = hip.lib().cavs_linear_workspace(type_, n, K, N, 0)
        _reaches_its_launch("cavs_linear_fwd", type_, FAR + off, K + off, FAR + off, K + off, None, 0, None, None, 0, None, 0, FAR, N, n, K, N, FAR, need)
