"""Norms of queries and keys for each head (ids 2013, 2014) without an epsilon: positions that fill no workgroup, against the formulas in 64 bits."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnnDouble
from tests.test_gpu_head_norm import U16, U32, rounded

pytestmark = pytest.mark.gpu

# positions: one, a few, one past what the narrowest head's workgroup takes (32), sequences in a batch
SHAPES = [(1, 1, 2, 1, 64), (1, 5, 6, 6, 48), (1, 33, 3, 1, 6), (2, 5, 2, 2, 128), (1, 3, 2, 1, 256), (3, 7, 5, 5, 64)]


def formulas(x, w, dy):
    x, w, dy = (t.astype(np.float64) for t in (x, w, dy))
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True))
    n, gw = x * r, dy * w
    return n * w, r * (gw - n * (gw * n).mean(-1, keepdims=True)), (dy * n).sum((0, 1, 2)), r, n


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("B,T,H,kvH,hs", SHAPES)
def test_no_epsilon(dev, B, T, H, kvH, hs, half):
    rng = np.random.default_rng(40 + T + hs)
    cuda, u = dev.cuda, U16 if half else U32
    # no row is zero: magnitudes from 0.5 up
    x = [rounded(np.sign(t) * (0.5 + abs(t)), half) for t in (rng.standard_normal((B, h, T, hs)) for h in (H, kvH))]
    dy = [rounded(rng.standard_normal(t.shape), half) for t in x]
    w = [rounded(1 + 0.3 * rng.standard_normal(hs), half) for _ in range(2)]
    hx, hdy, hw = ([dev.put(t, half) for t in ts] for ts in (x, dy, w))
    hy, hdx, hdw = ([dev.zeros(t.size, half) for t in ts] for ts in (x, x, w))
    cuda.QkNormRopeForward(B, T, H, kvH, hs, *hx, *hw, *hy, 0, 0.0)
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *hx, *hw, *hdy, *hdx, *hdw, 0, 0.0)
    # 1 / rms: hs roundings of the mean's terms, halved by the root, and root, quotient, products
    inv = (hs + 2) * U32 / 2 + 6 * U32
    for i in range(2):
        y, dx, dw, r, n = formulas(x[i], w[i], dy[i])
        assert (abs(dev.get(hy[i], y.shape) - y) <= inv * abs(y) + u * abs(y)).all()
        gw = abs(dy[i].astype(np.float64) * w[i])
        terms = r * (gw + abs(n) * (gw * abs(n)).mean(-1, keepdims=True))
        assert (abs(dev.get(hdx[i], dx.shape) - dx) <= (4 * inv + (hs + 8) * U32) * terms + u * abs(dx)).all()
        rows = x[i].size // hs
        got = dev.get(hdw[i])
        assert np.isfinite(got).all()
        assert (abs(got - dw) <= (inv + 2 * U32 + rows * U32) * abs(dy[i] * n).sum((0, 1, 2)) + u * abs(dw)).all()


def test_no_epsilon_in_double():
    """The double base type, to 1e-12 of the terms."""
    rng, cuda = np.random.default_rng(50), CudaDnnDouble(0)
    try:
        B, T, H, kvH, hs = 1, 5, 3, 1, 48
        x, dy = ([rng.standard_normal((B, h, T, hs)) for h in (H, kvH)] for _ in range(2))
        w = [1 + 0.3 * rng.standard_normal(hs) for _ in range(2)]
        put = lambda ts: [cuda.AllocMemory(np.asarray(t, np.float64).reshape(-1)) for t in ts]  # noqa: E731
        hdx, hdw = put([np.zeros(t.size) for t in x]), put([np.zeros(hs)] * 2)
        cuda.QkNormRopeBackward(B, T, H, kvH, hs, *put(x), *put(w), *put(dy), *hdx, *hdw, 0, 0.0)
        for i in range(2):
            _, dx, dw, _, n = formulas(x[i], w[i], dy[i])
            assert (abs(np.asarray(cuda.GetMemoryFloat(hdx[i])).reshape(dx.shape) - dx) <= 1e-12 * abs(dx).max()).all()
            assert (abs(np.asarray(cuda.GetMemoryFloat(hdw[i])) - dw) <= 1e-12 * abs(dy[i] * n).sum((0, 1, 2))).all()
    finally:
        cuda.Dispose()
