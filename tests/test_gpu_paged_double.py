"""Head norms, append and attention over pages in the double base type, against the definitions; their refusals."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnnDouble, CudaDnnError
from tests.test_gpu_head_norm import EPS, THETA, backward, forward
from tests.test_gpu_paged import head_norm, turned

pytestmark = pytest.mark.gpu
# sums of at most some hundred terms, angles of at most some hundred radians: both off by at most that many half steps of 2^-53 (1.1e-16)
TOL = 1e-13


@pytest.fixture()
def cuda():
    c = CudaDnnDouble(0)
    yield c
    c.Dispose()


def close(got, want):
    assert np.abs(got.reshape(want.shape) - want).max() <= TOL * max(np.abs(want).max(), 1e-300)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("B,T,H,kvH,hs", [(2, 5, 3, 1, 6), (1, 40, 4, 2, 64), (2, 3, 2, 2, 198), (1, 2, 1, 1, 256)])
def test_head_norms(cuda, B, T, H, kvH, hs, rope):
    rng = np.random.default_rng(hs)
    hr = cuda.CreateRope(0, 0, 1, B, T, H, hs, THETA) if rope else 0
    x, w = [rng.standard_normal((B, h, T, hs)) for h in (H, kvH)], [1 + 0.3 * rng.standard_normal(hs) for _ in range(2)]
    dy = [rng.standard_normal(t.shape) for t in x]
    hx, hw, hdy = ([cuda.AllocMemory(t) for t in ts] for ts in (x, w, dy))
    hy, hdx, hdw = ([cuda.AllocMemory(t.size) for t in ts] for ts in (x, x, w))
    cuda.QkNormRopeForward(B, T, H, kvH, hs, *hx, *hw, *hy, hr, EPS)
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *hx, *hw, *hdy, *hdx, *hdw, hr, EPS)
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *hx, *hw, *hdy, *hdx, *hdw, hr, EPS, True)
    for i in range(2):
        close(cuda.GetMemoryFloat(hy[i]), forward(x[i], w[i], rope))
        dx, dw = backward(x[i], w[i], dy[i], rope)
        close(cuda.GetMemoryFloat(hdx[i]), dx)
        close(cuda.GetMemoryFloat(hdw[i]), 2 * dw.sum((0, 1, 2)))
    for code, at, value in ((90001, 4, 7), (90001, 0, 0), (90010, 1, T + 1), (90001, 11, hx[0]), (90014, 5, 9999)):
        a = [B, T, H, kvH, hs, *hx, *hw, *hy]
        a[at if at < 11 else 10] = value
        if at == 11:
            a[9] = a[10] = hy[0]
        with pytest.raises(CudaDnnError) as e:
            cuda.QkNormRopeForward(*a, 0, EPS)
        assert e.value.code in (code, 90010) if at == 11 else e.value.code == code


@pytest.mark.parametrize("H,kvH,hs,page", [(3, 1, 6, 5), (4, 2, 64, 16), (2, 2, 256, 8)])
def test_paged(cuda, H, kvH, hs, page):
    rng = np.random.default_rng(hs)
    plans, totals, width, pages = [[7, 3, 0], [1, 9, 2], [1, 0, 1]], [9, 12, 3], 4, 14
    rows = [rng.standard_normal((t, H + 2 * kvH, hs)) for t in totals]
    w = [1 + 0.3 * rng.standard_normal(hs) for _ in range(2)]
    hw = [cuda.AllocMemory(t) for t in w]
    hk, hv = (cuda.AllocMemory(np.full(pages * kvH * page * hs, np.nan)) for _ in range(2))
    hr = cuda.CreateRope(0, 0, 1, 1, width * page, H, hs, THETA)
    table = np.stack([rng.permutation(pages)[:width] if b == 0 else np.zeros(width) for b in range(3)]).astype(np.float64)
    perm = rng.permutation(pages)
    for b in range(3):
        table[b] = perm[4 * b:4 * b + 4]
    have = [0, 0, 0]
    strides = (kvH * page * hs, hs, kvH * hs)
    for plan in plans:
        new = np.concatenate([rows[b][have[b]:have[b] + n] for b, n in enumerate(plan)])
        have = [a + n for a, n in zip(have, plan)]
        N = len(new)
        ht, hs_, hl = cuda.AllocMemory(table), cuda.AllocMemory(np.concatenate([[0], np.cumsum(plan)])), cuda.AllocMemory(np.float64(have))
        hx, hq, hy = cuda.AllocMemory(new), cuda.AllocMemory(N * H * hs), cuda.AllocMemory(N * H * hs)
        sizes = (3, N, H, kvH, hs, pages, page, width)
        cuda.PagedAppend(*sizes, hx, hq, hk, hv, ht, hs_, hl, *strides, hr, True, *hw, EPS)
        cuda.AttnPagedForward(*sizes, hq, hk, hv, ht, hs_, hl, hy, *strides)
        got, q, at = cuda.GetMemoryFloat(hy).reshape(N, H, hs), cuda.GetMemoryFloat(hq).reshape(N, H, hs), 0
        for b, n in enumerate(plan):
            pos = np.arange(have[b])
            k, v = turned(head_norm(rows[b][:have[b], H:H + kvH], w[1]), pos), rows[b][:have[b], H + kvH:]
            qq = turned(head_norm(rows[b][:have[b], :H], w[0]), pos)
            for j in range(n):
                p = have[b] - n + j
                close(q[at + j], qq[p])
                for h in range(H):
                    s = k[:p + 1, h // (H // kvH)] @ qq[p, h] / np.sqrt(hs)
                    e = np.exp(s - s.max())
                    close(got[at + j, h], e / e.sum() @ v[:p + 1, h // (H // kvH)])
            at += n
    with pytest.raises(CudaDnnError) as e:
        cuda.AttnPagedForward(*sizes, hq, hk, hv, ht, hs_, hl, hq, *strides)
    assert e.value.code == 90001
    with pytest.raises(CudaDnnError) as e:
        cuda.PagedAppend(*sizes, hx, hq, hk, hv, ht, hs_, hl, strides[0], strides[1], hs - 1, hr, True, *hw, EPS)
    assert e.value.code == 90001
    with pytest.raises(CudaDnnError) as e:
        cuda.PagedAppend(3, N, H, kvH, hs, pages + 1, page, width, hx, hq, hk, hv, ht, hs_, hl, *strides, hr, True, *hw, EPS)
    assert e.value.code == 90010
