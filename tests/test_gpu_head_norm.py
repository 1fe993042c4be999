"""Norms of queries and keys for each head with the rotation (ids 2013, 2014), against the formulas in 64 bits and against differences."""
import numpy as np
import pytest

from tests.conftest import bf16_round
from mycaffe_amd.cudadnn import CudaDnnError

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
EPS, THETA = 1e-5, 10000.0


def rounded(a, half):
    return bf16_round(a) if half else np.float32(a)


def turn(x, back=False):
    """(..., T, hs) turned to positions 0 .. T - 1"""
    T, hs = x.shape[-2:]
    a = np.arange(T)[:, None] * THETA ** (-np.arange(0, hs, 2) / hs)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(-1j * a if back else 1j * a)
    return np.stack([z.real, z.imag], -1).reshape(x.shape)


def forward(x, w, rope):
    y = w * x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    return turn(y) if rope else y


def backward(x, w, dy, rope):
    g = turn(dy, True) if rope else dy
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    n = x * r
    gw = g * w
    return r * (gw - n * (gw * n).mean(-1, keepdims=True)), g * n


def pair_size(x):
    return np.repeat(np.hypot(x[..., 0::2], x[..., 1::2]), 2, -1)


SHAPES = [(1, 1, 1, 1, 64), (2, 5, 6, 6, 48), (2, 33, 8, 2, 128), (1, 100, 12, 12, 64), (3, 7, 3, 1, 6), (1, 3, 2, 2, 2), (2, 9, 2, 1, 256), (1, 17, 5, 3, 198),
          (4, 257, 7, 1, 96), (1, 2100, 2, 2, 32)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rope,weights", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("B,T,H,kvH,hs", SHAPES)
def test_forward_and_backward(dev, B, T, H, kvH, hs, rope, weights, half):
    rng = np.random.default_rng(B * T + hs)
    cuda = dev.cuda
    hr = cuda.CreateRope(0, 0, 1, B, T, H, hs, THETA) if rope else 0
    x = [rounded(rng.standard_normal((B, h, T, hs)) * 2, half) for h in (H, kvH)]
    w = [rounded(1 + 0.3 * rng.standard_normal(hs), half) for _ in range(2)] if weights else [np.ones(hs, np.float32)] * 2
    dy = [rounded(rng.standard_normal(t.shape), half) for t in x]
    hx, hdy = [dev.put(t, half) for t in x], [dev.put(t, half) for t in dy]
    hw = [dev.put(t, half) for t in w] if weights else [0, 0]
    hy, hdx, hdw = ([dev.zeros(t.size, half) for t in ts] for ts in (x, x, w))
    cuda.QkNormRopeForward(B, T, H, kvH, hs, *hx, *hw, *hy, hr, EPS)
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *hx, *hw, *hdy, *hdx, *hdw, hr, EPS)
    u = U16 if half else U32
    # 1 / rms: hs roundings of the mean's terms, halved by the root, and root, quotient, products; a rotation: two products, a sum, a rounded cosine and sine
    inv = (hs + 2) * U32 / 2 + 6 * U32
    rot = 4 * U32 if rope else 0
    for i in range(2):
        x64, w64, dy64 = x[i].astype(np.float64), w[i].astype(np.float64), dy[i].astype(np.float64)
        want = forward(x64, w64, rope)
        plain = forward(x64, w64, False)
        tol = (inv + rot) * (pair_size(plain) if rope else abs(plain)) + u * abs(want) + 1e-37
        assert (abs(dev.get(hy[i], x[i].shape) - want) <= tol).all()
        dx, dw = backward(x64, w64, dy64, rope)
        g = turn(dy64, True) if rope else dy64
        gs = pair_size(g) if rope else abs(g)
        r = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + EPS)
        n = abs(x64 * r)
        # every term as above; the mean of hs products once more
        terms = r * (gs * abs(w64) + n * (gs * abs(w64) * n).mean(-1, keepdims=True))
        tol = (4 * inv + rot + (hs + 8) * U32) * terms + u * abs(dx) + 1e-37
        assert (abs(dev.get(hdx[i], x[i].shape) - dx) <= tol).all()
        rows = x64.size // hs
        tol = (inv + rot + 2 * U32 + rows * U32) * (gs * n).sum((0, 1, 2)) + u * abs(dw.sum((0, 1, 2)))
        assert (abs(dev.get(hdw[i]) - dw.sum((0, 1, 2))) <= tol).all()
    # in place, and the weights' gradients added to what is there
    once = [dev.get(h) for h in hdw]
    keep = [dev.get(h) for h in hy]
    grads = [dev.get(h) for h in hdx]
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *hx, *hw, *hdy, *hdy, *hdw, hr, EPS, True)
    for i in range(2):
        assert np.array_equal(dev.get(hdy[i]), grads[i])
        assert (abs(dev.get(hdw[i]) - 2 * once[i].astype(np.float64)) <= 2 * u * abs(2 * once[i]) + 2 * u * abs(once[i]) + 1e-30).all()
    cuda.QkNormRopeForward(B, T, H, kvH, hs, *hx, *hw, *hx, hr, EPS)
    for i in range(2):
        assert np.array_equal(dev.get(hx[i]), keep[i])
    if hr:
        cuda.FreeRope(hr)


def test_gradient_against_differences(dev):
    """central differences of the fp32 forward pass"""
    rng = np.random.default_rng(3)
    B, T, H, kvH, hs = 1, 3, 2, 1, 8
    cuda = dev.cuda
    hr = cuda.CreateRope(0, 0, 1, B, T, H, hs, THETA)
    x = [np.float32(rng.standard_normal((B, h, T, hs))) for h in (H, kvH)]
    w = [np.float32(1 + 0.3 * rng.standard_normal(hs)) for _ in range(2)]
    dy = [np.float32(rng.standard_normal(t.shape)) for t in x]

    def loss(x, w):
        hx, hw, hy = [dev.put(t) for t in x], [dev.put(t) for t in w], [dev.zeros(t.size) for t in x]
        cuda.QkNormRopeForward(B, T, H, kvH, hs, *hx, *hw, *hy, hr, EPS)
        return sum((dev.get(h, t.shape).astype(np.float64) * t).sum() for h, t in zip(hy, dy))
    hdx, hdw = [dev.zeros(t.size) for t in x], [dev.zeros(hs) for _ in w]
    cuda.QkNormRopeBackward(B, T, H, kvH, hs, *[dev.put(t) for t in x], *[dev.put(t) for t in w], *[dev.put(t) for t in dy], *hdx, *hdw, hr, EPS)
    step = 2.0 ** -7
    for which, grads in ((x, [dev.get(h) for h in hdx]), (w, [dev.get(h) for h in hdw])):
        for i in range(2):
            for at in rng.choice(which[i].size, 6, replace=False):
                value = []
                for s in (step, -step):
                    moved = [t.copy() for t in which]
                    moved[i].reshape(-1)[at] += np.float32(s)
                    value.append(loss(moved, w) if which is x else loss(x, moved))
                # second differences of order step^2; the forward pass's own roundings over the step
                assert abs((value[0] - value[1]) / (2 * step) - grads[i][at]) < 30 * step ** 2 + 200 * U32 / step * 4
    cuda.FreeRope(hr)


def test_zero_rows_and_not_finite(dev):
    """a row of zeros stays one and has a finite gradient; a row with a value that is not finite leaves the others alone"""
    rng = np.random.default_rng(4)
    hs = 64
    for half in (False, True):
        x = rounded(rng.standard_normal((1, 4, 3, hs)), half)
        x[0, 0, 1] = 0
        bad = x.copy()
        bad[0, 2, 1, 5] = np.inf
        dy, w = rounded(rng.standard_normal(x.shape), half), rounded(np.ones(hs), half)
        got = []
        for t in (x, bad):
            h = [dev.put(t, half), dev.put(x[:, :1], half)]
            y, dx = [dev.zeros(x.size, half), dev.zeros(x[:, :1].size, half)], [dev.zeros(x.size, half), dev.zeros(x[:, :1].size, half)]
            hw = [dev.put(w, half), dev.put(w, half)]
            dev.cuda.QkNormRopeForward(1, 3, 4, 1, hs, *h, *hw, *y, 0, EPS)
            dev.cuda.QkNormRopeBackward(1, 3, 4, 1, hs, *h, *hw, dev.put(dy, half), dev.put(dy[:, :1], half), *dx, 0, 0, 0, EPS)
            got.append((dev.get(y[0], x.shape), dev.get(dx[0], x.shape)))
        assert (got[0][0][0, 0, 1] == 0).all() and np.isfinite(got[0][1]).all()
        for a, b in zip(*got):
            keep = np.ones(x.shape[:3], bool)
            keep[0, 2, 1] = False
            assert np.array_equal(a[keep], b[keep])


def test_refusals(dev):
    B, T, H, kvH, hs = 2, 5, 4, 2, 64
    q, k, w = dev.zeros(B * T * H * hs), dev.zeros(B * T * kvH * hs), dev.zeros(hs)
    yq, yk, w2, w3 = dev.zeros(B * T * H * hs), dev.zeros(B * T * kvH * hs), dev.zeros(hs), dev.zeros(hs)
    dq, dk = dev.zeros(B * T * H * hs), dev.zeros(B * T * kvH * hs)
    rope, short = (dev.cuda.CreateRope(0, 0, 1, B, t, H, hs, THETA) for t in (T, T - 1))
    f, g = dev.cuda.QkNormRopeForward, dev.cuda.QkNormRopeBackward
    good, back = [B, T, H, kvH, hs, q, k, w, w, yq, yk], [B, T, H, kvH, hs, q, k, w, w, yq, yk, dq, dk, w2, w3]
    f(*good, rope)
    g(*back, rope)

    def bad(code, call, a, at, value, *more):
        a = list(a)
        a[at] = value
        with pytest.raises(CudaDnnError) as e:
            call(*a, *more)
        assert e.value.code == code
    for call, a in ((f, good), (g, back)):
        for i in range(5):
            for v in (0, -1, 1 << 40):
                bad(90001, call, a, i, v)
        bad(90001, call, a, 4, 63)
        bad(90010, call, a, 1, 6)
        bad(90010, call, a, 3, 3)
        bad(90011, call, a, 5, dev.zeros(B * T * H * hs, True))
        bad(90011, call, a, 7, dev.zeros(hs, True))
        bad(90010, call, a, 7, dev.zeros(hs - 2))
        bad(90001, call, a, 0, B, short)
        bad(90201, call, a, 0, B, 77)
        bad(90001, call, a, 0, B, rope, float("nan"))
    bad(90001, f, good, 10, yq)          # both outputs in one place
    bad(90010, f, good, 9, w)            # too small before it is a clash
    bad(90001, f, good, 7, yq)
    bad(90001, g, back, 12, dq)
    bad(90001, g, back, 14, w2)
    bad(90001, g, back, 13, w)
    bad(90001, g, back, 7, dq)
    with pytest.raises(CudaDnnError):
        view = dev.cuda.CreateMemoryPointer(q, hs, B * T * H * hs - hs)
        f(B, T - 1, H, kvH, hs, q, k, w, w, view, yk)
    for r in (rope, short):
        dev.cuda.FreeRope(r)
