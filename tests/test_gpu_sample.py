"""SAMPLE_FWD (csrc/sample.hip) against the definition in 64 bits: the same token, and the logarithm of its share.

A weight is held as a whole number of 2^-bits of the largest, bits = min(50, 63 - log2(vocabulary), rounded up), so it is off by at most half of one and by 2^-50 of
itself; n such roundings, each anywhere within half a step, add up to less than 8 sqrt(n / 12) steps (8 standard deviations).  That is how far a sum may be
off, and how near to a border a random number, or a sum that top-p compares, may not be for the token to be told: no row of these tests is nearer."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn, CudaDnnDouble, CudaDnnError
from oracle import serving_ref as S
from tests.conftest import bf16_round

pytestmark = pytest.mark.gpu


def off(vocab):
    bits = min(50, 63 - int(np.ceil(np.log2(vocab))))
    return 8 * np.sqrt(vocab / 12) * 2.0 ** -bits + 2.0 ** -48


@pytest.fixture(params=["f32", "bf16", "f64"])
def kind(request):
    c = (CudaDnnDouble if request.param == "f64" else CudaDnn)(0)
    yield c, request.param
    c.Dispose()


def stored(x, kind):
    return bf16_round(x).astype(np.float64) if kind == "bf16" else np.asarray(x, np.float32 if kind == "f32" else np.float64).astype(np.float64)


def draw(cuda, kind, x, u, temperature=None, k=None, p=None, m=None, rows=None, stride=0, logs=True):
    """ids and logarithms of one call; x (rows, vocab) as stored, everything else a number a row."""
    n, vocab = (len(u), x.shape[1])
    put = lambda v: 0 if v is None else cuda.AllocMemory(np.asarray(v, cuda.DTYPE))  # noqa: E731
    width = stride or vocab
    full = np.full((x.shape[0], width), 1e4)
    full[:, :vocab] = x
    hx = cuda.AllocMemory(np.asarray(full, np.float32).reshape(-1), bHalfSize=True) if kind == "bf16" else put(full.reshape(-1))
    h = [put(v) for v in (u, temperature, k, p, m, rows)]
    out = [put(np.full(n, -9.0)) for _ in range(2)]
    cuda.SampleForward(n, vocab, hx, h[0], out[0], h[1], h[2], h[3], h[4], out[1] if logs else 0, h[5], x.shape[0] if rows is not None else 0, stride)
    got = [np.asarray(cuda.GetMemoryFloat(o), np.float64) for o in out]
    for handle in [hx] + h + out:
        if handle:
            cuda.FreeMemory(handle)
    return got


def check(cuda, kind, x, u, temperature=None, k=None, p=None, m=None, rows=None, stride=0):
    as_stored = lambda v: None if v is None else np.asarray(v, cuda.DTYPE).astype(np.float64)  # noqa: E731
    x = stored(x, kind)
    u, temperature, k, p, m = (as_stored(v) for v in (u, temperature, k, p, m))
    ids, logs = draw(cuda, kind, x, u, temperature, k, p, m, rows, stride)
    for i in range(len(u)):
        row = i if rows is None else rows[i]
        if not 0 <= row < x.shape[0]:
            assert ids[i] == -1 and logs[i] == 0
            continue
        want, log, near = S.sample(x[int(row)], u[i], *(d if v is None else v[i] for v, d in ((temperature, 1.0), (k, 0), (p, 1.0), (m, 0.0))))
        assert near > off(x.shape[1]), "row %d: choose other numbers" % i
        assert ids[i] == want, (i, ids[i], want)
        # the sum's own error, some half steps of the numbers it is made of in 64 bits, and in fp32 one rounding of the result, half a step, 2^-24 of it
        assert abs(logs[i] - log) <= (2.0 ** -24 if cuda.DTYPE == np.float32 else 0) * abs(log) + off(x.shape[1]) + 2.0 ** -48 * max(1.0, abs(log)), (i, logs[i], log)
    return ids


def logits(rng, rows, vocab, spread=2.5):
    x = rng.standard_normal((rows, vocab)) * spread
    for r in x:
        r[rng.integers(0, vocab, 12)] += 3 + 7 * rng.random(12)
    return x


VOCABS = [1, 2, 3, 63, 64, 65, 257, 1000, 4096, 4099, 32000, 50261, 131072]


@pytest.mark.parametrize("vocab", VOCABS)
def test_each_filter_alone_and_all(kind, vocab):
    cuda, t = kind
    rng = np.random.default_rng(vocab)
    n = 6
    x, u = logits(rng, n, vocab), rng.random(n)
    heat, k, p, m = 0.3 + rng.random(n), 1 + np.floor(rng.random(n) ** 3 * vocab), 0.05 + 0.9 * rng.random(n), 0.001 + 0.3 * rng.random(n)
    check(cuda, t, x, u)
    check(cuda, t, x, u, heat)
    check(cuda, t, x, u, heat, k)
    check(cuda, t, x, u, heat, None, p)
    check(cuda, t, x, u, heat, None, None, m)
    check(cuda, t, x, u, heat, k, p, m)
    assert np.array_equal(check(cuda, t, x, u, np.zeros(n), k, p, m), stored(x, t).argmax(1))


@pytest.mark.parametrize("vocab", [1 << 20, (1 << 20) - 1, 300007])
def test_large_vocabularies(kind, vocab):
    cuda, t = kind
    rng = np.random.default_rng(1)
    x, u = logits(rng, 2, vocab), np.array([0.999, 0.31])
    check(cuda, t, x, u)
    check(cuda, t, x, u, [3.0, 1.0], [200000, 40], [0.7, 0.95])


def test_many_rows_each_with_its_own_settings(kind):
    cuda, t = kind
    rng = np.random.default_rng(4)
    n, vocab = 700, 911
    x = logits(rng, n, vocab)
    some = lambda v, o: np.where(rng.random(n) < 0.4, o, v)  # noqa: E731
    check(cuda, t, x, rng.random(n), some(0.2 + 2 * rng.random(n), 0.0), some(1 + np.floor(rng.random(n) * 100), 0), some(rng.random(n), 1.0), some(0.3 * rng.random(n), 0.0))


def test_equal_logits_go_by_their_index(kind):
    """Every weight is one: the borders are whole numbers, and what is kept are the first ones.  More of them than are compared one by one."""
    cuda, t = kind
    for vocab in (7, 1000, 5000, 70001):
        x = np.zeros((6, vocab))
        u = np.array([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.90625])
        k = np.array([1, 3, min(vocab, 4000) // 2, vocab - 1, vocab, vocab + 5], float)
        x = stored(x, t)
        ids, _ = draw(cuda, t, x, u, None, k)
        kept = np.minimum(k, vocab)
        want = np.minimum(np.floor(u * kept), kept - 1)
        assert np.array_equal(ids, want), (vocab, ids, want)
        p = np.array([0.5, 0.125, 0.75, 0.25, 1.0, 2.0 ** -20])
        ids, logs = draw(cuda, t, x, u, None, None, p)
        kept = np.where(p >= 1, vocab, np.maximum(1, np.ceil(p * vocab)))
        assert np.array_equal(ids, np.floor(u * kept)), (vocab, ids, kept)
        assert np.abs(logs + np.log(kept)).max() <= 1e-6
        # a plateau below the largest, its first ones kept
        x = np.full((6, vocab), -1.0)
        x[:, vocab - 1] = 0.0
        check(cuda, t, x, np.array([0.1, 0.3, 0.45, 0.6, 0.77, 0.93]), None, np.minimum(vocab - 1, np.array([2, 2, 3, 1500, 2500, 6000.0])), np.array([1, 0.9, 0.95, 0.99, 1, 0.6]))


def test_few_values_many_times(kind):
    """Sixteen-bit logits: thousands of equal ones at the border of top-k and of top-p."""
    cuda, t = kind
    rng = np.random.default_rng(3)
    x = np.round(rng.standard_normal((5, 60000)) * 4) / 4
    check(cuda, t, x, rng.random(5), [0.7, 1, 1.5, 3, 9], [30, 3000, 30001, 40000, 0], [1, 0.8, 0.93, 0.4, 0.55])


def test_infinities_and_what_is_not_a_number(kind):
    cuda, t = kind
    inf, nan = np.inf, np.nan
    x = np.array([[nan, 1.0, -inf, 0.5, nan], [-inf] * 5, [nan] * 5, [inf, 3.0, inf, -inf, nan], [-inf, -inf, -3e38, -inf, -inf], [-0.0, 0.0, -0.0, 0.0, -inf]])
    for u in (0.0, 0.3, 0.999):
        check(cuda, t, x, np.full(6, u))
        check(cuda, t, x, np.full(6, u), np.full(6, 0.5), np.full(6, 3.0), np.full(6, 0.7), np.full(6, 0.1))
        check(cuda, t, x, np.full(6, u), np.zeros(6))
    ids, _ = draw(cuda, t, stored(x, t), np.full(6, 0.6))
    assert ids[3] in (0, 2) and ids[1] == ids[2] == -1


def test_numbers_at_the_ends_of_their_ranges(kind):
    cuda, t = kind
    rng = np.random.default_rng(8)
    x = logits(rng, 1, 500)
    n = 12
    x = np.repeat(x, n, 0)
    nan, inf = np.nan, np.inf
    u = np.array([0, 1, 2, -1, nan, 1 - 2.0 ** -24, 2.0 ** -30, 0.5, 0.5, 0.5, 0.5, 0.5])
    check(cuda, t, x, u)
    half = np.full(n, 0.3703)
    check(cuda, t, x, half, np.array([nan, -1, 0, 1e-30, 1e-3, 1e30, 1e-44, 5, 0.01, 100, 0.1, 1e4]))
    check(cuda, t, x, half, None, np.array([nan, -5, 0, 0.5, 1, 1.9, 499, 500, 501, 1e30, 2, 3]))
    check(cuda, t, x, half, None, None, np.array([nan, -1, 0, 1, 2, 1e-30, 1 - 2.0 ** -24, 0.5, inf, 0.9, 0.1, 0.99]))
    check(cuda, t, x, half, None, None, None, np.array([nan, -1, 0, 1, 1.5, inf, 1e-30, 0.5, 0.02, 0.9, 0.1, 0.99]))
    # all logits of one weight, whatever they are
    ids, _ = draw(cuda, t, stored(x[:1], t), [0.5], [inf])
    assert ids[0] == 250


def test_rows_by_their_numbers_and_strides(kind):
    cuda, t = kind
    rng = np.random.default_rng(5)
    x = logits(rng, 9, 77)
    rows = [8, 0, 0, -1, 3, 9, 7, float("nan"), 5, 2, 1]
    check(cuda, t, x, rng.random(11), np.full(11, 0.8), None, np.full(11, 0.9), None, rows, 80)
    check(cuda, t, x, rng.random(11), None, None, None, None, rows, 79)
    check(cuda, t, x, rng.random(9), None, np.full(9, 5.0), None, None, None, 131)


def test_draws_follow_the_weights(kind):
    """Evenly spread random numbers draw every token as often as its weight says, to the last one."""
    cuda, t = kind
    w = np.array([1, 2, 4, 8, 16, 32, 1, 64, 128, 256, 512, 1024]) / 2048.0
    n = 2048
    x = np.repeat(np.log2(w)[None], n, 0)
    ids, _ = draw(cuda, t, stored(x, t), (np.arange(n) + 0.5) / n, np.full(n, 1 / np.log(2.0)))
    assert np.array_equal(np.bincount(ids.astype(int), minlength=12), w * n)


def test_more_rows_than_an_axis_of_a_launch_has():
    """2^22 rows and some, of three logits each; the largest logit, and draws at the borders of equal ones."""
    cuda = CudaDnn(0)
    rng = np.random.default_rng(20)
    n = (1 << 22) + 5
    x = rng.integers(-2, 3, (n, 3)).astype(np.float32)
    heat = np.where(np.arange(n) % 2, 0.0, 1.0)
    u = rng.integers(0, 8, n) / 8 + 1 / 16
    ids, _ = draw(cuda, "f32", x, u, heat, logs=False)
    w = np.cumsum(np.exp(np.float64(x)), 1)
    want = np.where(np.arange(n) % 2, x.argmax(1), (w <= u[:, None] * w[:, -1:]).sum(1))
    assert np.array_equal(ids, want)
    cuda.Dispose()


def test_calls_in_turn_leave_nothing_behind(kind):
    cuda, t = kind
    rng = np.random.default_rng(6)
    x = logits(rng, 33, 2049)
    u = rng.random(33)
    first = draw(cuda, t, stored(x, t), u, np.full(33, 0.9), np.full(33, 70.0), np.full(33, 0.8))
    for _ in range(3):
        check(cuda, t, logits(rng, 5, 40000), rng.random(5), None, None, np.full(5, 0.5))
        again = draw(cuda, t, stored(x, t), u, np.full(33, 0.9), np.full(33, 70.0), np.full(33, 0.8))
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_refusals(kind):
    cuda, t = kind
    x = cuda.AllocMemory(np.zeros(400, cuda.DTYPE))
    n = [cuda.AllocMemory(np.zeros(8, cuda.DTYPE)) for _ in range(8)]
    good = dict(nRows=4, nVocab=100, hLogits=x, hRandom=n[0], hIds=n[1], hTemperature=n[2], hTopK=n[3], hTopP=n[4], hMinP=n[5], hLogProb=n[6], hRows=n[7])

    def refused(**change):
        with pytest.raises(CudaDnnError):
            cuda.SampleForward(**{**good, **change})

    for bad in (0, -1, (1 << 24) + 1):
        refused(nRows=bad)
    for bad in (0, -4, (1 << 20) + 1, 101):
        refused(nVocab=bad)
    refused(nRowStride=99)
    refused(nRowStride=101)
    refused(nRowStride=1 << 60)
    refused(nLogitsRows=5)
    refused(nLogitsRows=-1)
    refused(nRows=9, nVocab=4)
    refused(hLogits=0)
    refused(hRandom=0)
    refused(hIds=0)
    for name in ("hLogits", "hRandom", "hTemperature", "hTopK", "hTopP", "hMinP", "hRows", "hLogProb"):
        refused(hIds=good[name])
    refused(hLogProb=n[0])
    if cuda.DTYPE == np.float32:
        half = cuda.AllocMemory(8, bHalfSize=True)
        for name in ("hRandom", "hIds", "hTemperature", "hTopK", "hTopP", "hMinP", "hRows", "hLogProb"):
            refused(**{name: half})
        cuda.FreeMemory(half)
    cuda.SampleForward(**good)
