"""SAMPLE_FWD where rows are long and many enough to be cut into slices (csrc/sample.hip): everything that decides how a row is finished, at both sizes of slices.
Tolerances are those of test_gpu_sample.py."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn
from tests.test_gpu_sample import check, draw, logits, stored

pytestmark = pytest.mark.gpu

# cut: from 24576 logits on, 49152 for more than 128 rows, 2048 for more than 512; into slices of 2048 logits if these are fewer than 4096 and 128 a row, else of 8192
SIZES = [(600, 2048), (513, 4097), (4, 24576), (16, 32768), (6, 100003), (40, 50261), (129, 49152), (90, 100003), (1, 600000), (2, (1 << 20) - 3), (1, 1 << 20)]


@pytest.fixture(params=["f32", "bf16"])
def kind(request):
    c = CudaDnn(0)
    yield c, request.param
    c.Dispose()


def some(rng, n, value, off, share=0.4):
    return np.where(rng.random(n) < share, off, value)


@pytest.mark.parametrize("n,vocab", SIZES)
def test_every_row_with_its_own_settings(kind, n, vocab):
    cuda, t = kind
    rng = np.random.default_rng(vocab)
    x, u = logits(rng, n, vocab), rng.random(n)
    heat = 0.3 + 2 * rng.random(n)
    check(cuda, t, x, u)
    check(cuda, t, x, u, heat)
    check(cuda, t, x, u, some(rng, n, heat, 0.0), some(rng, n, 1 + np.floor(rng.random(n) * 200), 0), some(rng, n, 0.05 + 0.9 * rng.random(n), 1.0),
          some(rng, n, 0.3 * rng.random(n), 0.0))


@pytest.mark.parametrize("k", [1, 2, 250, 256, 257, 3000, 4090, 4100, 9000, 40000, 65534, 65535, 65536])
def test_top_k_of_every_length(kind, k):
    """Few candidates compared one by one, more in bins, more than a list holds, all tokens but one, all of them; with and without top-p behind it."""
    cuda, t = kind
    rng = np.random.default_rng(k)
    n, vocab = 9, 65535
    x, u = logits(rng, n, vocab), rng.random(n)
    check(cuda, t, x, u, None, np.full(n, float(k)))
    check(cuda, t, x, u, np.full(n, 1.5), np.full(n, float(k)), 0.05 + 0.9 * rng.random(n))
    check(cuda, t, x, u, np.full(n, 0.7), np.full(n, float(k)), None, np.full(n, 0.01))


@pytest.mark.parametrize("spread", [0.0001, 0.3, 3.0, 40.0])
def test_top_p_of_every_length(kind, spread):
    """From a head of a few tokens to one of nearly all; logits close together, which leave many tokens in one bin."""
    cuda, t = kind
    rng = np.random.default_rng(7)
    n, vocab = 10, 60001
    x, u = rng.standard_normal((n, vocab)) * spread, rng.random(n)
    p = np.array([2.0 ** -20, 0.001, 0.1, 0.5, 0.9, 0.99, 0.999, 0.999999, 1.0, 0.3])
    heat = np.full(n, 1.0 if spread < 1 else 2.0)
    # sums that decide for equal values are decided by an index, and stand where a few weights of the same size meet
    check(cuda, t, x, u, heat, None, p)
    check(cuda, t, x, u, heat, None, None, p)


def test_equal_logits_go_by_their_index(kind):
    """A whole row in one bin, more tokens than a list holds; and behind a peak."""
    cuda, t = kind
    n, vocab = 16, 40009
    u = (np.arange(n) + 0.5) / n
    k = np.array([1, 2, 3, 255, 256, 257, 4095, 4096, 4097, 20000, vocab - 1, vocab, vocab + 1, 5, 6, 7], float)
    kept = np.minimum(k, vocab)
    ids, logs = draw(cuda, t, stored(np.zeros((n, vocab)), t), u, None, k)
    assert np.array_equal(ids, np.floor(u * kept))
    assert (abs(logs + np.log(kept)) <= (2.0 ** -24 + 2.0 ** -46) * np.log(kept)).all()
    p = np.where(np.arange(n) % 2, 0.5, 0.25)
    ids, _ = draw(cuda, t, stored(np.zeros((n, vocab)), t), u, None, None, p)
    assert np.array_equal(ids, np.floor(u * np.ceil(p * vocab)))
    # of k tokens the fewest that add up to half of them
    ids, _ = draw(cuda, t, stored(np.zeros((n, vocab)), t), u, None, k, np.full(n, 0.5))
    assert np.array_equal(ids, np.floor(u * np.ceil(0.5 * kept)))
    x = np.zeros((n, vocab))
    x[:, 777] = 1.0
    ids, _ = draw(cuda, t, stored(x, t), np.full(n, 1 - 2.0 ** -24), None, k)
    assert np.array_equal(ids, np.where(k == 1, 777, np.where(kept - 2 >= 777, kept - 1, np.maximum(kept - 2, 777))))


def test_few_values_many_times(kind):
    """Borders that fall among thousands of equal logits."""
    cuda, t = kind
    rng = np.random.default_rng(8)
    n, vocab = 12, 50001
    x = rng.integers(-3, 4, (n, vocab)).astype(float)
    check(cuda, t, x, rng.random(n), np.full(n, 0.9), 1 + np.floor(rng.random(n) * vocab))
    check(cuda, t, x, rng.random(n), np.full(n, 0.9), None, 0.05 + 0.9 * rng.random(n))
    check(cuda, t, x, rng.random(n), np.full(n, 0.9), 1 + np.floor(rng.random(n) * vocab), 0.05 + 0.9 * rng.random(n), 0.1 * rng.random(n))


def test_infinities_and_what_is_not_a_number(kind):
    cuda, t = kind
    rng = np.random.default_rng(9)
    n, vocab = 20, 30011
    x = logits(rng, n, vocab)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, rng.integers(0, vocab, 9)] = np.inf
    x[3, 1:] = -np.inf
    x[4, :-1] = np.nan
    x[5, ::2] = -np.inf
    x[6, 2048:] = -np.inf
    x[7, :8192] = np.nan
    x[8] = 3e38 * np.sign(x[8])
    x[9] = -3e38
    x[10, 5:] = -3e38
    heat = np.full(n, 0.9)
    for args in ((), (heat,), (heat, np.full(n, 30.0)), (heat, None, np.full(n, 0.9)), (heat, None, None, np.full(n, 0.05)), (heat, np.full(n, 300.0), np.full(n, 0.473), np.full(n, 0.01))):
        ids = check(cuda, t, x, rng.random(n), *args)
        assert ids[0] == -1 and ids[1] == -1 and ids[3] == 0 and ids[4] == vocab - 1
    assert (check(cuda, t, x, rng.random(n), np.zeros(n))[:2] == -1).all()


def test_rows_by_their_numbers_and_strides(kind):
    cuda, t = kind
    rng = np.random.default_rng(10)
    x = logits(rng, 50, 25001)
    rows = rng.permutation(np.concatenate([np.arange(50), rng.integers(0, 50, 40), np.full(30, -1), [50, 1e9, -5, np.nan]]).astype(float))
    m = len(rows)
    for stride in (25001, 25002, 25008, 25009):
        check(cuda, t, x, rng.random(m), np.full(m, 0.8), np.full(m, 50.0), np.full(m, 0.9), None, rows, stride)
        check(cuda, t, x, rng.random(m), some(rng, m, 0.8, 0.0), None, None, None, rows, stride)


def test_the_same_tokens_alone_and_among_others(kind):
    """A row alone, which one workgroup does, and the same one among many, which are cut into slices: the same id and the same logarithm to the last bit."""
    cuda, t = kind
    rng = np.random.default_rng(11)
    n, vocab = 520, 12003
    x, u = stored(logits(rng, n, vocab), t), rng.random(n)
    settings = [0.3 + rng.random(n), some(rng, n, 1 + np.floor(rng.random(n) * 300), 0), some(rng, n, rng.random(n), 1.0), some(rng, n, 0.2 * rng.random(n), 0.0)]
    ids, logs = draw(cuda, t, x, u, *settings)
    for i in range(0, n, 5):
        one, log = draw(cuda, t, x[i:i + 1], u[i:i + 1], *[s[i:i + 1] for s in settings])
        assert one[0] == ids[i] and log[0] == logs[i], i


def test_calls_of_all_kinds_in_turn(kind):
    """Nothing that a call leaves in its memory reaches the next one."""
    cuda, t = kind
    rng = np.random.default_rng(12)
    for n, vocab in ((30, 30000), (3, 200000), (600, 4200), (1, 900), (30, 30000), (12, 65536)):
        x, u = logits(rng, n, vocab), rng.random(n)
        check(cuda, t, x, u, np.full(n, 0.9), some(rng, n, 40, 0), some(rng, n, 0.9, 1.0))
        check(cuda, t, x, u)


def test_without_memory_for_slices(monkeypatch):
    """The same tokens from one workgroup a row where the memory that slices take is not to be had (fp32: host data in 16 bits takes such memory itself)."""
    cuda, rng = CudaDnn(0), np.random.default_rng(13)
    n, vocab = 30, 30011
    x, u = stored(logits(rng, n, vocab), "f32"), rng.random(n)
    args = [np.full(n, 0.9), some(rng, n, 40, 0), some(rng, n, 0.9, 1.0)]
    want = draw(cuda, "f32", x, u, *args)
    monkeypatch.setenv("MYCAFFE_HIP_SCRATCH_LIMIT", "20000")
    small = CudaDnn(0)
    got = draw(small, "f32", x, u, *args)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    for c in (cuda, small):
        c.Dispose()
