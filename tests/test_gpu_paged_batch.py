"""Serving from state on the device: the plan of a step, keys and values into pages, attention behind a shared prefix, the draw of the next tokens, step after step."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn, CudaDnnDouble
from mycaffe_amd.layers import Blob, CausalSelfAttentionLayer, InnerProductLayer, PagedBatch
from oracle import serving_ref as S
from tests.conftest import BF16_RTOL, FP32_RTOL, assert_close, bf16_round
from tests.test_gpu_layer_paged import blob, weights
from tests.test_gpu_sample import off

pytestmark = pytest.mark.gpu

# new tokens of five places, places that begin behind others, groups that share from here on
STEPS = [dict(new=[70, 0, 0, 0, 0]),
         dict(new=[1, 8, 3, 0, 20], begin={1: (0, 64), 2: (0, 70)}, share=([0, 3], [64])),
         dict(new=[1, 1, 1, 0, 1]),
         dict(new=[1, 1, -1, 40, 1]),
         dict(new=[1, 1, 5, 1, 1], begin={2: (0, 48)}, share=([0, 3], [48])),
         dict(new=[1, 1, 1, 1, 90]),                # the last one does not fit: it waits
         dict(new=[1, 1, 1, -1, 60]),               # it does, with the pages of the one that ends
         dict(new=[1, 1, 1, 0, 1], share=([0, 1, 3], [0, 48])),
         dict(new=[0, 1, 1, 30, 1], share=()),
         dict(new=[1, 1, 1, 1, 1], share=([0, 3, 5], [48, 0]))]


@pytest.mark.parametrize("width", [10, 1000])        # tables wide enough for attention to take prefixes by themselves, and not
@pytest.mark.parametrize("kind", ["f32", "bf16", "f64"])
def test_steps_together(kind, width):
    rng = np.random.default_rng(3)
    half, H, hs, page, B, rows, pages, vocab = kind == "bf16", 4, 64, 16, 5, 96, 17, 331
    C = H * hs
    cuda = (CudaDnnDouble if kind == "f64" else CudaDnn)(0)
    real = np.float64 if kind == "f64" else np.float32
    value = (lambda v: bf16_round(np.float32(v))) if half else real
    layers = [CausalSelfAttentionLayer(cuda, H, C, 256, True, True, rope, half=half, qk_norm=norm) for rope, norm in ((True, True), (True, False))]
    embed = value(rng.standard_normal((vocab, C)))
    one = blob(cuda, np.zeros((1, 1, C), real), half)
    for layer in layers:
        w = weights(rng, C, hs)
        layer.Setup(one, *[real(v) for v in w.values()][:6 if layer.qk_norm else 4])
    head = InnerProductLayer(cuda, vocab, False, 2, half)
    head.Setup(one, real(rng.standard_normal((vocab, C)) / 4))
    served = PagedBatch(cuda, B, rows, pages, page, width)
    tops, logits = [Blob(cuda, half=half) for _ in layers], Blob(cuda, half=half)
    heat, k, p, m = (np.array(v, real) for v in ([0.8, 1.0, 0.0, 1.3, 0.9], [0, 40, 5, 200, 0], [0.9, 1.0, 0.5, 0.95, 0.8], [0, 0, 0, 0.02, 0]))
    settings, u = [blob(cuda, v) for v in (heat, k, p, m)], Blob(cuda, (B,))
    text = [[] for _ in range(B)]                   # tokens of the sequence of every place, and its rows of every layer that were computed for it
    known = [[[] for _ in layers] for _ in range(B)]
    lens, table, free, shared, origin = np.zeros(B), np.full((B, width), -1.0), np.concatenate([[pages], np.arange(pages - 1, -1, -1)]), np.zeros(B), np.full(B, -1.0)
    drawn = [[] for _ in range(B)]
    waited = 0
    done = []

    def end(b):
        done.append((text[b], known[b]))
        text[b], known[b] = [], [[] for _ in layers]

    for step in STEPS:
        if "begin" in step:
            served.Begin(step["begin"])
            for b, (other, n) in step["begin"].items():
                origin[b], shared[b] = other, n
        if "share" in step:
            served.Share(*step["share"])
        new = np.array(step["new"])
        served.Step(new)
        before = lens
        want = S.plan(new, lens, table, free, rows, page, origin, shared)
        lens, table, free, shared = np.array(want["lens"]), want["table"], want["free"], np.array(want["shared"], float)
        assert np.array_equal(served.lens.mutable_cpu_data, lens) and np.array_equal(served.table.mutable_cpu_data, table)
        assert np.array_equal(served.free.mutable_cpu_data[:1 + int(free[0])], free[:1 + int(free[0])])
        assert np.array_equal(served.starts.mutable_cpu_data, want["starts"]) and np.array_equal(served.last.mutable_cpu_data, want["last"])
        assert np.array_equal(served.positions.mutable_cpu_data[:want["starts"][-1]], want["positions"])
        starts = np.array(want["starts"])
        x = np.full((1, rows, C), np.nan, real)     # rows behind the last one are nobody's
        for b in range(B):
            n = starts[b + 1] - starts[b]
            if new[b] < 0:
                end(b)
                drawn[b] = []
            waited += new[b] > 0 and n == 0
            if n == 0:
                continue
            if before[b] == 0 and shared[b]:
                text[b] = text[int(origin[b])][:int(shared[b])]
                for i, _ in enumerate(layers):
                    known[b][i].append((int(shared[b]), None))
            fresh = (drawn[b] + list(rng.integers(0, vocab, n)))[:n]
            x[0, starts[b]:starts[b + 1]] = embed[fresh]
            text[b] = text[b] + [int(f) for f in fresh]
            assert len(text[b]) == lens[b]
        bx = blob(cuda, x, half)
        for layer, top in zip(layers, tops):
            layer.ForwardPaged(bx, served, top)
        head.Forward(tops[0], logits)
        u.mutable_cpu_data = rng.random(B).astype(real)
        served.Sample(logits, u, *settings)
        z, numbers = np.asarray(logits.mutable_cpu_data, np.float64).reshape(rows, vocab), np.asarray(u.mutable_cpu_data, np.float64)
        ids, logs = served.ids.mutable_cpu_data, served.logprobs.mutable_cpu_data
        for i, top in enumerate(tops):
            y = top.mutable_cpu_data.reshape(rows, C)
            for b in range(B):
                known[b][i].append((starts[b + 1] - starts[b], y[starts[b]:starts[b + 1]]))
        for b in range(B):
            if want["last"][b] < 0:
                assert ids[b] == -1 and logs[b] == 0
                continue
            token, log, near = S.sample(z[want["last"][b]], numbers[b], float(heat[b]), float(k[b]), float(p[b]), float(m[b]))
            assert near > off(vocab) and ids[b] == token
            assert abs(logs[b] - log) <= (0 if kind == "f64" else 2.0 ** -24) * abs(log) + off(vocab) + 2.0 ** -48 * max(1.0, abs(log))
            drawn[b] = [int(ids[b])]
    assert waited == 1
    for b in range(B):
        end(b)
    # every row is the one of a pass over its whole sequence; both are within the bar of what is right.  In the double base type the pass rotates by
    # angles of fp32: position times a frequency below 0.75 that is off by some 2^-24 of itself, so off by at most 128 * 0.75 * 3 * 2^-24 = 1.7e-5 where the exact
    # angle is used over pages; the bar of an fp32 pass, which rotates by the same angles and rounds everything else too, holds that
    bar = 2 * BF16_RTOL if half else 2 * FP32_RTOL if kind == "f32" else FP32_RTOL
    for words, got in done:
        if not words:
            continue
        for layer, parts in zip(layers, got):
            top = Blob(cuda, half=half)
            layer.Forward(blob(cuda, embed[words][None], half), top)
            whole, at = top.mutable_cpu_data.reshape(len(words), C), 0
            for n, part in parts:
                if part is not None and n:
                    assert_close(part, whole[at:at + n], bar)
                at += n
            assert at == len(words)
    served.Dispose()
    cuda.Dispose()
