"""The causal attention layer with norms of queries and keys: its training step in both base types, and inference of many sequences over pages."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn, CudaDnnDouble
from mycaffe_amd.layers import Blob, CausalSelfAttentionLayer, PagedSequences, TransformerBlockLayer
from tests.conftest import BF16_RTOL, FP32_RTOL, assert_close, bf16_round

pytestmark = pytest.mark.gpu


def blob(cuda, values, half=False):
    b = Blob(cuda, values.shape, half)
    b.mutable_cpu_data = values
    return b


def weights(rng, C, hs):
    return dict(w_attn=rng.standard_normal((3 * C, C)) / np.sqrt(C), b_attn=0.1 * rng.standard_normal(3 * C), w_proj=rng.standard_normal((C, C)) / np.sqrt(C),
                b_proj=0.1 * rng.standard_normal(C), w_qnorm=1 + 0.2 * rng.standard_normal(hs), w_knorm=1 + 0.2 * rng.standard_normal(hs))


def step(cuda, w, x, dy, H, rope, sdpa, backward=True):
    """output, gradient of the input, gradients of the parameters"""
    B, T, C = x.shape
    layer = CausalSelfAttentionLayer(cuda, H, C, T, True, sdpa, rope, training=True, qk_norm=True)
    bx, top = blob(cuda, x), Blob(cuda)
    layer.Setup(bx, *w.values())
    layer.Forward(bx, top)
    y = top.mutable_cpu_data
    if not backward:
        return y
    params = layer.c_attn.blobs + layer.c_proj.blobs + layer.norms
    top.mutable_cpu_diff = dy
    for p in params:
        cuda.set(p.count(), p.gpu_diff, 0.0)
    layer.Backward(top, bx)
    return y, bx.mutable_cpu_diff, [p.mutable_cpu_diff for p in params]


@pytest.mark.parametrize("sdpa", [False, True])
@pytest.mark.parametrize("rope", [False, True])
def test_training_step(rope, sdpa):
    """gradients in double against central differences of the layer's own forward pass, along random directions; fp32 against double"""
    rng = np.random.default_rng(1)
    B, T, H, hs = 2, 9, 3, 16
    C = H * hs
    w, x, dy = weights(rng, C, hs), rng.standard_normal((B, T, C)), rng.standard_normal((B, T, C))
    cuda = CudaDnnDouble(0)
    y, dx, grads = step(cuda, w, x, dy, H, rope, sdpa)
    names = ["w_attn", "b_attn", "w_proj", "b_proj", "w_qnorm", "w_knorm"]
    for name, grad in [("x", dx)] + list(zip(names, grads)):
        d = rng.standard_normal(grad.shape)
        value = []
        for h in (1e-5, -1e-5):
            if name == "x":
                value.append((step(cuda, w, x + h * d, dy, H, rope, sdpa, False) * dy).sum())
            else:
                value.append((step(cuda, dict(w, **{name: w[name] + h * d.reshape(w[name].shape)}), x, dy, H, rope, sdpa, False) * dy).sum())
        # the difference: third derivatives times 1e-10, and 2^-53 of a sum of some 10^3 terms over 1e-5
        assert abs((value[0] - value[1]) / 2e-5 - (grad * d).sum()) <= 1e-6 * np.abs(grad * d).sum(), name
    cuda.Dispose()
    f = CudaDnn(0)
    yf, dxf, gf = step(f, w, np.float32(x), np.float32(dy), H, rope, sdpa)
    for a, b in [(yf, y), (dxf, dx)] + list(zip(gf, grads)):
        assert_close(a, b, FP32_RTOL)
    f.Dispose()


def test_block_with_norms():
    """a Llama-style block that trains with them: its attention's norm weights get gradients, and they are those of differences"""
    rng = np.random.default_rng(2)
    B, T, H, C, hid = 1, 6, 2, 32, 48
    x, dy = rng.standard_normal((B, T, C)), rng.standard_normal((B, T, C))
    p = dict(attn_weight=rng.standard_normal((3 * C, C)) / 6, attn_proj_weight=rng.standard_normal((C, C)) / 6, fc_weight=rng.standard_normal((hid, C)) / 6,
             fc2_weight=rng.standard_normal((hid, C)) / 6, proj_weight=rng.standard_normal((C, hid)) / 6, rms1_weight=np.ones(C), rms2_weight=np.ones(C),
             attn_qnorm_weight=1 + 0.2 * rng.standard_normal(C // H), attn_knorm_weight=1 + 0.2 * rng.standard_normal(C // H))
    cuda = CudaDnnDouble(0)

    def run(p, backward=False):
        layer = TransformerBlockLayer(cuda, H, C, T, "silu", False, 1e-5, True, training=True, enable_llama_style_head=True, hidden_dim=hid, qk_norm=True)
        bx, top = blob(cuda, x), Blob(cuda)
        layer.Setup(bx, p)
        layer.Forward(bx, top)
        y = top.mutable_cpu_data
        if backward:
            top.mutable_cpu_diff = dy
            for n in layer.attn1.norms:
                cuda.set(n.count(), n.gpu_diff, 0.0)
            layer.Backward(top, bx)
            return [n.mutable_cpu_diff for n in layer.attn1.norms]
        return (y * dy).sum()
    for name, grad in zip(("attn_qnorm_weight", "attn_knorm_weight"), run(p, True)):
        d = rng.standard_normal(grad.shape)
        diff = (run(dict(p, **{name: p[name] + 1e-5 * d})) - run(dict(p, **{name: p[name] - 1e-5 * d}))) / 2e-5
        assert abs(diff - (grad * d).sum()) <= 1e-6 * np.abs(grad * d).sum()
    cuda.Dispose()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rope,norm", [(True, True), (True, False), (False, False)])
def test_serving(half, rope, norm):
    """Three sequences that begin, grow by chunks and single tokens and end at different times: every row is the one of a pass over its whole sequence."""
    rng = np.random.default_rng(3)
    H, hs, ps, width = 4, 64, 16, 8
    C = H * hs
    cuda = CudaDnn(0)
    layer = CausalSelfAttentionLayer(cuda, H, C, width * ps, True, True, rope, half=half, qk_norm=norm)
    w = weights(rng, C, hs)
    one = blob(cuda, np.zeros((1, 1, C)), half)
    layer.Setup(one, *[np.float32(v) for v in w.values()][:6 if norm else 4])
    data = {n: np.float32(rng.standard_normal((1, t, C))) for n, t in (("a", 100), ("b", 45), ("c", 70))}
    if half:
        data = {n: bf16_round(v) for n, v in data.items()}
    want = {}
    for n, v in data.items():
        top = Blob(cuda, half=half)
        layer.Forward(blob(cuda, v, half), top)
        want[n] = top.mutable_cpu_data[0]
    seqs, top = PagedSequences(cuda, 14, ps, width), Blob(cuda, half=half)
    plans = [{"a": 60}, {"a": 1, "b": 30}, {"b": 1, "a": 38}, {"a": 1, "b": 14}, None, {"c": 68}, {"c": 1}, {"c": 1}]
    got = {n: [] for n in data}
    for plan in plans:
        if plan is None:
            seqs.End("a")
            seqs.End("b")
            continue
        rows = np.concatenate([data[n][0, seqs.length(n):seqs.length(n) + k] for n, k in plan.items()])
        seqs.Step(plan)
        layer.ForwardPaged(blob(cuda, rows[None], half), seqs, top)
        y, at = top.mutable_cpu_data[0], 0
        for n, k in plan.items():
            got[n].append(y[at:at + k])
            at += k
    # both are within the bar of what is right
    for n in data:
        assert_close(np.concatenate(got[n]), want[n], 2 * (BF16_RTOL if half else FP32_RTOL), n)
    with pytest.raises(ValueError):
        layer.ForwardPaged(blob(cuda, np.zeros((1, 7, C)), half), seqs, top)
    cuda.Dispose()
