"""What the layers keep for serving over pages, and what they refuse, without a device."""
import pytest

from mycaffe_amd.layers import Blob, CausalSelfAttentionLayer, PagedSequences, TransformerBlockLayer
from tests.test_layers_kept import Context


def serve(cuda, layers, seqs, C=16):
    x, y = Blob(cuda, (1, seqs.tokens, C)), Blob(cuda)
    for layer in layers:
        layer.ForwardPaged(x, seqs, y)


def attention(cuda, theta=10000.0, heads=2):
    layer = CausalSelfAttentionLayer(cuda, heads, 16, 32, enable_rotary_positional_embedding=True, rope_theta=theta, qk_norm=True)
    layer.Setup(Blob(cuda, (1, 1, 16)), None, None, None, None)
    return layer


def test_layers_share_the_angles_of_their_pages():
    cuda = Context()
    layers, seqs = [attention(cuda) for _ in range(3)], PagedSequences(cuda, 6, 4, 4)
    seqs.Step({"a": 5, "b": 1})
    serve(cuda, layers, seqs)
    ropes = lambda: sorted(h for h, kind in cuda.live.items() if kind == "rope")  # noqa: E731
    assert len(ropes()) == 1
    seqs.Step({"a": 1})
    serve(cuda, layers, seqs)
    assert len(ropes()) == 1
    # another base, another head size: their own; other sequences: theirs
    serve(cuda, [attention(cuda, theta=500.0)], seqs)
    serve(cuda, [attention(cuda, heads=4)], seqs)
    assert len(ropes()) == 3
    other = PagedSequences(cuda, 6, 4, 2)
    other.Step({"x": 2})
    serve(cuda, layers[:1], other)
    assert len(ropes()) == 4
    mine = ropes()[-1]
    seqs.Dispose()
    assert ropes() == [mine]
    seqs.Dispose()
    other.Dispose()
    assert not ropes()


def test_norms_of_heads_are_the_causal_attention_s():
    with pytest.raises(ValueError):
        TransformerBlockLayer(Context(), 2, 16, 8, block_type="encoder", qk_norm=True)
    TransformerBlockLayer(Context(), 2, 16, 8, block_type="encoder")
    assert TransformerBlockLayer(Context(), 2, 16, 8, qk_norm=True).attn1.qk_norm
