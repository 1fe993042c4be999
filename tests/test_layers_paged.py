"""What the layers keep for serving over pages, and what they refuse, without a device."""
import pytest

from mycaffe_amd.layers import TransformerBlockLayer
from tests.test_layers_kept import Context


def test_norms_of_heads_are_the_causal_attention_s():
    with pytest.raises(ValueError):
        TransformerBlockLayer(Context(), 2, 16, 8, block_type="encoder", qk_norm=True)
    TransformerBlockLayer(Context(), 2, 16, 8, block_type="encoder")
    assert TransformerBlockLayer(Context(), 2, 16, 8, qk_norm=True).attn1.qk_norm
