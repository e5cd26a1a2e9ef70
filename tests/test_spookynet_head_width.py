"""Softmax attention's heads hold up to 128 features on every device: a wider one is refused when the model is built."""
import pytest

from xnn_b200.models.spookynet import SpookyNet


def test_wide_heads_are_refused_at_once():
    for width, heads in ((129, 1), (256, 1), (512, 2)):
        with pytest.raises(ValueError, match="128"):
            SpookyNet(n_features=width, n_interactions=1, attention="softmax", attention_heads=heads, d4_dispersion=False)
    for width, heads, kind in ((128, 1, "softmax"), (256, 2, "softmax"), (256, 1, "exact")):
        assert SpookyNet(n_features=width, n_interactions=1, attention=kind, attention_heads=heads, d4_dispersion=False)
