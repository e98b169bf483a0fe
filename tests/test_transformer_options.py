"""Options of the Transformer that do not go together are refused, not dropped."""
import pytest

from tsplit_b200.models import transformer

SIZES = dict(vocab_size=20, d_model=16, num_heads=2, d_ff=16, num_blocks=1, maxlen1=5, maxlen2=5, batch_size=2)


def test_attention_across_has_no_dropout():
    with pytest.raises(ValueError, match="dropout"):
        transformer(**SIZES, cross_attention=True, dropout_rate=0.1)
    assert transformer(**SIZES, cross_attention=True).hp.cross_attention
    assert not transformer(**SIZES, dropout_rate=0.1).hp.cross_attention
