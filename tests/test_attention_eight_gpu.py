"""Attention for training with five to eight queries per head on sequences too long for groups of four: one group of
eight rows.  The comparison of test_attention_small_gpu."""
import pytest

from test_attention_small_gpu import test_sizes as compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("size", [(2, 8, 5, 3000), (2, 16, 8, 1000), (2, 8, 7, 2049), (1, 8, 6, 8193)], ids=str)
def test_sizes(size, masked):
    compare(size, masked)
