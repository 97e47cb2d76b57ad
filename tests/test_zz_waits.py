"""Collected behind every other GPU test: none of the attention kernels' waits has run out in any of them."""
import pytest

pytestmark = pytest.mark.gpu


def test_no_block_gave_up(ops):
    assert ops.attn_gave_up() == 0
