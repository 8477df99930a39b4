"""What the C entries of the model operators refuse before any CUDA call, beside test_operators_cpu.py."""
import pytest

from test_operators_cpu import qk


@pytest.mark.parametrize('order', [-1, 2, 7])
def test_qk_norm_entry_refuses_an_unknown_order(order):
    """Such an order was taken for norm, then rotate."""
    from noise_b200 import _lib
    assert _lib.load().noise_qk_norm_rope(qk(_lib.QK_NORM, order=order, q=1 << 22, k=1 << 23, ko=1 << 24, rope=1 << 25), 0, None, 0, None) == 1
