"""What the C entries of the model operators refuse before any CUDA call, beside test_operators_cpu.py."""
import pytest

from test_operators_cpu import qk
from test_operators_cpu import window as window_block


@pytest.mark.parametrize('order', [-1, 2, 7])
def test_qk_norm_entry_refuses_an_unknown_order(order):
    """Such an order was taken for norm, then rotate."""
    from noise_b200 import _lib
    assert _lib.load().noise_qk_norm_rope(qk(_lib.QK_NORM, order=order, q=1 << 22, k=1 << 23, ko=1 << 24, rope=1 << 25), 0, None, 0, None) == 1


@pytest.mark.parametrize('B,Tk,H,Hk,D,window,wide,portable', [
    (1, 17001, 4, 2, 64, 17001, 16, 8), (2, 9001, 20, 1, 96, 8990, 16, 8), (1, 65536, 64, 8, 128, 65536, 16, 8),
    (1, 4096, 8, 8, 128, 4096, 8, 8), (1, 2048, 8, 8, 64, 1024, 8, 8), (64, 8192, 32, 8, 128, 4096, 1, 1),
    (1, 1, 1, 1, 64, 0, 1, 1), (1 << 10, 65536, 8, 8, 128, 65536, 1, 1),
])
def test_token_clusters_stay_within_what_the_device_places(B, Tk, H, Hk, D, window, wide, portable):
    """Clusters of 16 CTAs are not placed by every device: without them such a call has 8, and no other call changes."""
    from noise_b200 import _lib
    a = window_block(_lib.WINDOW, B=B, Tq=1, Tk=Tk, H=H, Hk=Hk, D=D, window=window, lengths=1 << 20,
                     qs=(H * D, H * D, D), ks=(Tk * Hk * D, Hk * D, D), vs=(Tk * Hk * D, Hk * D, D))
    count = _lib.load().noise_window_token_ctas
    assert count(a, 148, 16) == wide and count(a, 148, 8) == portable
    assert count(a, 0, 16) == -1 and count(window_block(_lib.WINDOW, H=3, lengths=1 << 20), 148, 16) == -1
