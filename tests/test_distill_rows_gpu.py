"""The distillation calls on rows that differ from their neighbours: rows without an entry between rows with entries.

Tolerances as in test_distill_gpu.py."""
import pytest
import torch

from test_distill_gpu import check_grad, expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('N,V,K,cap,dtype', [
    (3001, 4099, 5, 0.0, torch.float32),     # several CTAs of four warps after one another on each SM
    (4001, 1003, 40, 15.0, torch.bfloat16),  # one warp a row
    (7, 70001, 5, 0.0, torch.bfloat16),      # several CTAs a row
])
def test_gradient_alone_of_rows_without_entries_between_others(N, V, K, cap, dtype):
    """A row without entries leaves the gradient early, while the next row's CTA takes over its shared memory: the
    neighbours' gradients are those of their rows, every time."""
    from noise_b200.distill import distill_backward, distill_loss
    g = torch.Generator().manual_seed(N)
    z = torch.randn(N, V, generator=g).mul_(4).to(dtype)
    ids, t, up = torch.randint(0, V, (N, K), generator=g), torch.randn(N, K, generator=g), torch.randn(N, generator=g)
    ids[::2] = -1
    ids[1::4, 0] = V  # a row that only lacks its first entry
    dev = [x.cuda() for x in (z, ids, t)]
    loss, lse = distill_loss(*dev, softcap=cap)
    got = distill_backward(up.cuda(), *dev, lse, softcap=cap)
    assert (loss[::2] == 0).all() and (got[::2] == 0).all()
    for _ in range(5):
        assert torch.equal(distill_backward(up.cuda(), *dev, lse, softcap=cap), got)
    some = torch.arange(0, N, (N // 200) | 1)
    want, q, p, slope, E = expected(z[some], ids[some], t[some], 1.0, cap)
    check_grad(got[some.cuda()], up[some], q, p, slope, E, 1.0, dtype)
