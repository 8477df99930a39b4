"""The distillation calls on rows without an entry between rows with entries, on logits far beyond the soft cap, and
on rows that a mask covers.

Tolerances as in test_distill_gpu.py where nothing else is said."""
import pytest
import torch

from oracle import operators as oo
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


@pytest.mark.parametrize('cap,tau', [(15.0, 1.0), (2.0, 1.0), (20.0, 0.5), (30.0, 0.5)])  # c / tau up to 40, and beyond
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradient_far_beyond_the_soft_cap(cap, tau, dtype):
    """The slope of logits of 3 to 10 soft caps is 1e-2 to 1e-8, and as exact as any: with u = 2^-24, z / c is off by 2 u of
    itself and the exponent 2 |z| / c by 2 u more, so the slope 4 e / (1 + e)^2 by 8 |z| / c u and the roundings of e, of
    1 / (1 + e) twice and of the products, 20 u. What the exponentials flush to zero is below 2^-126."""
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    g = torch.Generator().manual_seed(int(cap))
    N, V, K = 6, 2003, 7
    far = (3 + 7 * torch.rand(N, V, generator=g)) * (torch.randint(0, 2, (N, V), generator=g) * 2 - 1)
    far[1] = far[1].abs()
    far[2] = -far[2].abs()
    far[3, ::2] *= 0.1
    far[4] = 2 * far[2]  # a whole row at the lower end: every exp(s) is as small as it gets, and slopes go down to 1e-17
    z = (far * cap).to(dtype)
    ids, t, up = torch.randint(0, V, (N, K), generator=g), torch.randn(N, K, generator=g), torch.randn(N, generator=g)
    _, q, p, _, E = expected(z, ids, t, tau, cap)
    slope = 1 / torch.cosh(z.double() / cap).square()  # the oracle's 1 - tanh^2 has no digits left at 20 caps
    scale = up.double().abs()[:, None] * tau
    want = up.double()[:, None] * tau * (q - p) * slope
    S = (8 * z.double().abs() / cap + 20) * 2.0 ** -24
    tol = scale * slope * ((q + p) * E + (q - p).abs() * S) + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -126 * (1 + scale)
    dev = [x.cuda() for x in (z, ids, t)]
    kw = dict(softcap=cap, temperature=tau)
    _, lse = distill_loss(*dev, **kw)
    for got in (distill_loss_grad(*dev, dloss=up.cuda(), **kw)[1], distill_backward(up.cuda(), *dev, lse, **kw)):
        err = (got.double().cpu() - want).abs()
        assert (err <= tol).all(), ((err / want.abs().clamp(min=1e-300))[err > tol].max(), (err > tol).sum())


@pytest.mark.parametrize('mask', ['lowest', -1e30, -1e10, -60000.0])
@pytest.mark.parametrize('N,V,dtype,tau', [(6, 2003, torch.float32, 1.0), (6, 70001, torch.bfloat16, 0.5),
                                           (1500, 333, torch.float32, 2.0), (1500, 333, torch.float16, 1.0)])
def test_rows_masked_as_a_whole(mask, N, V, dtype, tau):
    """Logits that are a mask's value, or the type's lowest, in a whole row, in all but a few columns, and beside half of it:
    the row is that of its differences, and a row whose loss has no weight gets zeros, not NaN. The differences between
    columns that count are 0 or of normal size, so the relative error is that of normal logits:
    E = 2^-20 + 12 * 2^-24 * 20 / temperature + (V / 1024 + 16) 2^-24."""
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    mask = torch.finfo(dtype).min if mask == 'lowest' else max(mask, torch.finfo(dtype).min)
    g = torch.Generator().manual_seed(V)
    K = 5
    z = torch.randn(N, V, generator=g).mul_(2).to(dtype)
    z[0::6] = mask
    z[1::6, 3:] = mask                      # its entries lie on masked columns, all but one
    z[2::6, 1::2] = mask
    z[3::6] = mask
    z[4::6], z[4::6, ::2] = mask, mask / 2  # half of the row counts
    z[5::6, 5:] = -torch.inf
    z[5::6, :5] = mask
    ids, t, up = torch.randint(0, V, (N, K), generator=g), torch.randn(N, K, generator=g), torch.randn(N, generator=g)
    ids[1::6, 0] = 1
    ids[4::6] = ids[4::6] // 2 * 2          # (an entry that does not count has a loss beyond the type)
    ids[5::6] = ids[5::6] % 5
    up[3::6] = 0.0
    want, q, p, _ = oo.distill(z, ids, t, tau)
    E = 2.0 ** -20 + 12 * 2.0 ** -24 * 20 / tau + (V / 1024 + 16) * 2.0 ** -24
    dev = [x.cuda() for x in (z, ids, t)]
    loss, lse = distill_loss(*dev, temperature=tau)
    both, grad = distill_loss_grad(*dev, dloss=up.cuda(), temperature=tau)
    for got in (loss, both):
        got = got.double().cpu()
        fits, beyond = want < 3.4e38, want > 3.41e38  # fp32 ends at 3.403e38
        assert ((got - want).abs() <= 2 * tau * tau * E + 2.0 ** -20 * want.abs())[fits].all()
        assert (got[beyond] == torch.inf).all()
    slope = torch.ones_like(q)
    for got in (grad, distill_backward(up.cuda(), *dev, lse, temperature=tau)):
        check_grad(got, up, q, p, slope, E, tau, dtype)
        assert (got[3::6] == 0).all()


@pytest.mark.parametrize('N,V,dtype', [(6, 501, torch.bfloat16), (1300, 130, torch.float32), (3, 70001, torch.float16)])
def test_inputs_are_only_read(N, V, dtype):
    """Logits that are columns of a wider matrix: its bits stay, those around the view among them."""
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    g = torch.Generator().manual_seed(V)
    wide = torch.full((N + 2, V + 5), float('nan'), dtype=dtype, device='cuda')
    z = wide[1:-1, 3:3 + V]
    z.copy_(torch.randn(N, V, generator=g))
    ids, t = torch.randint(0, V, (N, 7), generator=g).cuda(), torch.randn(N, 7, generator=g).cuda()
    bits = {2: torch.int16, 4: torch.int32}[wide.element_size()]
    before = wide.view(bits).clone(), ids.clone(), t.clone()
    for cap in (0.0, 15.0):
        loss, lse = distill_loss(z, ids, t, softcap=cap)
        distill_loss_grad(z, ids, t, softcap=cap)
        distill_backward(torch.ones_like(loss), z, ids, t, lse, softcap=cap)
    assert torch.equal(wide.view(bits), before[0]) and torch.equal(ids, before[1]) and torch.equal(t, before[2])


@pytest.mark.parametrize('dtype,cap', [(torch.float32, 0.0), (torch.float32, 15.0), (torch.bfloat16, 0.0), (torch.float16, 50.0)])
@pytest.mark.parametrize('K', [3, 1024])
def test_the_longest_rows_that_one_pass_takes(dtype, cap, K):
    """noise_distill_max_vocab logits a row: a cluster of 8 CTAs whose shared memory is full."""
    from noise_b200 import _lib
    from noise_b200.distill import distill_loss, distill_loss_grad
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    V = int(_lib.load().noise_distill_max_vocab(code, int(cap > 0)))
    g = torch.Generator().manual_seed(K)
    wide = torch.randn(2, V + 1, generator=g).mul_(2).to(dtype)
    z = wide[:, 1:]  # from an element that is not 16-byte aligned
    ids, t, up = torch.randint(0, V, (2, K), generator=g), torch.randn(2, K, generator=g), torch.rand(2, generator=g) + 1
    want, q, p, slope, E = expected(z, ids, t, 1.0, cap)
    dev = [wide.cuda()[:, 1:], ids.cuda(), t.cuda()]
    loss, grad = distill_loss_grad(*dev, dloss=up.cuda(), softcap=cap)
    tol = 2 * E[:, 0] + 2.0 ** -22 * want.abs()
    assert ((loss.double().cpu() - want).abs() <= tol).all()
    assert ((distill_loss(*dev, softcap=cap)[0].double().cpu() - want).abs() <= tol).all()
    check_grad(grad, up, q, p, slope, E, 1.0, dtype)
