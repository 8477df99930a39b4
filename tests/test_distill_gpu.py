"""The distillation loss and its gradient against float64 (oracle/operators.py).

Tolerances: the kernel's s has at most 4 roundings of its size (and tanh's 2 ulp), exp and log 2 ulp each, the
difference s - lse one rounding of their size: E = 2^-20 + 12 * 2^-24 max|s| bounds the relative error of
every exp(s - lse) and p_k, and sums of positive terms add at most (V / 1024 + 16) * 2^-24. The loss is off by at
most temperature^2 times E plus 2^-22 of itself; a gradient by |dloss| temperature (q + p) E, by 4 * 2^-24 of
(q + p) for the soft cap's slope, and by its rounding to the type, u = eps / 2 of its value."""
import pytest
import torch

from oracle import operators as oo

pytestmark = pytest.mark.gpu
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}

CASES = [  # N, V, K, dtype, teacher, ids, temperature, softcap, layout
    (5, 1000, 8, 'fp32', 'fp32', torch.int32, 1.0, 0.0, 'plain'),
    (3, 4096, 32, 'fp32', 'fp32', torch.int32, 1.0, 15.0, 'plain'),
    (7, 1237, 16, 'bf16', 'bf16', torch.int64, 2.0, 0.0, 'plain'),
    (4, 5003, 100, 'fp16', 'fp32', torch.int32, 0.7, 30.0, 'plain'),
    (1, 1, 1, 'fp32', 'fp32', torch.int64, 1.0, 0.0, 'plain'),
    (9, 3, 5, 'bf16', 'fp16', torch.int32, 1.0, 5.0, 'plain'),
    (2, 131071, 64, 'bf16', 'fp32', torch.int32, 1.0, 15.0, 'plain'),
    (3, 70001, 1024, 'fp32', 'fp32', torch.int32, 4.0, 0.0, 'plain'),
    (6, 501, 7, 'bf16', 'fp32', torch.int64, 1.0, 0.0, 'view'),
    (4, 300, 256, 'fp32', 'fp32', torch.int32, 1.0, 2.0, 'view'),
    (600, 777, 3, 'bf16', 'fp32', torch.int32, 1.0, 0.0, 'plain'),
    (1500, 777, 3, 'bf16', 'fp32', torch.int32, 1.0, 0.0, 'plain'),  # more rows than CTAs of four warps: one warp a row
    (1300, 130, 70, 'fp32', 'bf16', torch.int64, 1.0, 15.0, 'view'),
    (1201, 5, 2, 'fp16', 'fp16', torch.int32, 2.0, 3.0, 'plain'),
]


def build(case):
    N, V, K, dt, tdt, idt, tau, cap, layout = case
    g = torch.Generator().manual_seed(N * 131 + V + K)
    z = torch.randn(N, V, generator=g, dtype=torch.float64).mul_(4).to(DT[dt])
    ids = torch.randint(0, V, (N, K), generator=g)  # ids may repeat
    if K > 2:
        ids[:, 1] = ids[:, 0]
        ids[0, K - 1], ids[N - 1, K // 2] = -1, V  # absent
    t = torch.randn(N, K, generator=g).mul_(3).to(DT[tdt])
    if N > 2:
        ids[1] = -5                   # a row without entries
        t[2] = torch.finfo(DT[tdt]).min  # equal shares at the type's lowest value
    if N > 3:
        t[3] = -torch.inf             # a row whose entries hold nothing
    if N > 4 and K > 1:
        t[4, 1:] = -torch.inf
        z[4, (int(ids[4, 0]) + 1) % V] = -torch.inf if V > 1 else 0
    up = torch.randn(N, generator=g)
    dev = [z, ids.to(idt), t]
    if layout == 'view':  # rows of a wider matrix, from an odd column
        wide = torch.full((N, V + 5), float('nan'), dtype=DT[dt], device='cuda')
        wide[:, 3:3 + V] = z.cuda()
        cols = torch.zeros(N, 2 * K, dtype=idt, device='cuda')
        cols[:, ::2] = dev[1].cuda()
        dev = [wide[:, 3:3 + V], cols[:, ::2], t.cuda()]
    else:
        dev = [x.cuda() for x in dev]
    return z, ids, t, up, dev, dict(temperature=tau, softcap=cap)


def expected(z, ids, t, tau, cap):
    loss, q, p, slope = oo.distill(z, ids, t, tau, cap)
    s = (cap * torch.tanh(z.double() / cap) if cap else z.double()) / tau
    finite = torch.where(s.isfinite(), s.abs(), 0.0).amax(1, keepdim=True)
    finite = torch.maximum(finite, torch.where(t.double().abs() < 1e30, t.double().abs(), 0.0).amax(1, keepdim=True) / tau)
    E = 2.0 ** -20 + 12 * 2.0 ** -24 * finite + (z.shape[1] / 1024 + 16) * 2.0 ** -24
    return loss, q, p, slope, E


def check_grad(got, up, q, p, slope, E, tau, dtype):
    want = up.double()[:, None] * tau * (q - p) * slope
    u = torch.finfo(dtype).eps / 2
    tol = up.double().abs()[:, None] * tau * (q + p) * (E * slope + 4 * 2.0 ** -24 * 4) + u * want.abs()
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.double().cpu() - want).abs()
    assert (err <= tol + 1e-37).all(), (err - tol).max().item()


@pytest.mark.parametrize('case', CASES)
def test_loss_and_gradient(case):
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    z, ids, t, up, dev, kw = build(case)
    tau, cap = kw['temperature'], kw['softcap']
    want, q, p, slope, E = expected(z, ids, t, tau, cap)
    loss, lse = distill_loss(*dev, **kw)
    ok = want.isfinite()
    tol = tau * tau * E[:, 0] * 2 + 2.0 ** -22 * want.abs()
    assert ((loss.double().cpu() - want).abs() <= tol)[ok].all(), ((loss.double().cpu() - want).abs() - tol)[ok].max()
    assert torch.equal(loss.cpu()[~ok].double(), want[~ok])
    both = distill_loss_grad(*dev, dloss=up.cuda(), **kw)
    assert ((both[0].double().cpu() - want).abs() <= tol)[ok].all()
    check_grad(both[1], up, q, p, slope, E, tau, z.dtype)
    check_grad(distill_backward(up.cuda(), *dev, lse, **kw), up, q, p, slope, E, tau, z.dtype)
    check_grad(distill_loss_grad(*dev, **kw)[1], torch.ones_like(up), q, p, slope, E, tau, z.dtype)
    again = distill_loss_grad(*dev, dloss=up.cuda(), **kw)
    assert torch.equal(both[0], again[0]) and torch.equal(both[1], again[1])
    if case[8] == 'view':
        assert dev[0].isfinite().all() or case[0] > 4  # the view was only read


@pytest.mark.parametrize('N,V,K', [(2, 200003, 180), (400, 3001, 90), (1400, 1201, 200)])
def test_entries_that_repeat_or_meet_in_the_table(N, V, K):
    """More than 32 entries: ids that all fall on one place of the table of ids, each named twice and far apart; one id
    that every entry names; ids that follow one another. Twice, with equal bits."""
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    places = 64
    while places < 2 * K:
        places *= 2
    every = torch.arange(V)
    place = ((every * 2654435769) % 2 ** 32 >> 16) % places
    few = every[place == place.bincount().argmax()][:K // 2]
    g = torch.Generator().manual_seed(K)
    z, t = torch.randn(N, V, generator=g).mul_(3), torch.randn(N, K, generator=g)
    ids = torch.randint(0, V, (N, K), generator=g)
    ids[0] = torch.cat([few, few, every[:K]])[:K]
    ids[1] = 77
    if N > 2:
        ids[2] = every[100:100 + K]
    up = torch.rand(N, generator=g)
    dev = [x.cuda() for x in (z, ids.int(), t)]
    loss, lse = distill_loss(*dev)
    want, q, p, slope, E = expected(z, ids, t, 1.0, 0.0)
    for call in (lambda: distill_loss_grad(*dev, dloss=up.cuda())[1], lambda: distill_backward(up.cuda(), *dev, lse)):
        got = call()
        check_grad(got, up, q, p, slope, E, 1.0, z.dtype)
        assert torch.equal(got, call())


def test_gradient_matches_differences():
    """Central differences of the float64 loss: truncation h^2 ~ 1e-8, so 1e-6 holds beside the kernel's fp32."""
    from noise_b200.distill import distill_loss_grad
    g = torch.Generator().manual_seed(2)
    z, ids, t = torch.randn(3, 40, generator=g) * 3, torch.randint(0, 40, (3, 6), generator=g), torch.randn(3, 6, generator=g)
    for tau, cap in ((1.0, 15.0), (2.0, 0.0)):
        grad = distill_loss_grad(z.cuda(), ids.cuda(), t.cuda(), temperature=tau, softcap=cap)[1].cpu()
        for j in range(40):
            e = torch.zeros(3, 40, dtype=torch.float64)
            e[:, j] = 1e-4
            d = (oo.distill(z.double() + e, ids, t, tau, cap)[0] - oo.distill(z.double() - e, ids, t, tau, cap)[0]) / 2e-4
            assert (d - grad[:, j].double()).abs().max() < 2e-6


def test_special_logits():
    from noise_b200.distill import distill_loss, distill_loss_grad
    z = torch.zeros(4, 64, device='cuda')
    z[1, 3] = float('nan')
    z[2, 10] = -torch.inf  # the student gives a target no mass
    z[3] = -torch.inf
    z[3, 20] = 1.0
    ids = torch.tensor([[1, 2], [1, 2], [10, 2], [20, -1]], device='cuda')
    t = torch.zeros(4, 2, device='cuda')
    loss, _ = distill_loss(z, ids, t)
    assert loss[0].isfinite() and loss[1].isnan() and loss[2] == torch.inf and loss[3] == 0
    _, grad = distill_loss_grad(z, ids, t)
    assert grad[1].isnan().all() and grad[2, 10] == -0.5 and (grad[3] == 0).all()
    loss, _ = distill_loss(z[:0], ids[:0], t[:0])
    assert loss.shape == (0,)
    assert distill_loss_grad(z[:0], ids[:0], t[:0])[1].shape == (0, 64)


def test_streams_and_graph_replay():
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    g = torch.Generator(device='cuda').manual_seed(4)
    z = torch.randn(12, 9001, device='cuda', generator=g)
    ids = torch.randint(0, 9001, (12, 20), device='cuda', generator=g)
    t, up = torch.randn(12, 20, device='cuda', generator=g), torch.rand(12, device='cuda', generator=g)
    distill_loss_grad(z, ids, t), distill_backward(up, z, ids, t, distill_loss(z, ids, t)[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse = distill_loss(z, ids, t)
        out = (loss, distill_backward(up, z, ids, t, lse), *distill_loss_grad(z, ids, t))
    z.normal_(generator=g)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, lse = distill_loss(z, ids, t)
        want = (loss, distill_backward(up, z, ids, t, lse), *distill_loss_grad(z, ids, t))
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)
