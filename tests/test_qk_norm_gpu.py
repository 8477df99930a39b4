"""qk_norm_rope and its gradient against float64 (oracle/operators.py).

Tolerances: an output is rounded once to its type, u = eps / 2 of its value. What precedes is fp32: the
rotation (2 roundings a value), the row's mean (at most 16 + log2(16) additions deep, halved by the root), the
root (2 ulp) and the products after it (at most 6) stay below 32 * 2^-24 of the row's largest magnitude times
sqrt(2) (a rotation can cancel), taken as 48 * 2^-24. A gradient's parts are bounded by r max|g| sqrt(D), the
same count applies to them. A weight's gradient adds its rows in fp32, each thread at most 64 rows one after
the other in these sizes, then 3 + 8 + 32 levels: 128 * 2^-24 of the sum of the terms' magnitudes."""
import pytest
import torch

from oracle import operators as oo

pytestmark = pytest.mark.gpu
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
U32 = 2.0 ** -24


def rope_table(n, d, seed=0):
    ang = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    return torch.cat([ang.cos(), ang.sin()], 1).bfloat16().float()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def check_rows(got, want, dtype, floor):
    tol = half_step(dtype) * want.abs() + 48 * U32 * floor
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # its subnormal half step
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


CASES = [  # B, T, H, Hk, D, dtype, order, weights, positions, layout
    (2, 5, 8, 8, 64, 'bf16', 'rotate_norm', False, None, 'packed'),
    (1, 1, 1, 1, 16, 'fp32', 'rotate_norm', True, None, 'plain'),
    (3, 7, 6, 2, 96, 'fp32', 'norm_rotate', True, 'batch', 'packed'),
    (2, 33, 12, 4, 80, 'fp16', 'norm_rotate', True, 'row', 'plain'),
    (4, 1, 32, 8, 128, 'bf16', 'norm_rotate', True, 'batch', 'packed'),
    (1, 130, 5, 1, 256, 'bf16', 'rotate_norm', True, None, 'heads_first'),
    (2, 65, 3, 3, 48, 'bf16', 'norm_rotate', False, 'batch', 'plain'),
    (1, 2048, 7, 1, 32, 'fp16', 'rotate_norm', True, None, 'packed'),
    (2, 9, 4, 2, 64, 'bf16', 'rotate_norm', True, None, 'misaligned'),
    (3, 4, 4, 2, 64, 'fp32', 'rotate_norm', True, None, 'broadcast'),
]


def build(case):
    B, T, H, Hk, D, dt, order, weights, positions, layout = case
    dtype = DT[dt]
    g = torch.Generator().manual_seed(B * 1000 + T * 10 + D)

    def make(heads):
        x = torch.randn(B, T, heads, D, generator=g, dtype=torch.float64).mul_(2).to(dtype)
        return x

    q, k, dq, dk = make(H), make(Hk), make(H), make(Hk)
    if layout == 'broadcast':
        q, k = q[:, :1].expand(B, T, H, D), k[:, :1].expand(B, T, Hk, D)

    def place(x):
        if layout == 'heads_first':
            return x.cuda().transpose(1, 2).contiguous().transpose(1, 2)
        if layout == 'misaligned':
            flat = torch.empty(x.numel() + 1, dtype=dtype, device='cuda')
            flat[1:] = x.cuda().reshape(-1)
            return flat[1:].view(x.shape)
        if layout == 'broadcast':
            return x[:, :1].cuda().expand(x.shape)
        return x.cuda()

    if layout == 'packed':
        qkv = torch.cat([q, k, torch.full_like(k, float('nan'))], 2).cuda()
        qc, kc = qkv[:, :, :H], qkv[:, :, H:H + Hk]
    else:
        qc, kc = place(q), place(k)
    table = 4096 if T <= 2048 else T
    rope = rope_table(table, D)
    if positions == 'batch':
        pos = torch.randint(0, table, (B, T), generator=g, dtype=torch.int32)
    elif positions == 'row':
        pos = torch.randint(0, table, (T,), generator=g, dtype=torch.int32)
    else:
        pos = None
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)) for _ in range(2)) if weights else (None, None)
    c, s = oo.rotation(rope, (pos if pos is not None else torch.arange(T)).expand(B, T))
    kw = dict(positions=None if pos is None else pos.cuda(), order=order)
    if weights:
        kw.update(q_weight=wq.cuda(), k_weight=wk.cuda())
    return q, k, dq, dk, qc, kc, rope.cuda(), c, s, wq, wk, order, dtype, kw


@pytest.mark.parametrize('case', CASES)
def test_forward(case):
    from noise_b200.attention import qk_norm_rope
    q, k, _, _, qc, kc, rope, c, s, wq, wk, order, dtype, kw = build(case)
    for got, x, w in zip(qk_norm_rope(qc, kc, rope, **kw), (q, k), (wq, wk)):
        want = oo.norm_rope(x, c, s, w, order)
        check_rows(got, want, dtype, want.abs().amax(-1, keepdim=True) * 2 ** 0.5)


@pytest.mark.parametrize('case', CASES)
def test_backward(case):
    from noise_b200.attention import qk_norm_rope_backward
    q, k, dq, dk, qc, kc, rope, c, s, wq, wk, order, dtype, kw = build(case)
    got = qk_norm_rope_backward(dq.cuda(), dk.cuda(), qc, kc, rope, **kw)
    again = qk_norm_rope_backward(dq.cuda(), dk.cuda(), qc, kc, rope, **kw)
    for i, (x, dy, w) in enumerate(((q, dq, wq), (k, dk, wk))):
        want, dw, size = oo.norm_rope_backward(dy, x, c, s, w, order)
        r = (x.double().square().mean(-1, keepdim=True) + oo.EPS32).rsqrt()
        floor = r * dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5 * x.shape[-1] ** 0.5
        if w is not None:
            floor = floor * w.double().abs().max()
        check_rows(got[i], want, dtype, floor)
        assert torch.equal(got[i], again[i])
        if w is None:
            assert got[2 + i] is None
        else:
            assert ((got[2 + i].double().cpu() - dw).abs() <= 128 * U32 * size).all()
            assert torch.equal(got[2 + i], again[2 + i])


def test_gradient_matches_differences():
    """The formula's gradient against central differences of the kernel itself in fp32: a step of 2^-7 on inputs
    of size 1 leaves a truncation below h^2 |f'''| / 6 ~ 2^-14 and a rounding of 2 * 48 * 2^-24 |y| sum|dy| / (2h)."""
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(1, 3, 2, 32, generator=g).cuda(), torch.randn(1, 3, 1, 32, generator=g).cuda()
    dq, dk = torch.randn(q.shape, generator=g).cuda(), torch.randn(k.shape, generator=g).cuda()
    w = (1 + 0.2 * torch.randn(32, generator=g)).cuda()
    rope = rope_table(8, 32).cuda()
    h = 2.0 ** -7
    for order in ('rotate_norm', 'norm_rotate'):
        kw = dict(q_weight=w, k_weight=w, order=order)

        def loss(q, k):
            a, b = qk_norm_rope(q, k, rope, **kw)
            return ((a.double() * dq.double()).sum() + (b.double() * dk.double()).sum()).item()

        gq, gk, _, _ = qk_norm_rope_backward(dq, dk, q, k, rope, **kw)
        for x, gx, isq in ((q, gq, True), (k, gk, False)):
            for at in range(0, x.numel(), 7):
                e = torch.zeros_like(x)
                e.view(-1)[at] = h
                hi = loss(q + e, k) if isq else loss(q, k + e)
                lo = loss(q - e, k) if isq else loss(q, k - e)
                assert abs((hi - lo) / (2 * h) - gx.view(-1)[at].item()) < 5e-3, (order, at)


def test_out_in_place_into_a_cache_and_unknown_positions():
    from noise_b200.attention import qk_norm_rope
    g = torch.Generator().manual_seed(5)
    q, k = (torch.randn(2, 3, n, 64, generator=g).bfloat16().cuda() for n in (4, 2))
    rope = rope_table(16, 64).cuda()
    want = qk_norm_rope(q, k, rope)
    cache = torch.full((2, 10, 2, 64), 7.0, dtype=torch.bfloat16, device='cuda')
    qq = q.clone()
    got = qk_norm_rope(qq, k, rope, out=(qq, cache[:, 4:7]))
    assert torch.equal(qq, want[0]) and torch.equal(cache[:, 4:7], want[1]) and got[0] is qq
    assert (cache[:, :4] == 7).all() and (cache[:, 7:] == 7).all()
    pos = torch.tensor([0, 16, 2], dtype=torch.int32).cuda()
    y, z = qk_norm_rope(q, k, rope, positions=pos)
    assert y[:, 1].isnan().all() and z[:, 1].isnan().all() and y[:, [0, 2]].isfinite().all()
    assert torch.equal(y[:, [0, 2]], want[0][:, [0, 2]])


def test_empty_and_special_values():
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward
    rope = rope_table(16, 64).cuda()
    w = torch.ones(64, device='cuda')
    q, k = torch.empty(0, 3, 4, 64, device='cuda'), torch.empty(0, 3, 2, 64, device='cuda')
    assert qk_norm_rope(q, k, rope)[0].shape == q.shape
    g = qk_norm_rope_backward(q, k, q, k, rope, q_weight=w, k_weight=w)
    assert g[0].shape == q.shape and (g[2] == 0).all() and (g[3] == 0).all()
    q, k = torch.zeros(1, 3, 4, 64, device='cuda'), torch.zeros(1, 3, 2, 64, device='cuda')
    q[0, 1, 2, 5] = float('nan')  # stays in its row
    y, z = qk_norm_rope(q, k, rope)
    assert y[0, 1, 2].isnan().all() and y.isnan().sum() == 64 and (z == 0).all()


def test_streams_and_graph_replay():
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(2, 50, n, 64, generator=g).bfloat16().cuda() for n in (4, 2))
    rope, w = rope_table(64, 64).cuda(), torch.ones(64, device='cuda') * 1.5
    kw = dict(q_weight=w, k_weight=w)
    qk_norm_rope_backward(q, k, q, k, rope, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = qk_norm_rope(q, k, rope, **kw)
        d = qk_norm_rope_backward(*y, q, k, rope, **kw)
    q.copy_(torch.randn(q.shape, generator=g))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = qk_norm_rope(q, k, rope, **kw)
        d2 = qk_norm_rope_backward(*y2, q, k, rope, **kw)
    torch.cuda.synchronize()
    for a, b in zip((*y, *d), (*y2, *d2)):
        assert torch.equal(a, b)
