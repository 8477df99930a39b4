"""The sliding-window attention with sinks, its gradient and its single-token form against float64
(oracle/operators.py).

Tolerances. A score is a sum of D products in fp32 and its exponent one more rounding: with
Z = scale max sum_d |q_d k_d| over the pairs, every probability has a relative error of at most
delta = 2 (D 2^-24 Z + 2^-24 (2 Z + 8)) + 2^-21. P is then rounded to the input type, u = eps / 2 each, and the
products add in fp32. With A = sum p |v|: |out - want| <= (u + delta) A + u |want| + (keys) 2^-24 A, taken with
keys 2^-24 inside delta. fp16 holds P below 2^-14 with an absolute half step of 2^-25: keys 2^-25 max|v| more.
lse: delta + 2^-22 |lse|.

Gradients: P and dS are rounded to bf16 once each. dS = P (dP - Delta), where Delta comes from the rounded
output, itself off by (u + delta) A + u |out|; with size = P (|dO| |V|^T + |dO| . sum p |v|), |dS| <= size and its error is
at most (3 u + 2 delta) size. Then |dV - want| <= (u + delta) P^T |dO| + u |want|, |dQ - want| <= (3 u + 2 delta) size |K| + u |want|,
and the same for dK."""
import pytest
import torch

from oracle import operators as oo

pytestmark = pytest.mark.gpu
DT = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def deltas(q, k, scale=None):
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    Z = scale * (q.double().abs().amax(tuple(range(q.dim() - 1))) * k.double().abs().amax((0, 1, 2))).sum().item()
    Z = min(Z, scale * q.double().norm(dim=-1).max().item() * k.double().nan_to_num().norm(dim=-1).max().item())
    return 2 * (D * 2.0 ** -24 * Z + 2.0 ** -24 * (2 * Z + 8)) + 2.0 ** -21 + k.shape[1] * 2.0 ** -24


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, dtype=torch.float64).to(dtype)


CASES = [  # B, Tq, Tk, H, Hk, D, window, sinks, dtype, lengths, offset
    (1, 1, 1, 1, 1, 64, 0, 0, 'bf16', None, None),
    (2, 100, 100, 2, 2, 64, 1000, 0, 'bf16', None, None),
    (1, 128, 128, 2, 1, 64, 20, 3, 'bf16', None, None),
    (2, 257, 257, 4, 2, 64, 64, 4, 'fp16', None, None),
    (1, 700, 700, 2, 1, 64, 100, 70, 'bf16', None, None),
    (1, 513, 513, 3, 1, 128, 37, 130, 'bf16', None, None),
    (2, 300, 300, 4, 4, 128, 127, 0, 'fp16', None, None),
    (4, 260, 260, 2, 1, 128, 50, 5, 'bf16', (260, 0, 131, 1), None),
    (3, 300, 300, 2, 2, 64, 90, 2, 'bf16', (128, 300, 257), None),
    (2, 40, 333, 2, 1, 64, 60, 9, 'bf16', None, None),
    (2, 40, 333, 2, 1, 96, 333, 0, 'bf16', (333, 300), None),
    (1, 130, 400, 2, 2, 40, 80, 200, 'fp16', None, 100),
    (1, 33, 65, 5, 5, 8, 16, 1, 'bf16', None, 3),
    (1, 640, 640, 1, 1, 72, 0, 1, 'bf16', None, None),
    (1, 1500, 1500, 2, 1, 64, 1024, 4, 'bf16', None, None),
    (1, 1300, 1300, 1, 1, 128, 700, 1, 'bf16', (1201,), None),
]


def build(case, extra=1):
    B, Tq, Tk, H, Hk, D, window, sinks, dt, lengths, offset = case
    g = torch.Generator().manual_seed(Tq * 7 + Tk + D + window)
    q, k, v = (randn(g, B, *s, D, dtype=DT[dt]) for s in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    do = randn(g, B, Tq, H, D, dtype=DT[dt])
    kw = {}
    qc, kc, vc, dc = q.cuda(), k.cuda(), v.cuda(), do.cuda()
    if lengths is not None:
        kw['lengths'] = torch.tensor(lengths, dtype=torch.int32).cuda()
        off = Tk - Tq if offset is None else offset
        for b, n in enumerate(lengths):  # padding holds anything
            kc[b, n:], vc[b, n:] = float('nan'), float('inf')
            qc[b, max(0, n - off):], dc[b, max(0, n - off):] = float('nan'), float('nan')
    if offset is not None:
        kw['offset'] = offset
    return q, k, v, do, qc, kc, vc, dc, window, sinks, lengths, offset, kw


def check_forward(out, lse, q, k, v, window, sinks, lengths, offset, dtype):
    want, wlse, mag = oo.window_attention(q, k, v, window, sinks, lengths, offset)
    d, u = deltas(q, k), torch.finfo(dtype).eps / 2
    tol = (u + d) * mag + u * want.abs()
    if dtype == torch.float16:
        tol = tol + (k.shape[1] * v.double().abs().max() + 1) * 2.0 ** -25
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())
    have = wlse.isfinite()
    got = lse.double().cpu()
    assert torch.equal(got.isfinite(), have) and (got[~have] == -torch.inf).all()
    assert ((got - wlse)[have].abs() <= d + 2.0 ** -22 * wlse[have].abs() + 2.0 ** -21).all()


@pytest.mark.parametrize('case', CASES)
def test_forward(case):
    from noise_b200.attention import window_attention
    q, k, v, _, qc, kc, vc, _, window, sinks, lengths, offset, kw = build(case)
    out, lse = window_attention(qc, kc, vc, window, sinks, **kw)
    check_forward(out, lse, q, k, v, window, sinks, lengths, offset, q.dtype)
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    again, lse2 = window_attention(qc, kc, vc, window, sinks, status=status, **kw)
    assert torch.equal(out, again) and torch.equal(lse, lse2) and status.item() == 0


def check_backward(got, do, q, k, v, window, sinks, lengths, offset):
    want = oo.window_attention_backward(do, q, k, v, window, sinks, lengths, offset)
    d, u = deltas(q, k), 2.0 ** -8
    for name, g, w, mag, part in zip(('dq', 'dk', 'dv'), got, want[:3], want[3:], (3 * u + 2 * d, 3 * u + 2 * d, u + d)):
        err = (g.double().cpu() - w).abs()
        tol = part * mag + u * w.abs()
        assert (err <= tol).all(), (name, (err - tol).max().item(), err.max().item())
        # a wrong sum would also show as a bias: the errors' norm stays near the roundings' (well below their bound)
        if w.norm() > 0:
            assert err.norm() <= 2 * u * w.norm() + 0.5 * (part * mag).norm(), (name, err.norm() / w.norm())


@pytest.mark.parametrize('case', [c for c in CASES if c[8] == 'bf16'] + [
    (1, 1000, 1000, 8, 1, 64, 30, 5, 'bf16', None, None),      # split: shared heads, few key tiles, sinks
    (1, 2100, 2100, 2, 2, 64, 40, 3, 'bf16', None, None),      # split sinks, even tiles whole
    (2, 900, 900, 6, 1, 128, 800, 0, 'bf16', (900, 333), None),
    (2, 1100, 1300, 4, 1, 96, 64, 140, 'bf16', (1300, 900), None),
])
def test_backward(case):
    from noise_b200.attention import window_attention, window_attention_backward
    q, k, v, do, qc, kc, vc, dc, window, sinks, lengths, offset, kw = build(case)
    out, lse = window_attention(qc, kc, vc, window, sinks, **kw)
    got = window_attention_backward(dc, qc, kc, vc, out, lse, window, sinks, **kw)
    check_backward(got, do, q, k, v, window, sinks, lengths, offset)
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    again = window_attention_backward(dc, qc, kc, vc, out, lse, window, sinks, status=status, **kw)
    assert status.item() == 0
    for a, b in zip(got, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize('D,factor,window,sinks', [(64, 8, 100, 3), (128, 8, 400, 0), (64, 2.0 ** -40, 50, 1)])
def test_backward_of_large_and_tiny_scores(D, factor, window, sinks):
    """-lse / scale and -Delta go through the tensor core on the keys' side: scores of up to a few hundred keep their
    differences (their sums' error is deltas' term in Z, |lse| being at most Z + log Tk), and vanishing ones their size."""
    from noise_b200.attention import window_attention, window_attention_backward
    g = torch.Generator().manual_seed(D + window)
    q, k, v, do = (randn(g, 1, 333, n, D, dtype=torch.bfloat16) for n in (2, 1, 1, 2))
    q = q * factor
    c = [t.cuda() for t in (q, k, v, do)]
    out, lse = window_attention(*c[:3], window, sinks)
    check_backward(window_attention_backward(c[3], *c[:3], out, lse, window, sinks), do, q, k, v, window, sinks, None, None)


def test_oracle_gradient_matches_differences():
    """The float64 formulas that the kernel is held to, against central differences of the float64 forward."""
    g = torch.Generator().manual_seed(31)
    q, k, v, do = (torch.randn(1, 9, n, 8, generator=g, dtype=torch.float64) for n in (2, 1, 1, 2))
    lengths = (8,)
    grads = oo.window_attention_backward(do, q, k, v, 3, 1, lengths)[:3]
    for x, gx in zip((q, k, v), grads):
        for at in range(0, x.numel(), 5):
            old = x.view(-1)[at].item()
            vals = []
            for h in (1e-5, -1e-5):
                x.view(-1)[at] = old + h
                vals.append((oo.window_attention(q, k, v, 3, 1, lengths)[0] * do).sum().item())
            x.view(-1)[at] = old
            assert abs((vals[0] - vals[1]) / 2e-5 - gx.reshape(-1)[at].item()) < 1e-8


def test_backward_layouts_graph_and_stream():
    """Strided operands and gradients; a captured forward and backward that follows its inputs; another stream."""
    from noise_b200.attention import window_attention, window_attention_backward
    g = torch.Generator().manual_seed(19)
    qkv = randn(g, 2, 310, 8, 64, dtype=torch.bfloat16).cuda()
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    do = randn(g, 2, 4, 310, 64, dtype=torch.bfloat16).cuda().transpose(1, 2)
    lengths = torch.tensor([310, 211], dtype=torch.int32, device='cuda')
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    kw = dict(lengths=lengths, status=status)

    def both(q, k, v, do):
        out, lse = window_attention(q, k, v, 100, 4, **kw)
        return (out, lse, *window_attention_backward(do, q, k, v, out, lse, 100, 4, **kw))

    want = both(q, k, v, do)
    for a, b in zip(want, both(*(t.contiguous() for t in (q, k, v, do)))):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = both(q, k, v, do)
    qkv.copy_(randn(g, *qkv.shape, dtype=torch.bfloat16))
    lengths.copy_(torch.tensor([40, 309]))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = both(q, k, v, do)
    torch.cuda.synchronize()
    assert status.item() == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_layouts():
    """Views of a packed projection, heads before tokens, a cache's rows, misaligned and broadcast operands."""
    from noise_b200.attention import window_attention
    g = torch.Generator().manual_seed(11)
    qkv = randn(g, 2, 150, 8, 64, dtype=torch.bfloat16)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    c = qkv.cuda()
    out, lse = window_attention(c[:, :, :4], c[:, :, 4:6], c[:, :, 6:], 33, 2)
    check_forward(out, lse, q, k, v, 33, 2, None, None, q.dtype)
    t = [x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(window_attention(*t, 33, 2)[0], out)
    cache = torch.zeros(2, 400, 2, 64, dtype=torch.bfloat16, device='cuda')
    cache[:, 20:170] = k.cuda()
    assert torch.equal(window_attention(t[0], cache[:, 20:170], t[2], 33, 2)[0], out)
    flat = torch.zeros(q.numel() + 3, dtype=torch.bfloat16, device='cuda')
    flat[3:] = q.cuda().reshape(-1)
    assert torch.equal(window_attention(flat[3:].view(q.shape), t[1], t[2], 33, 2)[0], out)
    one = k[:, :, :1].cuda()
    a = window_attention(t[0], one.expand(2, 150, 4, 64), one.expand(2, 150, 4, 64), 33, 2)[0]
    assert torch.equal(a, window_attention(t[0], one, one, 33, 2)[0])


def test_scores_of_any_size():
    """Rows whose maximum keeps growing along the keys rescale many times; large scores keep their differences."""
    from noise_b200.attention import window_attention
    g = torch.Generator().manual_seed(12)
    for D in (64, 128):
        q, v = randn(g, 1, 600, 1, D, dtype=torch.bfloat16), randn(g, 1, 600, 1, D, dtype=torch.bfloat16)
        ramp = torch.linspace(0.01, 6, 600, dtype=torch.float64)[None, :, None, None]
        k = (q.double().mean(1, keepdim=True).sign() * ramp).to(torch.bfloat16)
        q = (q.double().abs() * q.double().mean(1, keepdim=True).sign()).to(torch.bfloat16)
        out, lse = window_attention(q.cuda(), k.cuda(), v.cuda(), None, 0)
        check_forward(out, lse, q, k, v, 600, 0, None, None, q.dtype)
        out, lse = window_attention(q.cuda(), -k.cuda(), v.cuda(), 200, 10)
        check_forward(out, lse, q, -k, v, 200, 10, None, None, q.dtype)
        out, lse = window_attention(q.cuda() * 0, k.cuda(), v.cuda(), 200, 10, scale=3.0)
        check_forward(out, lse, q * 0, k, v, 200, 10, None, None, q.dtype)


def test_forward_graph_and_stream():
    from noise_b200.attention import window_attention
    g = torch.Generator().manual_seed(13)
    q, k, v = (randn(g, 2, 300, n, 64, dtype=torch.bfloat16).cuda() for n in (4, 2, 2))
    lengths = torch.tensor([300, 211], dtype=torch.int32, device='cuda')
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    window_attention(q, k, v, 100, 4, lengths=lengths, status=status)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = window_attention(q, k, v, 100, 4, lengths=lengths, status=status)
    q.copy_(randn(g, *q.shape, dtype=torch.bfloat16))
    lengths.copy_(torch.tensor([10, 299]))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = window_attention(q, k, v, 100, 4, lengths=lengths, status=status)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and status.item() == 0


TOKENS = [  # B, Tk, H, Hk, D, window, sinks, dtype, lengths
    (1, 1, 1, 1, 64, 0, 0, 'bf16', (1,)),
    (3, 50, 4, 2, 64, 10, 2, 'bf16', (50, 0, 7)),
    (2, 700, 8, 8, 64, 1000, 0, 'fp16', (700, 333)),
    (2, 2048, 8, 1, 128, 1024, 4, 'bf16', (2048, 1500)),
    (5, 400, 40, 2, 96, 399, 0, 'bf16', (1, 2, 17, 399, 400)),
    (1, 5000, 3, 1, 128, 4000, 64, 'fp16', (4990,)),
    (70, 130, 16, 8, 40, 128, 1, 'bf16', tuple(range(61, 131))),
    (2, 333, 6, 3, 8, 0, 5, 'bf16', (333, 4)),
    (1, 17001, 4, 2, 64, 17001, 0, 'bf16', (17001,)),     # clusters of 16 CTAs
    (2, 9001, 20, 1, 96, 8990, 3, 'fp16', (9001, 5)),
]


@pytest.mark.parametrize('case', TOKENS)
def test_token(case):
    from noise_b200.attention import window_attention_token
    B, Tk, H, Hk, D, window, sinks, dt, lengths = case
    g = torch.Generator().manual_seed(B + Tk + D)
    q, k, v = randn(g, B, H, D, dtype=DT[dt]), randn(g, B, Tk, Hk, D, dtype=DT[dt]), randn(g, B, Tk, Hk, D, dtype=DT[dt])
    kc, vc = k.cuda(), v.cuda()
    for b, n in enumerate(lengths):
        kc[b, n:], vc[b, n:] = float('nan'), float('inf')
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = window_attention_token(q.cuda(), kc, vc, ln, window, sinks)
    u, d = torch.finfo(DT[dt]).eps / 2, deltas(q, k)
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        want, _, mag = oo.window_attention(q[b:b + 1, None], k[b:b + 1, :n], v[b:b + 1, :n], window, sinks)
        tol = (u + d) * mag + u * want.abs()
        if dt == 'fp16':
            tol = tol + (n * v.double().abs().max() + 1) * 2.0 ** -25
        err = (out[b].double().cpu() - want[0, 0]).abs()
        assert (err <= tol[0, 0]).all(), (b, (err - tol[0, 0]).max())
    # a cache with heads before tokens, and queries that are rows of a packed projection
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
    packed = torch.cat([q.cuda(), q.cuda()], 1)[:, H:]
    assert torch.equal(window_attention_token(packed, kt, vt, ln, window, sinks), out)


def test_token_graph_follows_lengths():
    from noise_b200.attention import window_attention_token
    g = torch.Generator().manual_seed(17)
    q, k, v = (randn(g, 2, *s, 64, dtype=torch.bfloat16).cuda() for s in ((8,), (900, 2), (900, 2)))
    ln = torch.tensor([20, 1], dtype=torch.int32, device='cuda')
    window_attention_token(q, k, v, ln, 500, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_token(q, k, v, ln, 500, 4)
    for lengths in ((900, 0), (501, 777)):
        ln.copy_(torch.tensor(lengths))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, window_attention_token(q, k, v, ln, 500, 4))


def test_empty_batches():
    from noise_b200.attention import window_attention, window_attention_backward, window_attention_token
    z = torch.zeros(0, 5, 2, 64, dtype=torch.bfloat16, device='cuda')
    assert window_attention(z, z, z, 3)[0].shape == z.shape
    assert window_attention_token(z[:, 0], z, z, torch.zeros(0, dtype=torch.int32, device='cuda'), 3).shape == (0, 2, 64)
    k = torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16, device='cuda')
    assert window_attention_backward(z, z, z, z, z, torch.zeros(0, 2, 5, device='cuda'), 3)[0].shape == z.shape
    out, lse = window_attention(k[:, :0], k, k, 3)
    assert out.shape == (2, 0, 2, 64) and lse.shape == (2, 2, 0)
