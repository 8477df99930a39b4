"""The sliding-window attention where test_window_gpu.py does not look: the token form's lse and the bits of its P."""
import pytest
import torch

from oracle import operators as oo
from test_window_gpu import DT, TOKENS, deltas, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('case', TOKENS)
def test_token_lse(case):
    """|lse - want| within delta (test_window_gpu.py: the relative error of the probabilities' sum) and its own rounding."""
    from noise_b200.attention import window_attention_token
    B, Tk, H, Hk, D, window, sinks, dt, lengths = case
    g = torch.Generator().manual_seed(B + Tk + D)
    q, k, v = randn(g, B, H, D, dtype=DT[dt]), randn(g, B, Tk, Hk, D, dtype=DT[dt]), randn(g, B, Tk, Hk, D, dtype=DT[dt])
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    args = (q.cuda(), k.cuda(), v.cuda(), ln, window, sinks)
    out, lse = window_attention_token(*args, with_lse=True)
    assert torch.equal(out, window_attention_token(*args)) and lse.shape == (B, H) and lse.dtype == torch.float32
    d = deltas(q, k)
    for b, n in enumerate(lengths):
        if n == 0:
            assert (lse[b] == -torch.inf).all()
            continue
        want = oo.window_attention(q[b:b + 1, None], k[b:b + 1, :n], v[b:b + 1, :n], window, sinks)[1][0, :, 0]
        assert ((lse[b].double().cpu() - want).abs() <= d + 2.0 ** -22 * want.abs() + 2.0 ** -21).all(), b


def test_token_lse_of_an_empty_batch():
    from noise_b200.attention import window_attention_token
    z = torch.zeros(0, 5, 2, 64, dtype=torch.bfloat16, device='cuda')
    out, lse = window_attention_token(z[:, 0], z, z, torch.zeros(0, dtype=torch.int32, device='cuda'), 3, with_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.parametrize('case', TOKENS)
def test_token_probabilities_have_two_parts(case):
    """P goes into its product as two numbers of the input type, so all of the error but the result's own rounding is fp32's
    delta and what the second part leaves: 2^-16 of bf16 (two roundings of 2^-8), 2^-22 of fp16 with the subnormal half
    step 2^-25 for each key. test_window_gpu.py grants one part, u sum p |v|, 256 times as much in bf16."""
    from noise_b200.attention import window_attention_token
    B, Tk, H, Hk, D, window, sinks, dt, lengths = case
    g = torch.Generator().manual_seed(B + Tk + D)
    q, k, v = randn(g, B, H, D, dtype=DT[dt]) / 8, randn(g, B, Tk, Hk, D, dtype=DT[dt]), randn(g, B, Tk, Hk, D, dtype=DT[dt])
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = window_attention_token(q.cuda(), k.cuda(), v.cuda(), ln, window, sinks)
    u, d = torch.finfo(DT[dt]).eps / 2, deltas(q, k)
    for b, n in enumerate(lengths):
        if not n:
            continue
        want, _, mag = oo.window_attention(q[b:b + 1, None], k[b:b + 1, :n], v[b:b + 1, :n], window, sinks)
        tol = (u * u + d) * mag + u * want.abs()
        if dt == 'fp16':
            tol = tol + (n * v.double().abs().max() + 1) * 2.0 ** -25
        err = (out[b].double().cpu() - want[0, 0]).abs()
        assert (err <= tol[0, 0]).all(), (b, (err / tol[0, 0]).max())


@pytest.mark.parametrize('D,H,Hk,Tq,Tk,offset,window,sinks,lengths', [
    (64, 2, 1, 40, 300, 100, 64, 3, None), (128, 2, 2, 130, 512, 7, 200, 0, None), (64, 4, 2, 1, 200, 0, 5, 1, None),
    (96, 3, 1, 257, 700, 130, 60, 140, (700, 300)), (128, 2, 1, 20, 150, 60, 20, 2, (70, 80)),
])
def test_rows_behind_the_last_query_hold_anything(D, H, Hk, Tq, Tk, offset, window, sinks, lengths):
    """A prompt's part over a preallocated cache: the rows behind it are no key of any query, whatever they hold, and their
    gradients are zero."""
    from noise_b200.attention import window_attention, window_attention_backward
    from test_window_gpu import check_backward, check_forward
    g = torch.Generator().manual_seed(D + Tq)
    B, bf = 2, torch.bfloat16
    q, k, v, do = (randn(g, B, *s, D, dtype=bf) for s in ((Tq, H), (Tk, Hk), (Tk, Hk), (Tq, H)))
    c = [x.cuda() for x in (q, k, v, do)]
    c[1][:, offset + Tq:], c[2][:, offset + Tq:] = float('nan'), float('inf')
    kw = dict(offset=offset)
    if lengths:
        kw['lengths'] = torch.tensor(lengths, dtype=torch.int32).cuda()
    out, lse = window_attention(*c[:3], window, sinks, **kw)
    check_forward(out, lse, q, k, v, window, sinks, lengths, offset, bf)
    got = window_attention_backward(c[3], *c[:3], out, lse, window, sinks, **kw)
    check_backward(got, do, q, k, v, window, sinks, lengths, offset)
    assert (got[1][:, offset + Tq:] == 0).all() and (got[2][:, offset + Tq:] == 0).all()
