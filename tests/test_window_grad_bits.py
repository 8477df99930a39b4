"""How many bits dS has on its way into dQ and dK: two bf16 numbers, of which a lost second one would stay within the
bounds of test_window_gpu.py.

The gradient is held to its formula with what the call was given, out among it: Delta = dO . out as saved, so that the
rounding of out is no part of the error. Rows see few keys and scores are small, so that what fp32 adds up is small too. With
u = 2^-8 (bf16) and d as in test_window_gpu.py for these few keys:
  dS is cut after 8 bits, the rest (below 2^-7 |dS|) rounded to 8: 2^-15 |dS|
  fp32: P is off by d of itself, dP and Delta by D 2^-24 of their terms' sum, each less than d of size =
  P (|dO| |V|^T + |dO| . |out|): 2 d size in all
  |dQ - want| <= u |want| + 2^-15 |dS| |K| + 2 d size |K|, the same for dK; P is one bf16 number:
  |dV - want| <= u |want| + (u + d) P^T |dO|."""
import pytest
import torch

from oracle import operators as oo
from test_window_gpu import deltas, randn

U = 2.0 ** -8
CASES = [(64, 2, 1, 300, 24, 0), (128, 3, 3, 270, 30, 5), (96, 4, 2, 200, 16, 9)]  # D, H, Hk, T, window, sinks


def inputs(D, H, Hk, T):
    g = torch.Generator().manual_seed(D + T)
    q, k, v, do = (randn(g, 1, T, n, D, dtype=torch.bfloat16) for n in (H, Hk, Hk, H))
    return q / 16, k, v, do


def formula(q, k, v, do, out, window, sinks, rounded=lambda ds: ds):
    """dq, dk, dv with Delta from out, and their bounds."""
    T, H, D = q.shape[1:]
    group, scale = H // k.shape[2], D ** -0.5
    seen = oo.visible(T, T, 0, window, sinks, T)
    d = deltas(q, k) - (T - window - sinks - 1) * 2.0 ** -24
    grads = [torch.zeros(x.shape, dtype=torch.float64) for x in (q, k, v)]
    tols = [torch.zeros_like(x) for x in grads]
    for h in range(H):
        kv = h // group
        Q, K, V, G, O = q[0, :, h].double(), k[0, :, kv].double(), v[0, :, kv].double(), do[0, :, h].double(), out[0, :, h].double()
        P = torch.softmax((Q @ K.T * scale).masked_fill(~seen, -torch.inf), 1)
        exact = P * (G @ V.T - (G * O).sum(1, keepdim=True))
        size = P * (G.abs() @ V.abs().T + (G * O).abs().sum(1, keepdim=True))
        dS, part = rounded(exact) * scale, (2.0 ** -15 * exact.abs() + 2 * d * size) * scale
        grads[0][0, :, h], tols[0][0, :, h] = dS @ K, part @ K.abs()
        grads[1][0, :, kv] += dS.T @ Q
        tols[1][0, :, kv] += part.T @ Q.abs()
        grads[2][0, :, kv] += P.T @ G
        tols[2][0, :, kv] += (U + d) * (P.T @ G.abs())
    return grads, [t + U * w.abs() for t, w in zip(tols, grads)]


@pytest.mark.parametrize('D,H,Hk,T,window,sinks', CASES)
def test_the_bound_sees_a_lost_part(D, H, Hk, T, window, sinks):
    """In float64 with the roundings put in by hand: two parts of dS pass, one does not, in dQ and in dK."""
    q, k, v, do = inputs(D, H, Hk, T)
    out = oo.window_attention(q, k, v, window, sinks)[0].bfloat16()
    want, tol = formula(q, k, v, do, out, window, sinks)

    def cut(x):
        return (x.float().view(torch.int32) & -65536).view(torch.float32).double()

    def two(ds):
        return cut(ds) + (ds - cut(ds)).bfloat16().double()

    for rounded, passes in ((two, True), (cut, False), (lambda ds: ds.bfloat16().double(), False)):
        got, _ = formula(q, k, v, do, out, window, sinks, rounded)
        for i in (0, 1):
            assert ((got[i].bfloat16().double() - want[i]).abs() <= tol[i]).all() == passes, i


@pytest.mark.gpu
@pytest.mark.parametrize('D,H,Hk,T,window,sinks', CASES)
def test_gradient_keeps_sixteen_bits_of_dS(D, H, Hk, T, window, sinks):
    from noise_b200.attention import window_attention, window_attention_backward
    q, k, v, do = inputs(D, H, Hk, T)
    c = [x.cuda() for x in (q, k, v, do)]
    out, lse = window_attention(*c[:3], window, sinks)
    got = window_attention_backward(c[3], *c[:3], out, lse, window, sinks)
    want, tol = formula(q, k, v, do, out.cpu(), window, sinks)
    for name, a, w, t in zip(('dq', 'dk', 'dv'), got, want, tol):
        err = (a.double().cpu() - w).abs()
        assert (err <= t).all(), (name, (err / t).max().item())
