"""The attention operators and the distillation loss used together: a block with a head, forward and backward, against
float64 autograd; a sequence that generates token by token over a cache against the same attention over the whole
sequence; and DUST's exact attention-internal errors and distillation error.

Tolerances: relative L2 errors. The values pass about six roundings to bf16 one after the other (the projection, the
normed queries and keys, P, the output, dS, the gradients), each at most 2^-8 of its value, and dS subtracts two numbers
of its size: 8 * 2^-8 bounds the gradients' relative L2 error, 4 * 2^-8 the forward's; the differences a unit and sign
off would be of order 1. Losses: the logits' bf16 roundings, 2^-8 max|z| a logit, averaged over the entries."""
import pytest
import torch

from oracle import operators as oo

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def rel(got, want):
    got, want = got.double().cpu().reshape(-1), want.double().cpu().reshape(-1)
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize('H,Hk,D,order,window,sinks', [(8, 8, 64, 'rotate_norm', 40, 2), (6, 2, 128, 'norm_rotate', 100, 4)])
def test_block_and_head_forward_and_backward(H, Hk, D, order, window, sinks):
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward, window_attention, window_attention_backward
    from noise_b200.distill import distill_loss_grad
    from noise_b200.model import rope_table
    B, T, W, V, K = 2, 200, 192, 1000, 8
    g = torch.Generator().manual_seed(7)

    def param(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).div_(shape[-1] ** 0.5).bfloat16()

    x = torch.randn(B, T, W, generator=g, dtype=torch.float64).bfloat16()
    wqkv, wo, wh = param((H + 2 * Hk) * D, W), param(W, H * D), param(V, W)
    wq, wk = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    rope = rope_table(T) if D == 64 else torch.cat([f(torch.outer(torch.arange(T), 10000.0 ** (-torch.arange(0, D, 2) / D)))
                                                    for f in (torch.cos, torch.sin)], 1).bfloat16().float()
    ids = torch.randint(0, V, (B * T, K), generator=g)
    teacher = torch.randn(B * T, K, generator=g) * 2

    # float64 autograd
    leaves = [t.double().requires_grad_() for t in (x, wqkv, wo, wh, wq, wk)]
    X, Wqkv, Wo, Wh, Wq, Wk = leaves
    qkv = (X @ Wqkv.T).view(B, T, H + 2 * Hk, D)
    c, s = oo.rotation(rope, torch.arange(T).expand(B, T))
    Q = oo.norm_rope(qkv[:, :, :H], c, s, Wq, order)
    Kk = oo.norm_rope(qkv[:, :, H:H + Hk], c, s, Wk, order).repeat_interleave(H // Hk, 2)
    Vv = qkv[:, :, H + Hk:].repeat_interleave(H // Hk, 2)
    seen = oo.visible(T, T, 0, window, sinks, T)
    score = torch.einsum('bthd,bshd->bhts', Q, Kk) * D ** -0.5
    Y = torch.einsum('bhts,bshd->bthd', torch.softmax(score.masked_fill(~seen, -torch.inf), -1), Vv)
    Z = (Y.reshape(B, T, -1) @ Wo.T + X) @ Wh.T
    S = 15 * torch.tanh(Z.view(-1, V) / 15)
    logp = torch.log_softmax(teacher.double(), 1)
    loss = (logp.exp() * (logp - torch.log_softmax(S, 1).gather(1, ids))).sum(1)
    want = torch.autograd.grad(loss.sum(), leaves)

    # the operators, with torch's products around them
    cu = [t.cuda() for t in (x, wqkv, wo, wh)]
    xc, a, o, h = cu
    kw = dict(q_weight=wq.float().cuda(), k_weight=wk.float().cuda(), order=order)
    packed = (xc @ a.T).view(B, T, H + 2 * Hk, D)
    qr, kr, vr = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    rc = rope.cuda()
    q, k = qk_norm_rope(qr, kr, rc, **kw)
    y, lse = window_attention(q, k, vr, window, sinks)
    assert rel(y, Y.detach()) <= 4 * U
    stream = y.reshape(B, T, -1) @ o.T + xc
    logits = (stream @ h.T).view(-1, V)
    got_loss, dz = distill_loss_grad(logits, ids.cuda(), teacher.cuda(), softcap=15.0)
    assert (got_loss.double().cpu() - loss.detach()).abs().max() <= 2 * 8 * U * Z.detach().abs().max()
    dz = dz.view(B, T, V)
    dstream = dz @ h
    dwh = dz.reshape(-1, V).T @ stream.reshape(-1, W)
    dy = (dstream @ o).view(B, T, H, D)
    dwo = dstream.reshape(-1, W).T @ y.reshape(-1, H * D)
    dq, dk, dv = window_attention_backward(dy, q, k, vr, y, lse, window, sinks)
    dqr, dkr, dwq, dwk = qk_norm_rope_backward(dq, dk, qr, kr, rc, **kw)
    dpacked = torch.cat([dqr, dkr, dv], 2).reshape(B * T, -1)
    dwqkv = dpacked.T @ xc.reshape(-1, W)
    dx = (dpacked @ a).view(B, T, W) + dstream
    for name, gr, wa in zip(('x', 'wqkv', 'wo', 'wh', 'wq', 'wk'), (dx, dwqkv, dwo, dwh, dwq, dwk), want):
        assert rel(gr, wa) <= 8 * U, (name, rel(gr, wa))


def test_tokens_over_a_cache_equal_the_whole_sequence():
    """Each new token's key is normed, rotated and written into the cache by qk_norm_rope; its query attends over it."""
    from noise_b200.attention import qk_norm_rope, window_attention, window_attention_token
    from noise_b200.model import rope_table
    B, T, H, Hk, D, window, sinks = 3, 40, 8, 2, 64, 12, 3
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(B, T, H + 2 * Hk, D, generator=g).bfloat16().cuda()
    rope = rope_table(64).cuda()
    q, k = qk_norm_rope(qkv[:, :, :H], qkv[:, :, H:H + Hk], rope)
    whole, _ = window_attention(q, k, qkv[:, :, H + Hk:], window, sinks)
    kc = torch.full((B, 64, Hk, D), float('nan'), dtype=torch.bfloat16, device='cuda')
    vc = kc.clone()
    lengths = torch.zeros(B, dtype=torch.int32, device='cuda')
    for t in range(T):
        new = qkv[:, t:t + 1]
        pos = torch.full((B, 1), t, dtype=torch.int32, device='cuda')
        qt = torch.empty(B, 1, H, D, dtype=torch.bfloat16, device='cuda')
        qk_norm_rope(new[:, :, :H], new[:, :, H:H + Hk], rope, positions=pos, out=(qt, kc[:, t:t + 1]))
        vc[:, t] = new[:, 0, H + Hk:]
        lengths += 1
        y = window_attention_token(qt[:, 0], kc, vc, lengths, window, sinks)
        # the same sums with P rounded under another reference, and the output's own rounding: 2 u of sum p |v| each side
        mag = qkv[:, :, H + Hk:].float().abs().max()
        assert (y.float() - whole[:, t].float()).abs().max() <= 4 * U * mag, t
    assert torch.equal(kc[:, :T], k)


def _capture(B, T):
    from noise_b200.data import zipf_tokens
    from noise_b200.dust import Capture
    from noise_b200.model import Weights
    rows = zipf_tokens(B, T + 1, seed=5)
    w = Weights('cuda', seed=0)
    x, y = rows[:, :-1].contiguous(), rows[:, 1:].contiguous()
    return w, Capture(w, x, y)


@pytest.mark.parametrize('B,T', [(2, 128), (1, 1152)])  # 1,152 tokens: the 1,024 window binds
def test_exact_local_errors_match_float64(B, T):
    from noise_b200.dust import LocalInputs, exact_local_errors, layer_window
    w, cap = _capture(B, T)
    g = torch.Generator().manual_seed(21)
    targets = {i: (torch.randn(B, T, 512, generator=g) * 0.01).cuda() for i in range(8)}
    got = exact_local_errors(w, cap, targets)
    assert sorted(got) == ['gate', 'k', 'q', 'v', 've'] and len(got['q']) == 8 and len(got['ve']) == 4
    c, s = oo.rotation(w.rope(T).cpu(), torch.arange(T).expand(B, T))
    for layer in (0, 3, 5):
        li = LocalInputs(w, cap, layer)
        q, k, v = (li.raw[n].cpu().double().view(B, T, 8, 64).requires_grad_() for n in 'qkv')
        values, leaves = v, [q, k, v]
        if li.z is not None:
            zz = li.z.cpu().double().view(B, T, 8).requires_grad_()
            ve = li.ve.cpu().double().view(B, T, 8, 64).requires_grad_()
            values, leaves = v + 2 * torch.sigmoid(zz)[..., None] * ve, leaves + [zz, ve]
        Q, Kk = oo.norm_rope(q, c, s), oo.norm_rope(k, c, s)
        seen = oo.visible(T, T, 0, layer_window(layer), 0, T)
        sc = (torch.einsum('bthd,bshd->bhts', Q, Kk) / 8).masked_fill(~seen, -torch.inf)
        y = torch.einsum('bhts,bshd->bthd', torch.softmax(sc, -1), values)
        want = torch.autograd.grad((y * targets[layer].cpu().double().view(B, T, 8, 64)).sum(), leaves)
        for kind, wa in zip(('q', 'k', 'v', 'gate', 've'), want):
            site = f'value_embeds.{layer}' if kind == 've' else \
                f'transformer.h.{layer}.attn.' + dict(q='c_q', k='c_k', v='c_v', gate='ve_gate')[kind]
            assert rel(got[kind][site], wa) <= 8 * U, (layer, kind, rel(got[kind][site], wa))


def test_draws_converge_to_the_exact_errors():
    """One whole cycle of 512 orthogonal draws gives a query's directional differences in every direction; what is
    left beside the gradient is the second order of the step sigma = 0.1 on rows of size 1 and more, and the
    scores' bf16 noise divided by it: about a tenth each, so a cosine above 0.95 (opposite signs or a wrong
    scale of heads would leave it near 0)."""
    from noise_b200.dust import exact_local_errors, local_errors
    w, cap = _capture(1, 128)
    g = torch.Generator().manual_seed(22)
    targets = {i: (torch.randn(1, 128, 512, generator=g) * 0.01).cuda() for i in range(8)}
    exact = exact_local_errors(w, cap, targets, ('q',))['q']
    drawn = local_errors(w, cap, 'q', 512, targets, 0, 1)
    for site, e in exact.items():
        cos = torch.nn.functional.cosine_similarity(e.reshape(-1).double(), drawn[site].reshape(-1).double(), dim=0).item()
        assert cos > 0.95, (site, cos)


def test_dust_step_with_exact_local_errors():
    """A DUST update whose attention-internal errors are exact: it runs, moves every attention weight and is finite."""
    from noise_b200.data import zipf_tokens
    from noise_b200.dust import DUST, recipe
    from noise_b200.model import Weights
    from noise_b200.optim import make_optimizer
    r = recipe(1 / 64)
    r.exact_local = True
    w = Weights('cuda', seed=0)
    opt = make_optimizer(w, r.lr, r.betas, r.anvil_lr, r.anvil_wd, 10)
    rows = zipf_tokens(1, 129, seed=3)
    before = w.flat.clone()
    loss = DUST(w, r, 0).step(rows[:, :-1], rows[:, 1:], opt)
    assert 0 < loss < 20 and w.flat.isfinite().all()
    off = 0
    for name, v in w.named_parameters():
        if '.attn.' in name:
            assert not torch.equal(before[off:off + v.numel()], v.reshape(-1)), name
        off += v.numel()


def test_distill_error_of_a_capture():
    from noise_b200.dust import distill_error, reassemble
    w, cap = _capture(2, 128)
    cap.y[0, :5] = -1  # ignored targets carry no error
    g = torch.Generator().manual_seed(23)
    ids = torch.randint(0, 4096, (2, 128, 16), generator=g).cuda()
    t = (torch.randn(2, 128, 16, generator=g) * 2).cuda()
    loss, err = distill_error(cap, ids, t, temperature=2.0)
    want, q, p, slope = oo.distill(cap.logits.cpu(), ids.cpu().view(-1, 16), t.cpu().view(-1, 16), 2.0, 15.0)
    assert rel(loss, want) < 1e-6
    full = 2.0 * (q - p) * slope
    full[:5] = 0
    assert rel(err, full) < 1e-6 and (err[0, :5] == 0).all()
    x = cap.final.cpu().double()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + oo.EPS32)
    # tf32 products keep 10 bits of either operand: 2^-10 relative in all
    assert rel(reassemble(cap, 'lm_head', err), full.T @ x) <= 2e-3


def test_repeated_calls_look_at_each_tensor():
    """Checks are kept by shapes and strides; addresses and devices are each call's own. The attention calls copy an
    operand they cannot load from, so the results are the same bits. The distillation takes any address of an fp32, but
    the address decides which of a row's 99 logits a thread adds up: two orders of a sum of n positive fp32 terms differ
    by at most 2 n 2^-24 of it. So lse and with it the loss may differ by 2 * 99 * 2^-24, and by the roundings of the
    entries' sum (5 terms below 32, up to 4 roundings each: 20 * 32 * 2^-24); a gradient, at most 1, by 2 * 99 * 2^-24
    and its own roundings (8 * 2^-24)."""
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward, window_attention, window_attention_token
    from noise_b200.distill import distill_loss_grad
    g = torch.Generator().manual_seed(5)

    def odd(t):  # the same values, shape and strides at an address that the kernels cannot load from
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    q, k, v = (torch.randn(2, 40, n, 64, generator=g).bfloat16().cuda() for n in (4, 2, 2))
    rope = torch.randn(40, 64, generator=g).cuda()
    lengths = torch.tensor([40, 17], dtype=torch.int32, device='cuda')
    ids = torch.randint(0, 99, (8, 5), generator=g).int().cuda()
    z, teacher = torch.randn(8, 99, generator=g).cuda(), torch.randn(8, 5, generator=g).cuda()
    calls = [(lambda q, k, v: qk_norm_rope(q, k, rope), (q, k, v)),
             (lambda q, k, v: qk_norm_rope_backward(q, k, q, k, rope)[:2], (q, k, v)),
             (lambda q, k, v: window_attention(q, k, v, 9, 1, lengths=lengths), (q, k, v)),
             (lambda q, k, v: (window_attention_token(q, k, v, lengths, 9, 1),), (q[:, 0].contiguous(), k, v)),
             (lambda z, i, t: distill_loss_grad(z, i, t), (z, ids, teacher))]
    for call, args in calls:
        want = call(*args)
        for moved in (args, tuple(odd(t) for t in args), args):
            for a, b in zip(want, call(*moved)):
                if args[0] is z and moved is not args:
                    assert (a - b).abs().max() <= (2 * 99 + (640 if a.dim() == 1 else 8)) * 2.0 ** -24
                else:
                    assert torch.equal(a, b)
        with pytest.raises(ValueError, match='one CUDA device'):
            call(args[0], args[1].cpu(), args[2])
    with pytest.raises(ValueError, match='aligned'):
        qk_norm_rope(q, k, odd(rope))
