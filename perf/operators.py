"""Timing cases of the language-model operators: per-head norms with rotation (`qk_norm_rope`), sliding-window
attention with sinks (`window_attention`, its gradient and its single-token form) and the distillation
loss from a teacher's top logits (`distill_loss` and its gradient).

`run` computes a case in elementary torch operations in 32 bits, or, with `own` set, through noise_b200.
`exact` gives the same outputs from the operators' definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = torch.finfo(torch.float32).eps  # the norms' epsilon


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one block's queries and keys of a training batch, as views of the packed projection
        dict(name='norm-block', op='norm', grad=False, dtype='bf16', B=8, T=2048, H=8, Hk=8, D=64, weights=False,
             order='rotate_norm', packed=True, positions=False),
        # the newest tokens of 32 sequences that generate, each at its own position: latency
        dict(name='norm-token', op='norm', grad=False, dtype='bf16', B=32, T=1, H=32, Hk=8, D=128, weights=True,
             order='norm_rotate', packed=True, positions=True),
        # a training step with learned norm weights and grouped heads of an odd width, odd length
        dict(name='norm-train', op='norm', grad=True, dtype='bf16', B=6, T=3777, H=12, Hk=4, D=96, weights=True,
             order='norm_rotate', packed=True, positions=False),
        # the fixed model's attention over one training batch, with four sinks
        dict(name='attend-block', op='attend', grad=False, dtype='bf16', B=8, Tq=2048, Tk=2048, H=8, Hk=8, D=64,
             window=1024, sinks=4, ragged=False),
        # one long prompt with grouped heads
        dict(name='attend-long', op='attend', grad=False, dtype='fp16', B=1, Tq=16384, Tk=16384, H=16, Hk=4, D=128,
             window=4096, sinks=64, ragged=False),
        # forward and backward of the fixed model's attention
        dict(name='attend-train', op='attend', grad=True, dtype='bf16', B=8, Tq=2048, Tk=2048, H=8, Hk=8, D=64,
             window=1024, sinks=4, ragged=False),
        # a padded batch of odd lengths with grouped heads, forward and backward
        dict(name='attend-train-ragged', op='attend', grad=True, dtype='bf16', B=4, Tq=1999, Tk=1999, H=12, Hk=4, D=128,
             window=511, sinks=16, ragged=True),
        # one sequence that generates: the smallest call of a server
        dict(name='token-one', op='token', dtype='bf16', B=1, Tk=2048, H=8, Hk=8, D=64, window=1024, sinks=4),
        # 64 sequences that generate, long caches, grouped heads
        dict(name='token-many', op='token', dtype='bf16', B=64, Tk=8192, H=32, Hk=8, D=128, window=4096, sinks=4),
        # the head of one training batch: loss and gradient of the soft-capped logits
        dict(name='distill-head', op='distill', form='loss_grad', dtype='fp32', teacher='fp32', N=16384, V=4096, K=32,
             tau=1.0, cap=15.0),
        # a large odd vocabulary in bf16: loss, then the gradient from the losses' own gradient
        dict(name='distill-wide', op='distill', form='backward', dtype='bf16', teacher='bf16', N=2047, V=50257, K=64,
             tau=2.0, cap=0.0),
        # the losses alone of a few rows of a very large vocabulary
        dict(name='distill-few', op='distill', form='loss', dtype='bf16', teacher='fp32', N=8, V=131072, K=128, tau=1.0,
             cap=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'attend', 'attend', 'attend', 'token', 'token', 'distill', 'distill', 'distill'])
    if op == 'norm':
        hk = rng.choice([1, 2, 4, 8])
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        h = hk * rng.choice([1, 2, 3, 4])
        t = _log(rng, 1, 8192)
        b = max(1, min(_log(rng, 1, 64), 48_000_000 // (t * (h + hk) * d)))
        return dict(op=op, grad=rng.random() < 0.5, dtype=rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), B=b, T=t, H=h, Hk=hk,
                    D=d, weights=rng.random() < 0.5, order=rng.choice(['rotate_norm', 'norm_rotate']),
                    packed=rng.random() < 0.7, positions=rng.random() < 0.5)
    if op == 'attend':
        d = rng.choice([64, 64, 128, 128, 40, 96])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 2, 3, 4])
        grad = rng.random() < 0.5
        tk = _log(rng, 17, 8192)
        tq = tk if rng.random() < 0.7 else rng.randint(1, tk)
        window = min(tk, _log(rng, 16, 4096))
        b = max(1, min(rng.randint(1, 8), 300_000_000 // (tq * min(tk, window + 64) * h)))
        return dict(op=op, grad=grad, dtype='bf16' if grad else rng.choice(['bf16', 'fp16']), B=b, Tq=tq, Tk=tk, H=h, Hk=hk,
                    D=d, window=window, sinks=rng.choice([0, 1, 4, 16, 64, 150]), ragged=rng.random() < 0.4)
    if op == 'token':
        hk = rng.choice([1, 2, 4, 8])
        tk = _log(rng, 64, 16384)
        b = max(1, min(_log(rng, 1, 64), 500_000 // tk))
        return dict(op=op, dtype=rng.choice(['bf16', 'fp16']), B=b, Tk=tk, H=hk * rng.choice([1, 2, 4, 8]), Hk=hk,
                    D=rng.choice([64, 64, 128, 128, 96]), window=_log(rng, 16, tk), sinks=rng.choice([0, 1, 4, 16, 64]))
    v, form = _log(rng, 1000, 131072), rng.choice(['loss', 'backward', 'loss_grad'])
    # gradients of fp16 logits come from a scaled loss: the losses' own gradient carries the scale
    return dict(op=op, form=form, dtype=rng.choice(['bf16', 'fp32', 'bf16' if form == 'loss_grad' else 'fp16']),
                teacher=rng.choice(['bf16', 'fp32']), N=max(1, min(_log(rng, 1, 16384), 60_000_000 // v)), V=v,
                K=rng.choice([1, 5, 16, 32, 64, 100, 256]), tau=rng.choice([1.0, 1.0, 2.0, 0.7]),
                cap=rng.choice([0.0, 0.0, 15.0, 30.0]))


def _lengths(case, seed):
    """Valid tokens of each sequence, on the host: some full, some short, one of a larger batch empty."""
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    b, t = case['B'], case['Tk']
    n = (t * (0.35 + 0.65 * torch.rand(b, generator=g))).long().clamp(1, t)
    n[0] = t
    if b > 2 and case['op'] == 'attend':
        n[1] = 0
    return n


def _pairs(case, lengths):
    """Visible (query, key) pairs of one head, summed over the batch."""
    offset, total = case['Tk'] - case['Tq'], 0
    for n in lengths:
        p = torch.arange(offset, max(offset, min(n, case['Tk'])), dtype=torch.float64)
        lo = (p - case['window']).clamp(min=0)
        total += int((p + 1 - lo + lo.clamp(max=case['sinks'])).sum())
    return total


def work(case):
    op, size = case['op'], {'bf16': 2, 'fp16': 2, 'fp32': 4}
    if op == 'norm':
        n = case['B'] * case['T'] * (case['H'] + case['Hk']) * case['D']
        io, flops = 2, 8
        if case['grad']:
            io, flops = 4, 26
        return dict(bytes=io * n * size[case['dtype']], flops=flops * n)
    if op == 'attend':
        lengths = _lengths(case, 0).tolist() if case['ragged'] else [case['Tk']] * case['B']
        rows_q, rows_k = case['B'] * case['Tq'] * case['H'], case['B'] * case['Tk'] * case['Hk']
        pairs = _pairs(case, lengths) * case['H'] * case['D']
        nbytes, flops = 2 * case['D'] * (2 * rows_q + 2 * rows_k), 4 * pairs
        if case['grad']:
            nbytes += 2 * case['D'] * (2 * rows_q + 2 * rows_k)
            flops += 10 * pairs
        else:
            nbytes += 4 * rows_q
        return dict(bytes=nbytes, flops=flops)
    if op == 'token':
        keys = 0
        for n in _lengths(case, 0).tolist():
            lo = max(0, n - 1 - case['window'])
            keys += n - lo + min(case['sinks'], lo)
        return dict(bytes=2 * case['D'] * (2 * keys * case['Hk'] + 2 * case['B'] * case['H']),
                    flops=4 * keys * case['H'] * case['D'])
    n = case['N'] * case['V']
    io = 1 if case['form'] == 'loss' else 2
    return dict(bytes=n * io * size[case['dtype']] + case['N'] * (case['K'] * (4 + size[case['teacher']]) + 4),
                flops=n * (4 if io == 1 else 8))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _rope(length, dim, device):
    """[length, dim] cos | sin in fp32, rounded to bf16 as the model's tables are."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.outer(torch.arange(length, dtype=torch.float64), inv)
    return torch.cat([ang.cos(), ang.sin()], 1).bfloat16().float().to(device).contiguous()


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed * 1_000_003 + 11)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).mul_(scale).to(dtype)

    op, dt = case['op'], DTYPES[case['dtype']]
    st = dict(case=dict(case))
    if op == 'norm':
        b, t, h, hk, d = (case[n] for n in ('B', 'T', 'H', 'Hk', 'D'))
        if case['packed']:  # q | k | v of one projection
            qkv = normal(b, t, h + 2 * hk, d, dtype=dt, scale=1.5)
            st['q'], st['k'] = qkv[:, :, :h], qkv[:, :, h:h + hk]
        else:
            st['q'], st['k'] = normal(b, t, h, d, dtype=dt, scale=1.5), normal(b, t, hk, d, dtype=dt, scale=1.5)
        limit = t if not case['positions'] else t + 4096
        st['rope'] = _rope(limit, d, dev)
        st['positions'] = None
        if case['positions']:
            start = torch.randint(0, 4097, (b, 1), device=dev, generator=g)
            st['positions'] = (start + torch.arange(t, device=dev)).clamp(max=limit - 1).to(torch.int32)
        st['wq'] = st['wk'] = None
        if case['weights']:
            st['wq'], st['wk'] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        if case['grad']:
            st['dq'], st['dk'] = normal(b, t, h, d, dtype=dt, scale=0.1), normal(b, t, hk, d, dtype=dt, scale=0.1)
    elif op == 'attend':
        b, tq, tk, h, hk, d = (case[n] for n in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
        st['q'] = normal(b, tq, h, d, dtype=dt)
        st['k'] = normal(b, tk, hk, d, dtype=dt)
        st['v'] = normal(b, tk, hk, d, dtype=dt)
        st['lengths'] = _lengths(case, seed).to(dev, torch.int32) if case['ragged'] else None
        st['dout'] = normal(b, tq, h, d, dtype=dt, scale=0.1) if case['grad'] else None
        st['status'] = torch.zeros(1, dtype=torch.int32, device=dev)
    elif op == 'token':
        b, tk, h, hk, d = (case[n] for n in ('B', 'Tk', 'H', 'Hk', 'D'))
        st['q'] = normal(b, h, d, dtype=dt)
        st['k'] = torch.empty(b, tk, hk, d, dtype=dt, device=dev).normal_(generator=g)
        st['v'] = torch.empty(b, tk, hk, d, dtype=dt, device=dev).normal_(generator=g)
        st['lengths'] = _lengths(case, seed).to(dev, torch.int32)
    else:
        n, v, k = case['N'], case['V'], case['K']
        st['logits'] = torch.empty(n, v, dtype=dt, device=dev).normal_(0, 3.0, generator=g)
        # a teacher's top entries: falling logits, ids without repeats; some rows hold fewer than K
        st['teacher'] = (12 - 2.5 * torch.rand(n, k, device=dev, generator=g).cumsum(1)).to(DTYPES[case['teacher']])
        start = torch.randint(0, v, (n, 1), device=dev, generator=g)
        stride = max(1, v // k)
        ids = (start + stride * torch.arange(k, device=dev)) % v
        kept = torch.randint(max(1, k // 2), k + 1, (n, 1), device=dev, generator=g)
        st['ids'] = ids.masked_fill(torch.arange(k, device=dev) >= kept, -1).to(torch.int32).contiguous()
        scale = 1024.0 if case['dtype'] == 'fp16' else 1.0 / n
        st['dloss'] = torch.rand(n, device=dev, generator=g).mul_(scale) if case['form'] == 'backward' else None
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state['case']['op']
    if own:
        return {'norm': _own_norm, 'attend': _own_attend, 'token': _own_token, 'distill': _own_distill}[op](state)
    return {'norm': _plain_norm, 'attend': _plain_attend, 'token': _plain_token, 'distill': _plain_distill}[op](state)


def _own_norm(st):
    from noise_b200.attention import qk_norm_rope, qk_norm_rope_backward
    case = st['case']
    kw = dict(positions=st['positions'], q_weight=st['wq'], k_weight=st['wk'], order=case['order'])
    y = qk_norm_rope(st['q'], st['k'], st['rope'], **kw)
    if not case['grad']:
        return y
    grads = qk_norm_rope_backward(st['dq'], st['dk'], st['q'], st['k'], st['rope'], **kw)
    return tuple(y) + tuple(t for t in grads if t is not None)


def _own_attend(st):
    from noise_b200.attention import window_attention, window_attention_backward
    case = st['case']
    kw = dict(lengths=st['lengths'], status=st['status'])
    out, lse = window_attention(st['q'], st['k'], st['v'], case['window'], case['sinks'], **kw)
    if case['grad']:
        return (out, *window_attention_backward(st['dout'], st['q'], st['k'], st['v'], out, lse, case['window'],
                                                case['sinks'], **kw))
    return (out,) if case['ragged'] else (out, lse)


def _own_token(st):
    from noise_b200.attention import window_attention_token
    return window_attention_token(st['q'], st['k'], st['v'], st['lengths'], st['case']['window'], st['case']['sinks'])


def _own_distill(st):
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    case = st['case']
    args, kw = (st['logits'], st['ids'], st['teacher']), dict(temperature=case['tau'], softcap=case['cap'])
    if case['form'] == 'loss':
        return distill_loss(*args, **kw)[0]
    if case['form'] == 'loss_grad':
        return distill_loss_grad(*args, **kw)
    loss, lse = distill_loss(*args, **kw)
    return loss, distill_backward(st['dloss'], *args, lse, **kw)


def _turn(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def _turn_back(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_norm(st):
    case, outs, grads, wgrads = st['case'], [], [], []
    table = st['rope'][st['positions'].long()] if st['positions'] is not None else st['rope'][None, :case['T']]
    c, s = (h[:, :, None] for h in table.chunk(2, -1))
    for x, w, dy in ((st['q'], st['wq'], st.get('dq')), (st['k'], st['wk'], st.get('dk'))):
        rotate_first = case['order'] == 'rotate_norm'
        u = x.float()
        if rotate_first:
            u = _turn(u, c, s)
        r = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
        n = u * r
        y = n if w is None else n * w
        outs.append((y if rotate_first else _turn(y, c, s)).to(x.dtype))
        if dy is None:
            continue
        dz = dy.float() if rotate_first else _turn_back(dy.float(), c, s)
        if w is not None:
            wgrads.append((dz * n).reshape(-1, case['D']).sum(0))
            dz = dz * w
        du = r * (dz - n * (n * dz).mean(-1, keepdim=True))
        grads.append((_turn_back(du, c, s) if rotate_first else du).to(x.dtype))
    return tuple(outs + grads + wgrads)


def _plain_attend(st):
    case = st['case']
    b, tq, tk, h, hk, d = (case[n] for n in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
    window, sinks, grp, dev = case['window'], case['sinks'], case['H'] // case['Hk'], st['q'].device
    scale, offset = d ** -0.5, case['Tk'] - case['Tq']
    rows = torch.full((b,), tk, device=dev) if st['lengths'] is None else st['lengths'].long()

    def heads(x):  # [B, T, heads, D] -> [B, Hk, group, T, D] in 32 bits
        return x.float().view(b, x.shape[1], hk, -1, d).permute(0, 2, 3, 1, 4)

    q, k, v = heads(st['q']), heads(st['k']), heads(st['v'])
    out = torch.empty(b, hk, grp, tq, d, device=dev)
    lse = torch.empty(b, hk, grp, tq, device=dev)
    if case['grad']:
        do = heads(st['dout'])
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    for i0 in range(0, tq, 512):
        i1 = min(tq, i0 + 512)
        lo, hi = max(0, offset + i0 - window), offset + i1
        first = min(sinks, lo)  # sinks that the window's own keys do not hold
        keys = torch.cat([torch.arange(first, device=dev), torch.arange(lo, hi, device=dev)])
        p = torch.arange(offset + i0, offset + i1, device=dev)[:, None]
        seen = (keys <= p) & ((p - keys <= window) | (keys < sinks))
        seen = (seen & (p < rows[:, None, None]))[:, None, None]  # [B, 1, 1, q, keys]

        def span(x):
            return torch.cat([x[..., :first, :], x[..., lo:hi, :]], -2) if first else x[..., lo:hi, :]

        kk, vv, qq = span(k), span(v), q[..., i0:i1, :]
        s = torch.where(seen, qq @ kk.transpose(-1, -2) * scale, -torch.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-1e30)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        prob = e / total.clamp(min=1e-30)
        out[..., i0:i1, :] = prob @ vv
        lse[..., i0:i1] = (top + torch.log(total))[..., 0]
        if case['grad']:
            dd = torch.where(seen.any(-1, keepdim=True), do[..., i0:i1, :], 0)
            dp = dd @ vv.transpose(-1, -2)
            ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * scale
            dq[..., i0:i1, :] = ds @ kk
            for acc, part in ((dk, ds.transpose(-1, -2) @ qq), (dv, prob.transpose(-1, -2) @ dd)):
                part = part.sum(2, keepdim=True)
                acc[..., :first, :] += part[..., :first, :]
                acc[..., lo:hi, :] += part[..., first:, :]

    def back(x):
        return x.permute(0, 3, 1, 2, 4).reshape(b, x.shape[3], -1, d).to(st['q'].dtype)

    if case['grad']:
        return back(out), back(dq), back(dk), back(dv)
    return (back(out),) if case['ragged'] else (back(out), lse.reshape(b, h, tq))


def _plain_token(st):
    case = st['case']
    b, tk, h, hk, d = (case[n] for n in ('B', 'Tk', 'H', 'Hk', 'D'))
    q, keys = st['q'].float().view(b, hk, h // hk, d), torch.arange(tk, device=st['q'].device)
    p = st['lengths'].long()[:, None] - 1
    seen = ((keys <= p) & ((p - keys <= case['window']) | (keys < case['sinks'])))[:, None, None]
    s = q @ st['k'].float().permute(0, 2, 3, 1) * d ** -0.5
    s = torch.where(seen, s, -torch.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    out = (e / e.sum(-1, keepdim=True)) @ st['v'].float().permute(0, 2, 1, 3)
    return out.view(b, h, d).to(st['q'].dtype)


def _plain_distill(st):
    case, tau, cap = st['case'], st['case']['tau'], st['case']['cap']
    z = st['logits'].float()
    if cap:
        th = torch.tanh(z / cap)
        s = th * (cap / tau)
    else:
        s = z / tau
    top = s.amax(1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(1, keepdim=True)
    valid = st['ids'] >= 0
    ids = st['ids'].long().clamp(min=0)
    t = torch.where(valid, st['teacher'].float() / tau, -torch.inf)
    t = t - t.amax(1, keepdim=True)
    pe = torch.exp(t)
    mass = pe.sum(1, keepdim=True)
    prob = pe / mass
    logp = torch.where(valid, t, 0) - torch.log(mass)
    loss = tau * tau * (prob * (logp - s.gather(1, ids) + top + torch.log(total))).sum(1)
    if case['form'] == 'loss':
        return loss
    grad = (e / total).scatter_add_(1, ids, -prob)
    grad = grad * tau if not cap else grad * tau * (1 - th * th)
    if st['dloss'] is not None:
        grad = grad * st['dloss'][:, None]
    return loss, grad.to(st['logits'].dtype)


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {'norm': _exact_norm, 'attend': _exact_attend, 'token': _exact_token, 'distill': _exact_distill}[case['op']](
        case, st)


def _exact_norm(case, st):
    d = case['D']
    pos = st['positions'].long() if st['positions'] is not None else torch.arange(case['T'], device='cuda')[None]
    cs = st['rope'].double()[pos]
    turn = torch.complex(cs[..., :d // 2], -cs[..., d // 2:])[:, :, None]  # (a + ib)(c - is)
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((st['q'], st['wq'], st.get('dq')), (st['k'], st['wk'], st.get('dk'))):
        x = x.double().requires_grad_(case['grad'])
        w = None if w is None else w.double().requires_grad_(case['grad'])

        def rotate(u):
            u = torch.complex(u[..., :d // 2], u[..., d // 2:]) * turn
            return torch.cat([u.real, u.imag], -1)

        def norm(u):
            u = u / torch.sqrt(u.square().sum(-1, keepdim=True) / d + EPS)
            return u if w is None else u * w

        y = norm(rotate(x)) if case['order'] == 'rotate_norm' else rotate(norm(x))
        outs.append(y.detach())
        if case['grad']:
            found = torch.autograd.grad(y, [x] if w is None else [x, w], dy.double())
            grads.append(found[0])
            wgrads += found[1:]
    return tuple(outs + grads + wgrads)


def _exact_attend(case, st):
    b, tq, tk, h, hk, d = (case[n] for n in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
    if b * h * float(tq) * tk > 6e9:
        return None
    offset = tk - tq
    p, j = torch.arange(offset, tk, device='cuda')[:, None], torch.arange(tk, device='cuda')[None]
    base = (j <= p) & ((j >= p - case['window']) | (j < case['sinks']))
    out = torch.zeros(b, tq, h, d, dtype=torch.float64, device='cuda')
    lse = torch.full((b, h, tq), -torch.inf, dtype=torch.float64, device='cuda')
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(b, tk, hk, d, dtype=torch.float64, device='cuda') for _ in range(2))
    for bi in range(b):
        n = tk if st['lengths'] is None else int(st['lengths'][bi])
        rows = n - offset
        if rows <= 0:
            continue
        hidden = ~base[:rows, :n]
        for hi in range(h):
            kv = hi // (h // hk)
            leaves = [st['q'][bi, :rows, hi].double(), st['k'][bi, :n, kv].double(), st['v'][bi, :n, kv].double()]
            for x in leaves:
                x.requires_grad_(case['grad'])
            s = (leaves[0] @ leaves[1].T / math.sqrt(d)).masked_fill(hidden, -torch.inf)
            o = torch.softmax(s, 1) @ leaves[2]
            out[bi, :rows, hi] = o.detach()
            if case['grad']:
                gq, gk, gv = torch.autograd.grad(o, leaves, st['dout'][bi, :rows, hi].double())
                dq[bi, :rows, hi] = gq
                dk[bi, :n, kv] += gk
                dv[bi, :n, kv] += gv
            else:
                lse[bi, hi, :rows] = torch.logsumexp(s, 1)
            del s, o
    if case['grad']:
        return out, dq, dk, dv
    return (out,) if case['ragged'] else (out, lse)


def _exact_token(case, st):
    out = torch.zeros(case['B'], case['H'], case['D'], dtype=torch.float64, device='cuda')
    group = case['H'] // case['Hk']
    for bi in range(case['B']):
        n = int(st['lengths'][bi])
        lo = max(0, n - 1 - case['window'])
        keep = list(range(min(case['sinks'], lo))) + list(range(lo, n))
        k, v = st['k'][bi, keep].double(), st['v'][bi, keep].double()
        q = st['q'][bi].double().view(case['Hk'], group, case['D'])
        a = torch.softmax(torch.einsum('kgd,tkd->kgt', q, k) / math.sqrt(case['D']), -1)
        out[bi] = torch.einsum('kgt,tkd->kgd', a, v).reshape(case['H'], case['D'])
    return out


def _exact_distill(case, st):
    n, tau, cap = case['N'], case['tau'], case['cap']
    want_grad = case['form'] != 'loss'
    losses, grads = [], []
    step = max(1, 100_000_000 // case['V'])
    for i in range(0, n, step):
        z = st['logits'][i:i + step].double().requires_grad_(want_grad)
        s = (cap * torch.tanh(z / cap) if cap else z) / tau
        logq = torch.log_softmax(s, 1)
        ids = st['ids'][i:i + step].long()
        t = (st['teacher'][i:i + step].double() / tau).masked_fill(ids < 0, -torch.inf)
        logp = torch.log_softmax(t, 1)
        terms = logp.exp() * (logp.clamp(min=-1e300) - logq.gather(1, ids.clamp(min=0)))
        loss = tau ** 2 * terms.sum(1)
        losses.append(loss.detach())
        if want_grad:
            up = torch.ones_like(loss) if st['dloss'] is None else st['dloss'][i:i + step].double()
            grads.append(torch.autograd.grad(loss, z, up)[0])
    loss = torch.cat(losses)
    return (loss, torch.cat(grads)) if want_grad else loss
