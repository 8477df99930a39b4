"""Outputs of qk_norm_rope that meet its inputs, each other or themselves: refused by the C entry before any CUDA call,
for exactly the layouts whose rows share an element. In place and interleaved views of one buffer stay open."""
import itertools
import random

import pytest
import torch

BASE = 1 << 24  # a 16-byte aligned address that no call here reads; views are offsets in elements from it


def block(B, T, H, Hk, D, q, k, qo, ko, rope=1 << 40, dtype=1, **kw):
    """Views are (offset, (stride b, t, h)) in elements of a 2-byte type."""
    from noise_b200 import _lib
    at = [BASE + 2 * v[0] for v in (q, k, qo, ko)]
    return _lib.QK_NORM.pack(dtype, 0, B, T, H, Hk, D, 1e-6, rope, 16, kw.get('positions', 0), kw.get('pos_stride', 0),
                             kw.get('wq', 0), 0, at[0], at[1], 0, 0, at[2], at[3], *q[1], *k[1], 0, 0, 0, 0, 0, 0,
                             *qo[1], *ko[1], 0, 0)


def refused(*args, **kw):
    from noise_b200 import _lib
    return _lib.load().noise_qk_norm_overlap(block(*args, **kw), 0)


def elements(v, B, T, heads, D):
    return [v[0] + b * v[1][0] + t * v[1][1] + h * v[1][2] + d
            for b, t, h, d in itertools.product(range(B), range(T), range(heads), range(D))]


Q, K = (0, (768, 256, 64)), (10000, (384, 128, 64))  # [2, 3, 4, 64] and [2, 3, 2, 64]


@pytest.mark.parametrize('q,k,qo,ko,want', [
    (Q, K, (20000, Q[1]), (30000, K[1]), 0),
    (Q, K, Q, K, 0),                                                  # in place
    ((0, (1536, 512, 64)), (256, (1536, 512, 64)), (0, (1536, 512, 64)), (256, (1536, 512, 64)), 0),    # in place, packed
    (Q, K, (20000, (1536, 512, 64)), (20256, (1536, 512, 64)), 0),    # two views of one packed result
    ((0, (1536, 512, 64)), (256, (1536, 512, 64)), (0, (1536, 512, 64)), (384, (1536, 512, 64)), 0),    # k into v's place
    (Q, K, Q, Q, 1),                                                  # both results in one place
    (Q, Q, Q, (30000, K[1]), 1),                                      # q and k are one tensor, q in place
    ((0, (1536, 512, 64)), (256, (1536, 512, 64)), (128, (1536, 512, 64)), (9000, K[1]), 1),            # rows shifted by two heads
    (Q, K, (256, Q[1]), K, 1),                                        # shifted by a token
    (Q, K, (8, Q[1]), K, 1),                                          # shifted within a row
    (Q, K, (20000, (768, 256, 32)), K, 1),                            # a result whose rows overlap
    (Q, K, (20000, (256, 256, 64)), K, 1),                            # a result whose sequences overlap
    (Q, K, (20000, (768, 768, 64)), K, 1),                            # the same step for sequences and tokens
    (Q, K, K, (30000, K[1]), 1),                                      # q's result over k
    (Q, (0, Q[1]), (20000, Q[1]), (0, Q[1]), 1),                      # k is q's first heads, in place: q's side reads them
])
def test_refused_and_open_layouts(q, k, qo, ko, want):
    assert refused(2, 3, 4, 2, 64, q, k, qo, ko) == want


def test_tables_weights_and_positions():
    free = ((20000, Q[1]), (30000, K[1]))
    assert not refused(2, 3, 4, 2, 64, Q, K, *free, wq=BASE + 2 * 19000)
    assert refused(2, 3, 4, 2, 64, Q, K, *free, wq=BASE + 2 * 20000 - 128)
    assert refused(2, 3, 4, 2, 64, Q, K, *free, rope=BASE + 2 * 30000)
    assert refused(2, 3, 4, 2, 64, Q, K, *free, positions=BASE + 2 * 20000 - 16, pos_stride=3)
    assert not refused(2, 3, 4, 2, 64, Q, K, *free, positions=BASE + 2 * 20000 - 24, pos_stride=3)


def test_the_entry_itself_refuses():
    from noise_b200 import _lib
    assert _lib.load().noise_qk_norm_rope(block(2, 3, 4, 2, 64, Q, K, (8, Q[1]), K), 0, None, 0, None) == 1


def test_against_the_sets_of_elements():
    """Small layouts of every kind, nested and not: refused exactly where the sets of elements meet, but for in place."""
    rng = random.Random(3)
    counts = [0, 0]
    for _ in range(4000):
        B, T, H, Hk, D = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 3), 16

        def view(heads):
            steps = [16 * rng.choice([1, 1, 2, 3])]
            for n in rng.sample([heads, T], 2):
                steps.append(max(16, steps[-1] * n + 16 * rng.choice([0, 0, 0, 1, -1])))
            if rng.random() < 0.2:
                rng.shuffle(steps)
            return 8 * rng.randint(0, 60), (steps[2], steps[1], steps[0])

        q, k, qo, ko = view(H), view(Hk), view(H), view(Hk)
        if rng.random() < 0.4:
            qo = q
        if rng.random() < 0.4:
            ko = k
        if rng.random() < 0.5:
            far = 5000
            qo, q = (qo[0] + far, qo[1]), (q[0] + far, q[1])
        sets = [elements(v, B, T, n, D) for v, n in ((q, H), (k, Hk), (qo, H), (ko, Hk))]
        want = any(len(set(s)) < len(s) for s in sets[2:]) or bool(set(sets[2]) & set(sets[3]))
        want |= bool(set(sets[2]) & set(sets[1])) or bool(set(sets[3]) & set(sets[0]))
        for i in (0, 1):
            want |= sets[i] != sets[2 + i] and bool(set(sets[i]) & set(sets[2 + i]))
        assert refused(B, T, H, Hk, D, q, k, qo, ko) == want, (B, T, H, Hk, q, k, qo, ko)
        counts[want] += 1
    assert min(counts) > 300


@pytest.mark.gpu
def test_the_call_refuses_and_open_layouts_are_right():
    from noise_b200.attention import qk_norm_rope
    g = torch.Generator().manual_seed(6)
    rope = torch.randn(16, 64, generator=g).cuda()
    qkv = torch.randn(2, 9, 8, 64, generator=g).bfloat16().cuda()
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    want = qk_norm_rope(q, k, rope)
    for out in ((q, q[:, :, :2]), (qkv[:, :, 1:5], k), (qkv[:, :, 4:], torch.empty_like(k)),
                (torch.empty(2, 10, 4, 64, dtype=q.dtype, device='cuda').as_strided(q.shape, (576, 64, 64, 1)), k)):
        with pytest.raises(ValueError, match='overlaps'):
            qk_norm_rope(q, k, rope, out=out)
    with pytest.raises(ValueError, match='overlaps'):
        qk_norm_rope(q, q, rope, out=(q, torch.empty_like(q)))
    into = qkv.clone()
    got = qk_norm_rope(into[:, :, :4], into[:, :, 4:6], rope, out=(into[:, :, :4], into[:, :, 6:]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(into[:, :, 4:6], k)
    qk_norm_rope(q, k, rope, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
