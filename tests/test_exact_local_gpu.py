"""DUST's exact attention-internal errors against the draws that estimate them, for every kind.

The draws are independent, so their mean over n is e + noise / sqrt(n): with r the noise's norm over e's, the cosine c with e is
1 / sqrt(1 + r^2 / n), and 1 / c^2 - 1 = r^2 / n falls by 8 from n to 8 n where they converge to e itself. A bias b
leaves (b / |e|)^2 of it whatever n is. Half as much again is left for what a finite n scatters and the second order of sigma.
At gamma below 1 the credit of k, v, gate and ve decays with the distance of the later token, which is another number."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def measures(exact, drawn):
    e, d = exact.reshape(-1).double(), drawn.reshape(-1).double()
    c = torch.dot(e, d) / (e.norm() * d.norm())
    return (1 / c ** 2 - 1).item(), (torch.dot(e, d) / torch.dot(e, e)).item()


@pytest.mark.parametrize('kind', ['k', 'v', 'gate', 've'])
def test_draws_without_decay_converge_to_the_exact_errors(kind):
    from noise_b200.dust import exact_local_errors, local_errors
    from test_operators_chain_gpu import _capture
    w, cap = _capture(1, 128)
    g = torch.Generator().manual_seed(22)
    targets = {i: (torch.randn(1, 128, 512, generator=g) * 0.01).cuda() for i in range(8)}
    exact = exact_local_errors(w, cap, targets, (kind,))[kind]
    few = local_errors(w, cap, kind, 4096, targets, 0, 1, gamma=1.0)
    many = local_errors(w, cap, kind, 32768, targets, 0, 1, gamma=1.0)
    for site, e in exact.items():
        before, (left, gain) = measures(e, few[site])[0], measures(e, many[site])
        assert left <= 1.5 * before / 8 and left < 0.15, (site, before, left)
        assert abs(gain - 1) < 0.05, (site, gain)  # the part along e itself: noise / sqrt(n) on one direction of 65,536


def test_decay_is_not_what_the_exact_errors_have():
    """At the estimator's own gamma the part along the exact value errors is a sum of decayed credits: below 0.95 of it."""
    from noise_b200.dust import exact_local_errors, local_errors
    from test_operators_chain_gpu import _capture
    w, cap = _capture(1, 128)
    g = torch.Generator().manual_seed(22)
    targets = {i: (torch.randn(1, 128, 512, generator=g) * 0.01).cuda() for i in range(8)}
    exact = exact_local_errors(w, cap, targets, ('v',))['v']
    drawn = local_errors(w, cap, 'v', 32768, targets, 0, 1)
    for site, e in exact.items():
        assert 0.3 < measures(e, drawn[site])[1] < 0.95


def test_distillation_error_belongs_to_the_mean_over_targets():
    """Differences of the losses' sum over the tokens with a target give the error; the others' losses are there, their
    error is 0. The largest error per token is about 1, a step of 0.05 on fp32 logits leaves 1e-3 (h^2 / 6 of the third
    derivative, below 1, and 2^-20 of a loss of 20 over h)."""
    from noise_b200.dust import distill_error
    from test_operators_chain_gpu import _capture
    w, cap = _capture(1, 128)
    cap.y[0, 3] = -1
    g = torch.Generator().manual_seed(24)
    ids = torch.randint(0, 4096, (1, 128, 8), generator=g).cuda()
    t = (torch.randn(1, 128, 8, generator=g) * 2).cuda()
    loss, err = distill_error(cap, ids, t)
    assert loss[0, 3] > 0 and (err[0, 3] == 0).all()
    clean, h = cap.logits.clone(), 0.05
    for token in (0, 3, 77):
        at = int(ids[0, token, 0])
        ends = []
        for step in (h, -h):
            cap.logits.copy_(clean)
            cap.logits.view(128, 4096)[token, at] += step
            ends.append(distill_error(cap, ids, t)[0][cap.y >= 0].double().sum().item())
        assert abs((ends[0] - ends[1]) / (2 * h) - err[0, token, at].item()) < 2e-3, token
    cap.logits.copy_(clean)
