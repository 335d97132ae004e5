"""The ratio and e^d far from 1. Tolerances, in half steps of 2^-24: expf is off by 2 units in the last place at most (4), the weight by 1, and two
products by 1 each: 7 of each token's gradient. The KL term adds 1 - e^d, whose own subtraction is 1 more, a product and a sum: 10."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24


@pytest.mark.parametrize('n', [2001, 40000])
def test_far_ratios(n):
    from d1.policy_loss import policy_loss
    logp = torch.linspace(-60, 60, n, device='cuda')     # old is 0: the differences are exact
    old, adv = torch.zeros(n, device='cuda'), torch.ones(n, device='cuda')
    got = policy_loss(logp, old, adv, clip=1e30)
    want = -logp.double().exp() / n
    assert ((got.dlogp.double() - want).abs() <= 7 * HALF * want.abs()).all()
    assert abs(float(got.loss) - float(want.sum())) <= 8 * HALF * float(want.abs().sum())


@pytest.mark.parametrize('n', [2001, 40000])
def test_far_references(n):
    from d1.policy_loss import policy_loss
    ref = torch.linspace(-60, 60, n, device='cuda')
    zero = torch.zeros(n, device='cuda')
    got = policy_loss(zero, zero, zero, ref_logp=ref, kl_coef=1.0)
    d = ref.double()
    want = -torch.expm1(d) / n
    near = d.abs() < 0.5      # from the series: its sum's roundings are those of d, half of it at most
    assert ((got.dlogp.double() - want).abs() <= 10 * HALF * torch.where(near, d.abs(), d.exp() + 1) / n).all()
    kl = torch.expm1(d) - d
    assert abs(float(got.stats[1]) - float(kl.mean())) <= 10 * HALF * float((d.exp() + 1 + d.abs()).mean())
