"""Policies that are far from the rollout's or the reference's: powers that pass fp32 beside an advantage or a coefficient of 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SHAPES = [(1, 64), (3, 1001), (40, 2000)]   # a cluster's batch, odd rows, two launches


def inputs(shape, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    new = lambda: torch.randn(shape, device='cuda', generator=g)
    old = -new().abs()
    return old + 0.1 * new(), old, new(), new().abs()


@pytest.mark.parametrize('shape', SHAPES)
def test_a_reference_that_is_only_watched(shape):
    """kl_coef 0: the KL term is reported (infinite) and takes no part."""
    from d1.policy_loss import policy_loss
    logp, old, adv, ent = inputs(shape)
    ref = logp.clone()
    ref[:, 5] = logp[:, 5] + 100
    want = policy_loss(logp, old, adv, entropy=ent, ent_coef=0.01)
    got = policy_loss(logp, old, adv, ref_logp=ref, entropy=ent, ent_coef=0.01, kl_coef=0.0)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.dlogp, want.dlogp) and torch.equal(got.dentropy, want.dentropy)
    assert got.stats[1].isinf() and torch.equal(got.stats[[0, 2, 3, 4]], want.stats[[0, 2, 3, 4]])
    assert not policy_loss(logp, old, adv, ref_logp=ref, kl_coef=0.1).dlogp[:, 5].isfinite().any()


@pytest.mark.parametrize('shape', SHAPES)
def test_no_advantage_where_the_ratio_passes(shape):
    """An advantage of exactly 0 (a group of equal rewards): e^100 times it is 0, for each token and for each row."""
    from d1.policy_loss import policy_loss
    logp, old, adv, _ = inputs(shape, 1)
    logp[:, 7] = old[:, 7] + 100
    adv[:, 7] = 0
    got = policy_loss(logp, old, adv)
    assert got.loss.isfinite() and (got.dlogp[:, 7] == 0).all() and got.dlogp.isfinite().all()
    logp[:, 7] = old[:, 7]                 # the same tokens with a ratio of 1 add as little
    near = policy_loss(logp, old, adv)
    assert torch.equal(got.loss, near.loss) and torch.equal(got.dlogp, near.dlogp)
    logp[0, 7] = old[0, 7] + 100
    row = adv.new_zeros(shape[0])
    got = policy_loss(logp, old, row)
    assert got.loss == 0 and (got.dlogp == 0).all()
    adv[0, 7] = -1
    assert policy_loss(logp, old, adv).dlogp[0, 7].isinf()
    adv[0, 7], logp[0, 7] = 0, float('nan')
    assert policy_loss(logp, old, adv).dlogp[0, 7].isnan()


def test_no_weight_of_an_infinite_entropy():
    from d1.policy_loss import policy_loss
    logp, old, adv, ent = inputs((2, 50), 2)
    want = policy_loss(logp, old, adv, entropy=ent)
    ent[0, 3] = float('inf')
    got = policy_loss(logp, old, adv, entropy=ent)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.dlogp, want.dlogp) and (got.dentropy == 0).all()
