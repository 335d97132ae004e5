"""The C entry of the policy loss refuses bad arguments before any CUDA call (checked without a GPU), and
the Python call refuses tensors that are not on one."""
import pytest
import torch

BAD = 9002
P = 1 << 20  # an aligned address that is never read


@pytest.fixture(scope='module')
def lib():
    from d1 import _lib
    return _lib.library()


def args(**change):
    good = dict(logp=P, l1=8, old=2 * P, l2=8, adv=3 * P, l3=8, per_row=0, ref=4 * P, l4=8, entropy=5 * P, l5=8, mask=6 * P, l6=8, rows=3, length=8,
                low=0.2, high=0.2, kl=0.1, ent=0.01, by_row=0, loss=P, stats=P, dlogp=7 * P, dentropy=8 * P, work=P, s=None)
    return dict(good, **change).values()


def test_refusals(lib):
    nan = float('nan')
    for k, v in dict(logp=None, old=None, adv=None, l1=-1, l2=-1, l3=-1, l4=-1, l5=-1, l6=-1, rows=-1, length=-1, low=-0.1, high=nan, kl=nan, ent=nan,
                     logp_=P + 2, ref=4 * P + 1, entropy=5 * P + 2, dlogp=7 * P + 2, loss=P + 1, stats=P + 1, work=P + 4).items():
        assert lib.d1_policy_loss(*args(**{k.rstrip('_'): v})) == BAD, k
    for at in (P, 2 * P + 4, 3 * P + 92, 4 * P, 5 * P, 6 * P + 20, 8 * P):   # what the call reads, or the other gradient
        assert lib.d1_policy_loss(*args(dlogp=at)) == BAD, at
    assert lib.d1_policy_loss(*args(length=1 << 31)) == BAD and lib.d1_policy_loss(*args(rows=1 << 41)) == BAD
    assert lib.d1_policy_loss(*args(rows=3000, work=None)) == BAD             # needs its work buffer
    assert lib.d1_policy_loss(*args(rows=1 << 29, l1=0)) == BAD               # a mask of 2^32 tokens


def test_work_bytes(lib):
    size = lib.d1_policy_loss_work_bytes
    assert size(-1, 1) == size(1, -1) == size(1, 1 << 31) == size(1 << 41, 1) == -1
    assert size(0, 5) == size(1, 32768) == size(2048, 16) == 0
    assert size(2049, 1) > 4 * 2049 and size(1, 32769) > 0


def test_rows_without_tokens_need_no_work_buffer(lib):
    assert lib.d1_policy_loss_work_bytes(100000, 0) == 0


def test_host_tensors_are_refused():
    from d1.policy_loss import policy_loss
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        policy_loss(x, x, x)
