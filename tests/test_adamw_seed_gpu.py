"""The seed of AdamW's 8-bit rounding: part of its state, and read at each step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def optimizer(seed, bits=8):
    from d1.adamw import AdamW
    g = torch.Generator(device='cuda').manual_seed(2)
    params = [torch.randn(n, device='cuda', generator=g) for n in (1000, 77)]
    grads = [torch.randn(p.shape, device='cuda', generator=g) for p in params]
    return AdamW(params, grads, state_bits=bits, seed=seed)


def bits_of(opt):
    return [t.view(torch.uint8).clone() for t in (opt.m, opt.v)] + [p.clone() for p in opt.params]


@pytest.mark.parametrize('bits', [8, 32])
def test_a_run_resumes_in_an_optimizer_with_another_seed(bits):
    a, b = optimizer(9, bits), optimizer(4, bits)
    for _ in range(2):
        a.step()
    b.load_state_dict(a.state_dict())
    for p, q in zip(b.params, a.params):
        p.copy_(q)
    for _ in range(3):
        a.step()
        b.step()
    assert b.seed == 9 and all(torch.equal(x, y) for x, y in zip(bits_of(a), bits_of(b)))


def test_states_without_a_seed_and_later_seeds():
    a, b, c = optimizer(9), optimizer(9), optimizer(4)
    state = a.state_dict()
    del state['seed']
    b.load_state_dict(state)
    assert b.seed == 9
    c.seed = 9
    for opt in (a, b, c):
        opt.step()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(bits_of(a), bits_of(b), bits_of(c)))
    with pytest.raises(ValueError):
        a.load_state_dict(dict(state, other=1))
