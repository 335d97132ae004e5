"""The average form's gates at finite magnitudes up to where they leave fp32, and the same for the sum form's decays.

Tolerances, in half steps (2^-24 of the value): 2^x is off by 4 (ex2.approx: 2^-22), its correction by 2, the reciprocal by 2, 1 + E and a product by
1 each; the state's product, the input's and their sum by 3 more: 16 in all for one step. A sum form's decay (expf) is off by 4."""
import pytest
import torch

from test_gated_scan_gpu import check, factors

pytestmark = pytest.mark.gpu
STEP = 16 * 2.0 ** -24
TINY = 2.0 ** -126   # below it fp32 has fewer bits: products are 0 or as they round


def gates(most):
    g = torch.Generator(device='cuda').manual_seed(7)
    near = torch.randn(2048, device='cuda', generator=g) * 3
    far = (torch.rand(4096, device='cuda', generator=g) * 2 - 1) * most
    ends = torch.tensor([0.0, -0.0, 1e-30, 20.0, -20.0, 60.0, -60.0, 80.0, -80.0, 87.0, -87.0], device='cuda')
    return torch.cat((near, far, ends))


@pytest.mark.parametrize('form', ['average', 'sum'])
def test_a_decay_alone(form):
    """x = 0: y = a h0. And h0 = 0: y = (1 - a) x."""
    from d1.gated_scan import gated_scan
    gate = gates(87.0).view(1, 1, -1)
    n = gate.shape[-1]
    a, w = factors(gate, form)
    zero, one = torch.zeros(1, 1, n, device='cuda'), torch.ones(1, 1, n, device='cuda')
    y, _ = gated_scan(zero, gate, one[0], form=form)
    assert ((y.double() - a).abs() <= STEP * a + TINY).all()
    y, _ = gated_scan(one, gate, form=form)
    assert ((y.double() - w).abs() <= STEP * w + TINY).all()


def test_the_gates_gradient():
    """dgate = D (h - x) a (1 - a): each factor as above."""
    from d1.gated_scan import gated_scan, gated_scan_backward
    gate = gates(42.0).view(1, 1, -1)       # a (1 - a) a normal number
    n = gate.shape[-1]
    a, w = factors(gate, 'average')
    zero, one = torch.zeros(1, 1, n, device='cuda'), torch.ones(1, 1, n, device='cuda')
    y, _ = gated_scan(zero, gate, one[0])
    dx, dgate, dh0 = gated_scan_backward(one, zero, gate, y, one[0])
    assert ((dx.double() - w).abs() <= STEP * w).all() and ((dh0.double() - a).abs() <= STEP * a).all()
    assert ((dgate.double() - a * w).abs() <= 2 * STEP * a * w).all()


@pytest.mark.parametrize('T, B, D', [(40, 3, 34), (600, 1, 20)])
def test_rollouts_of_far_gates(T, B, D):
    g = torch.Generator(device='cuda').manual_seed(3)
    new = lambda *s: torch.randn(s, device='cuda', generator=g)
    gate = (torch.rand(T, B, D, device='cuda', generator=g) * 2 - 1) * 40
    check(new(T, B, D), gate, new(B, D), None, new(T, B, D), new(B, D), 'average')
