"""The gradient norm and the clipped step where the gradients' squares pass the range of
fp32: the norm within 1e-6, as elsewhere, and gradients that clipping brings back to size
are taken as such (fp32 roundings of the factor and the products, 2^-21 of m and of the
update, approximate root and reciprocal included)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('grad_type', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('scale', [1e18, 1e19, 3e19, 1e25, 1e34])
def test_large_gradients_are_clipped(scale, grad_type, bits):
    from d1.adamw import AdamW
    g = torch.Generator(device='cuda').manual_seed(3)
    sizes = [300, 129, 70000, 1, 4096]
    grads = [(scale * torch.randn(n, device='cuda', generator=g)).to(grad_type) for n in sizes]
    grads[3][0] = 1.0
    params = [torch.zeros(n, device='cuda') for n in sizes]
    opt = AdamW(params, grads, lr=1e-2, weight_decay=0.0, state_bits=bits, max_norm=0.5)
    opt.step()
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm
    for i, (p, x) in enumerate(zip(params, grads)):
        want = x.double() * (0.5 / norm)
        m, v = opt.moments(i)
        if bits == 32:
            assert ((m.double() - 0.1 * want).abs() <= 2.0 ** -21 * want.abs() + 1e-38).all()
        big = want.abs() > 1e-6          # eps no longer shows
        assert big.sum() > 0.9 * big.numel() or sizes[i] == 1
        assert ((p.double() + 1e-2 * want.sign()).abs()[big] <= 1e-2 * (2e-2 + 2.0 ** -18)).all()


def test_what_is_not_finite_stays_so():
    from d1.adamw import AdamW
    for bad in (math.inf, math.nan):
        p, g = torch.zeros(1000, device='cuda'), torch.full((1000,), 1e30, device='cuda')
        g[500] = bad
        opt = AdamW([p], [g], max_norm=1.0)
        opt.step()
        assert not opt.grad_norm.isfinite() and p[500].isnan()
