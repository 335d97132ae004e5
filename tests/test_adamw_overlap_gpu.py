"""AdamW refuses tensors that a step would write twice, or read while it writes them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_shared_memory_is_refused():
    from d1.adamw import AdamW
    flat, grad = torch.zeros(1000, device='cuda'), torch.zeros(1000, device='cuda')
    copy = torch.zeros(1000, device='cuda', dtype=torch.bfloat16)
    p, q, g, h = flat[:500], flat[500:], grad[:500], grad[500:]
    for bad in (lambda: AdamW([p, p], [g, h]), lambda: AdamW([p, flat[499:999]], [g, h]), lambda: AdamW([p, q], [g, p]),
                lambda: AdamW([p, q], [g, flat[100:600]]), lambda: AdamW([p, q], [g, h], copies=[copy[:500], copy[499:999]]),
                lambda: AdamW([p], [g], copies=[flat.view(torch.bfloat16)[:500]])):
        with pytest.raises(ValueError):
            bad()
    opt = AdamW([p, q], [g, g], copies=[copy[:500], copy[500:]])   # one gradient for two parameters is read only
    opt.step()
    with pytest.raises(ValueError):
        opt.set_grads([g, flat[400:900]])
    opt.set_grads([g, h])
    opt.step()
    assert int(opt.step_dev) == 2
