"""The training operators under another default type of torch than float32: the
same bits as under float32."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def results():
    from d1.adamw import AdamW
    from d1.imitation import JointHead
    from d1.layer_norm import layer_norm, layer_norm_backward
    from d1.token_logprob import token_logprob, token_logprob_backward
    f32 = dict(dtype=torch.float32, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(300, 40, generator=g, **f32)
    w, dlogp = torch.randn(40, generator=g, **f32), torch.randn(300, generator=g, **f32)
    y, mean, rstd = layer_norm(x, w)
    out = [y, mean, rstd, *layer_norm_backward(y, x, mean, rstd, w)]
    tokens = torch.arange(300, device='cuda') % 40
    r = token_logprob(x, tokens, top=3)
    out += [*r, token_logprob_backward(x, tokens, r.stats, r.entropy, dlogp, dlogp)]
    for bits in (32, 8):
        p, grad = torch.randn(1000, generator=g, **f32), torch.randn(1000, generator=g, **f32)
        opt = AdamW([p], [grad], state_bits=bits, max_norm=1.0)
        opt.step()
        out += [p, opt.grad_norm, *opt.moments(0)]
    h = torch.randn(64, 512, generator=g, **f32).bfloat16()
    legal = torch.full((64,), 0x3ff, dtype=torch.int16, device='cuda')
    head = JointHead(seed=1, ent_coef=0.01)
    out += [*head.update(h, torch.zeros(64, dtype=torch.int64, device='cuda'), legal), *head.params.values()]
    return out


@pytest.mark.parametrize('default', [torch.float64, torch.bfloat16])
def test_the_same_bits_under_another_default_type(default):
    from d1 import _rows
    want = results()
    _rows._F32.clear()
    torch.set_default_dtype(default)
    try:
        got = results()
    finally:
        torch.set_default_dtype(torch.float32)
        _rows._F32.clear()
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))
