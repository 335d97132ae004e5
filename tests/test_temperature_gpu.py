"""The smallest and largest temperatures: all of the probability on the largest logits, and
none of it anywhere in particular."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('vocab', [28, 700, 9000, 70000])
def test_extremes(vocab):
    from d1.token_logprob import LEAST, MOST, token_logprob, token_logprob_backward
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = torch.randn(5, vocab, device='cuda', generator=g)
    x[:, 3], x[:, 8], x[:, 9] = 9.0, 9.0, -math.inf
    tokens, ones = torch.tensor([3, 8, 9, 1, -1], device='cuda'), torch.ones(5, device='cuda')
    r = token_logprob(x, tokens, temperature=LEAST)
    assert torch.allclose(r.entropy, torch.full_like(ones, math.log(2)), atol=1e-5)
    assert torch.allclose(r.logp[:2], torch.full_like(ones[:2], -math.log(2)), atol=1e-5)
    assert (r.logp[2:4] == -math.inf).all() and r.logp[4] == 0
    r = token_logprob(x, tokens, temperature=MOST)
    assert torch.allclose(r.entropy, torch.full_like(ones, math.log(vocab - 1)), atol=1e-4)
    assert r.logp[2] == -math.inf and torch.allclose(r.logp[3], -torch.tensor(math.log(vocab - 1), device='cuda'), atol=1e-4)
    d = token_logprob_backward(x, tokens, r.stats, r.entropy, ones, ones, temperature=MOST)
    assert (d[:, 9] == 0).all() and d.isfinite().all()
