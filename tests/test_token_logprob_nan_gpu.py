"""The gradient of rows whose distribution is undefined (a NaN or +inf that is not left
out): NaN, but 0 for every token that is left out, by its bit or by a logit of -inf."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('vocab', [28, 301, 2500, 70001])
def test_left_out_tokens_have_no_gradient(vocab, dtype):
    from d1.token_logprob import token_logprob, token_logprob_backward
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = torch.randn(6, vocab, device='cuda', generator=g).to(dtype)
    x[0, 3], x[1, 5], x[2, 2] = math.nan, math.inf, math.inf
    x[:4, 1::7] = -math.inf
    x[3, 4] = math.nan
    x[0, 6], x[1, 6] = torch.finfo(dtype).min, torch.finfo(dtype).max
    legal = torch.randint(0, 256, (6, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
    legal[:, 0] |= 0b1111100
    j = torch.arange(vocab, device='cuda')
    bits = (legal[:, j >> 3].int() >> (j & 7).int()) & 1 == 1
    tokens = torch.tensor([2, 8, -1, 4, 4, 5], device='cuda')
    ones = torch.ones(6, device='cuda')
    for mask, on in ((None, torch.ones_like(bits)), (legal, bits)):
        for temperature in (1.0, 0.3):
            r = token_logprob(x, tokens, mask, temperature)
            for dentropy in (None, ones):
                d = token_logprob_backward(x, tokens, r.stats, r.entropy, ones, dentropy, mask, temperature)
                out = ~on | (x == -math.inf)
                assert (d[out] == 0).all()
                assert d[:4][~out[:4]].isnan().all() and d[4:].isfinite().all()
