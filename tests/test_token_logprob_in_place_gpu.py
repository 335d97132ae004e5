"""d1_token_logprob_backward with the gradient written over the logits: the bits
of the gradient written elsewhere, among them those of rows whose token is left
out by its logit (every thread of a row looks at that logit, which one of them
overwrites)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def backward(x, tokens, r, dlogp, dentropy, legal, out):
    from d1._lib import check, library, stream_of
    kind = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    check(library().d1_token_logprob_backward(
        x.data_ptr(), x.stride(0), kind, x.shape[0], x.shape[1], tokens.data_ptr(), None if legal is None else legal.data_ptr(),
        0 if legal is None else legal.stride(0), 0.9, r.stats.data_ptr(), r.entropy.data_ptr(), dlogp.data_ptr(),
        dentropy.data_ptr(), out.data_ptr(), out.stride(0), stream_of(x)))
    return out


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows, vocab, pitch', [(67, 12, 32), (5, 28, 28), (40000, 28, 32), (31, 301, 301), (9, 2048, 2056),
                                                (1, 70001, 70001), (3, 131072, 131072), (900, 9001, 9001)])
def test_in_place(rows, vocab, pitch, dtype):
    from d1.token_logprob import token_logprob
    g = torch.Generator(device='cuda').manual_seed(vocab + rows)
    x = torch.randn(rows, pitch, device='cuda', generator=g).to(dtype)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), device='cuda', generator=g)
    x[torch.arange(0, rows, 2, device='cuda'), tokens[::2]] = -math.inf
    mask = torch.randint(0, 256, (rows, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
    dlogp, dentropy = torch.randn(rows, device='cuda', generator=g), torch.randn(rows, device='cuda', generator=g)
    for legal in (None, mask):
        r = token_logprob(x, tokens, legal, 0.9)
        want = backward(x, tokens, r, dlogp, dentropy, legal, torch.empty_like(x))
        for _ in range(5):
            mine = torch.zeros(rows, pitch, device='cuda', dtype=dtype)[:, :vocab]
            mine.copy_(x)
            assert torch.equal(backward(mine, tokens, r, dlogp, dentropy, legal, mine), want)
