"""Gradients written beside their inputs, in other columns of the same buffer."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('n', [8, 40, 513, 2048])
def test_the_gradients_lie_beside_the_inputs(n):
    from d1.layer_norm import layer_norm, layer_norm_backward
    from d1.token_logprob import token_logprob, token_logprob_backward
    buf = torch.randn(37, 3 * n, device='cuda').bfloat16()
    x, dy, out = buf[:, :n], buf[:, n:2 * n], buf[:, 2 * n:]
    y, mean, rstd = layer_norm(x)
    want = layer_norm_backward(dy.clone(), x.clone(), mean, rstd)
    got = layer_norm_backward(dy, x, mean, rstd, out=out)
    assert all(((a - b).abs() <= 1e-2 * (1 + b.abs())).all() for a, b in zip(got, want))  # other vector widths, other sums
    tokens = torch.zeros(37, dtype=torch.int64, device='cuda')
    r = token_logprob(x, tokens)
    want = token_logprob_backward(x, tokens, r.stats, r.entropy, r.logp)
    assert torch.equal(token_logprob_backward(x, tokens, r.stats, r.entropy, r.logp, out=out), want)
