"""The row operators where torch records gradients: their gradients reach the inputs,
and are those of the backward entries.

Tolerances against torch's autograd in 64 bits, on fp32 inputs of unit size: a few
hundred roundings of 2^-24 and approximate exponentials (2^-22) of sums of a few
hundred terms, 1e-4 of the largest gradient.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def close(got, want):
    return bool(((got.double() - want).abs() <= 1e-4 * want.abs().max() + 1e-12).all())


def data(rows, n, seed=1):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(rows, n, device='cuda', generator=g)
    return x, 1 + 0.2 * torch.randn(n, device='cuda', generator=g), torch.randn(n, device='cuda', generator=g), g


@pytest.mark.parametrize('shape', [(1, 7), (33, 256), (4, 9, 130)])
def test_layer_norm(shape):
    from d1.layer_norm import layer_norm
    n = shape[-1]
    _, w, b, g = data(1, n)
    x = torch.randn(shape, device='cuda', generator=g)
    pull = torch.randn(shape, device='cuda', generator=g)
    for need in range(1, 8):
        own = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        ref = [t.double().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        y, mean, rstd = layer_norm(*own)
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
        (y * pull).sum().backward()
        (torch.nn.functional.layer_norm(ref[0], (n,), ref[1], ref[2]) * pull).sum().backward()
        for a, r in zip(own, ref):
            assert (a.grad is None) == (r.grad is None)
            assert a.grad is None or close(a.grad, r.grad)
        with torch.no_grad():
            plain = layer_norm(*own)
        assert all(torch.equal(a, p) and not p.requires_grad for a, p in zip((y, mean, rstd), plain))
    x = x.clone().requires_grad_()
    layer_norm(x)[0].sum().backward()          # a gradient that is one number, expanded; no weights
    assert x.grad.abs().max() <= 1e-4
    with pytest.raises(ValueError):
        layer_norm(x, out=torch.empty_like(x))
    with torch.no_grad():
        layer_norm(x, out=torch.empty_like(x))


@pytest.mark.parametrize('vocab', [28, 300, 9000])
def test_token_logprob(vocab):
    from d1.token_logprob import token_logprob, token_logprob_backward
    x, _, _, g = data(30, vocab)
    tokens = torch.randint(0, vocab, (30,), device='cuda', generator=g)
    legal = torch.randint(0, 256, (30, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
    j = torch.arange(vocab, device='cuda')
    on = (legal[:, j >> 3].int() >> (j & 7).int()) & 1 == 1
    tokens = torch.where(on.gather(1, tokens[:, None])[:, 0], tokens, on.int().argmax(1))
    a, b = torch.randn(30, device='cuda', generator=g), torch.randn(30, device='cuda', generator=g)
    for use_p, use_h in ((1, 1), (1, 0), (0, 1)):
        own, ref = x.clone().requires_grad_(), x.double().requires_grad_()
        r = token_logprob(own, tokens, legal, 0.8, top=3)
        assert r.logp.requires_grad and r.entropy.requires_grad
        assert not (r.stats.requires_grad or r.top_tokens.requires_grad or r.top_logp.requires_grad)
        lp = (ref / 0.8).masked_fill(~on, -1e300).log_softmax(1)
        h = -(lp.exp() * lp.masked_fill(~on, 0)).sum(1)
        for logp, entropy in ((r.logp, r.entropy), (lp.gather(1, tokens[:, None])[:, 0], h)):
            parts = [(a * logp).sum()] * use_p + [(b * entropy).sum() if use_p else entropy.sum()] * use_h
            sum(parts).backward()
        assert close(own.grad, ref.grad) and (own.grad[~on] == 0).all()
        plain = token_logprob(x, tokens, legal, 0.8, top=3)
        assert all(torch.equal(p, q) and not p.requires_grad for p, q in zip(plain, r))
    d = token_logprob_backward(x, tokens, plain.stats, plain.entropy, None, torch.ones(30, device='cuda'), legal, 0.8)
    assert torch.equal(d, own.grad)
    own = x.clone().requires_grad_()
    assert torch.autograd.grad(token_logprob(own, tokens).logp.sum(), own)[0].isfinite().all()   # no mask, no alternatives


def test_a_network_trains_with_torchs_own_backward():
    from d1.adamw import AdamW
    from d1.layer_norm import layer_norm
    from d1.token_logprob import token_logprob
    x, w, b, g = data(256, 64)
    head = (0.1 * torch.randn(28, 64, device='cuda', generator=g)).requires_grad_()
    w, b = w.requires_grad_(), b.requires_grad_()
    params = [head, w, b]
    grads = [torch.zeros_like(p) for p in params]
    for p, q in zip(params, grads):
        p.grad = q
    tokens = torch.randint(0, 28, (256,), device='cuda', generator=g)
    opt, losses = AdamW(params, grads, lr=1e-2), []
    for _ in range(30):
        for q in grads:
            q.zero_()
        r = token_logprob(layer_norm(x, w, b)[0] @ head.T, tokens)
        loss = -r.logp.mean()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0] - 0.5
    loss = -token_logprob(layer_norm(x, w, b)[0] @ head.T, tokens).logp.mean()
    opt.step()
    with pytest.raises(RuntimeError):      # the step has overwritten what the graph kept
        loss.backward()
