"""The clipped policy loss (d1.policy_loss) against its formula in 64 bits.

Tolerances. delta and d are differences rounded once (2^-24 of themselves, which e^delta passes on as
|delta| 2^-24 of itself, once more where e^delta is 2^(delta log2 e)), that power of two is off by 2^-22, a weight is 1 / n rounded up to twice, and
products and sums round once each: under 8 half steps of each term beside |delta| or |d|. Doubled below. The loss
adds the terms' errors: 2^-24 (16 + 2 |delta|) of the sum of their magnitudes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
LOW, HIGH, KL, ENT = 0.2, 0.28, 0.05, 0.01


def formula(s, clip=(LOW, HIGH), kl=KL, ent=ENT, mean='token'):
    """(loss, stats, dlogp, dentropy) and the tolerances of each, in 64 bits."""
    shape = s['logp'].shape
    m = torch.ones(shape, dtype=torch.bool, device='cuda') if s.get('mask') is None else s['mask'] != 0
    get = lambda k: torch.where(m, s[k].double(), 0.0) if s.get(k) is not None else None
    lp, old = get('logp'), get('old_logp')
    adv = s['advantage'].double()
    adv = torch.where(m, adv if adv.shape == shape else adv.unsqueeze(-1).expand(shape), 0.0)
    w = m.double()
    if mean == 'token':
        w = w / w.sum().clamp(min=1)
    else:
        n = w.sum(-1, keepdim=True)
        w = w / n.clamp(min=1) / (n > 0).sum().clamp(min=1)
    delta = lp - old
    r = delta.exp()
    cut = m & (((r > 1 + clip[1]) & (adv > 0)) | ((r < 1 - clip[0]) & (adv < 0)))
    policy = -torch.minimum(r * adv, r.clamp(1 - clip[0], 1 + clip[1]) * adv)
    old_kl = torch.expm1(delta) - delta
    dlogp, size = torch.where(cut, 0.0, -adv * r), (delta.abs() + 8) * (adv * r).abs()
    big = w * (policy.abs() + 1e-30)
    k3 = torch.zeros_like(lp)
    if s.get('ref_logp') is not None:
        d = get('ref_logp') - lp
        k3 = torch.expm1(d) - d
        dlogp = dlogp - kl * torch.expm1(d)
        size = size + abs(kl) * (d.abs() * d.exp() + 8 * torch.expm1(d).abs())
        big = big + w * abs(kl) * (k3 + d.abs() * torch.expm1(d).abs() / 8)
    h = get('entropy') if s.get('entropy') is not None else torch.zeros_like(lp)
    big = big + w * (ent * h).abs()
    terms = [policy, k3, h, cut.double(), old_kl]
    stats = torch.stack([(w * t).sum() for t in terms])
    loss = stats[0] + kl * stats[1] - ent * stats[2]
    reach = 16 + 2 * float(delta.abs().max()) if lp.numel() else 16
    tols = torch.stack([(w * t.abs()).sum() for t in terms]) * H * reach
    # the error of d (and delta) in e^d - d - 1 is d's times e^d - 1
    if s.get('ref_logp') is not None:
        tols[1] += 2 * H * (w * (d * torch.expm1(d)).abs()).sum()
    tols[4] += 2 * H * (w * (delta * torch.expm1(delta)).abs()).sum()
    return (loss, stats, dlogp * w, -ent * w), (big.sum() * H * reach, tols, 2 * H * size * w, 4 * H * abs(ent) * w)


def inputs(shape, seed=0, per_row=False, ref=True, entropy=True, mask=True):
    g = torch.Generator(device='cuda').manual_seed(seed + sum(shape))
    new = lambda *s: torch.randn(s, device='cuda', generator=g)
    s = {'old_logp': -new(*shape).abs()}
    s['logp'] = s['old_logp'] + 0.2 * new(*shape) * (new(*shape) > -1)
    s['advantage'] = new(*shape[:-1]) if per_row else new(*shape)
    s['ref_logp'] = s['old_logp'] + 0.3 * new(*shape) if ref else None
    s['entropy'] = new(*shape).abs() if entropy else None
    s['mask'] = None
    if mask:
        ends = torch.randint(0, shape[-1] + 1, shape[:-1], device='cuda', generator=g).reshape(-1)
        if ends.numel() > 1:
            ends[0] = 0                                                       # a row without a token
        s['mask'] = (torch.arange(shape[-1], device='cuda') < ends[:, None]).view(shape)
        for k, v in (('logp', -math.inf), ('old_logp', math.nan), ('ref_logp', math.inf), ('entropy', math.nan)):
            if s[k] is not None:
                s[k] = s[k].masked_fill(~s['mask'], v)
        if not per_row:
            s['advantage'] = s['advantage'].masked_fill(~s['mask'], math.nan)
    return s


def call(s, mean='token', kl=KL, ent=ENT, clip=(LOW, HIGH), **more):
    from d1.policy_loss import policy_loss
    return policy_loss(s['logp'], s['old_logp'], s['advantage'], ref_logp=s['ref_logp'], entropy=s['entropy'], mask=s['mask'], clip=clip,
                       kl_coef=kl, ent_coef=ent, mean=mean, **more)


def check(s, mean, **more):
    r = call(s, mean, **more)
    want, tols = formula(s, mean=mean, **more)
    for name, got, w, tol in zip(r._fields, r, want, tols):
        if got is None:
            assert name == 'dentropy' and s['entropy'] is None
            continue
        assert got.dtype == torch.float32 and got.shape == w.shape
        assert ((got.double() - w).abs() <= tol + w.abs() * H + 1e-38).all(), name
    return r


SHAPES = [(1,), (7,), (1, 1), (1, 16384), (3, 5), (40, 4), (2048, 8), (2049, 8), (5, 1023), (512, 129), (7, 4099), (1, 50021), (16384, 28),
          (3, 100000), (2, 3, 70)]


@pytest.mark.parametrize('mean', ['token', 'row'])
@pytest.mark.parametrize('mask', [True, False])
@pytest.mark.parametrize('shape', SHAPES)
def test_against_the_formula(shape, mask, mean):
    check(inputs(shape, mask=mask), mean)
    check(inputs(shape, mask=mask, per_row=len(shape) > 1, ref=False), mean)
    check(inputs(shape, mask=mask, per_row=len(shape) > 1, entropy=False), mean)
    check(inputs(shape, mask=mask, ref=False, entropy=False), mean)


@pytest.mark.parametrize('shape', [(6, 50), (300, 700)])
def test_coefficients_and_ranges(shape):
    s = inputs(shape)
    for more in (dict(kl=0.0, ent=0.0), dict(kl=2.0, ent=-0.3), dict(clip=(0.0, 0.0)), dict(clip=(1.0, 5.0)), dict(clip=(3.0, 0.1))):
        check(s, 'token', **more)
    assert torch.equal(call(s, clip=0.3).loss, call(s, clip=(0.3, 0.3)).loss)


def test_the_same_policy():
    """Ratios of 1: the loss is the negative mean advantage and nothing is clipped, at the border of an empty range too."""
    s = inputs((9, 300), ref=False, entropy=False, mask=False)
    s['logp'] = s['old_logp']
    r = call(s, clip=0.0)
    assert r.stats[3] == 0 and r.stats[4] == 0
    assert torch.equal(r.dlogp, -s['advantage'] * (1.0 / 2700))


@pytest.mark.parametrize('size', [40, 40000])
def test_borders(size):
    """Neighbouring fp32 log-probabilities on both sides of both borders: cut exactly where the exact difference is beyond."""
    out = {}
    for sign in (1.0, -1.0):
        base = torch.full((size,), -1.5, device='cuda')
        for border in (math.log1p(HIGH), math.log1p(-LOW)):
            at = torch.tensor(-1.5 + border, dtype=torch.float32)
            k = torch.arange(size, dtype=torch.int32) - size // 2
            lp = (at.view(torch.int32) + k).view(torch.float32).cuda()
            s = dict(logp=lp, old_logp=base, advantage=torch.full_like(lp, sign), ref_logp=None, entropy=None, mask=None)
            r = call(s)
            delta = lp.double() + 1.5
            cut = delta > math.log1p(HIGH) if sign > 0 else delta < math.log1p(-LOW)
            assert torch.equal(r.dlogp == 0, cut)
            out[sign, border] = float(r.stats[3])
    assert 0.3 < out[1.0, math.log1p(HIGH)] < 0.7 and 0.3 < out[-1.0, math.log1p(-LOW)] < 0.7


@pytest.mark.parametrize('shape', [(4, 6), (50, 1000)])
def test_nothing_counts(shape):
    s = inputs(shape)
    s['mask'] = torch.zeros(shape, dtype=torch.uint8, device='cuda')
    for mean in ('token', 'row'):
        r = call(s, mean)
        assert all((t == 0).all() for t in r)
    from d1.policy_loss import policy_loss
    none = torch.empty(0, 5, device='cuda')
    r = policy_loss(none, none, none, entropy=none)
    assert r.loss == 0 and (r.stats == 0).all() and r.dlogp.shape == (0, 5)
    s['mask'][2, 3] = 200                                  # one token: any byte but 0 keeps it
    s = {k: v if k == 'mask' else inputs(shape, mask=False)[k] for k, v in s.items()}
    for mean in ('token', 'row'):
        check(s, mean)


@pytest.mark.parametrize('mean', ['token', 'row'])
def test_pitches_and_alignment(mean):
    s = inputs((60, 520))
    for k in ('logp', 'old_logp', 'advantage', 'ref_logp', 'entropy', 'mask'):
        t = s[k]
        wide = torch.cat((t, t), 1)[:, :520]
        check(dict(s, **{k: wide}), mean)
        odd = torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)
        check(dict(s, **{k: odd}), mean)
    s = inputs((60, 520), per_row=True)
    check(dict(s, advantage=torch.stack((s['advantage'],) * 3, 1)[:, 1]), mean)
    s = inputs((60, 520), mask=False)
    s['mask'] = (torch.arange(520, device='cuda') % 3 > 0).expand(60, 520)
    check(s, mean)
    check(dict(s, advantage=s['advantage'][:1].expand(60, 520)), mean)


def test_ratios_beyond_fp32():
    """A ratio that overflows keeps its sign; one that vanishes has a zero gradient."""
    old = torch.tensor([-200.0, -200.0, 0.0, 0.0], device='cuda')
    logp = torch.tensor([0.0, 0.0, -200.0, -math.inf], device='cuda')
    s = dict(logp=logp, old_logp=old, advantage=torch.tensor([1.0, -1.0, 1.0, 1.0], device='cuda'), ref_logp=None, entropy=None, mask=None)
    r = call(s)
    assert r.loss == math.inf and r.dlogp.tolist() == [0.0, math.inf, 0.0, 0.0]


@pytest.mark.parametrize('size', [4, 40000])
def test_a_reference_far_away(size):
    """Where the reference holds a token for impossible the KL term is infinite and its gradient kl_coef; far below, the gradient
    does not cancel."""
    z = torch.full((size,), -1.0, device='cuda')
    for away in (-math.inf, -1e30, -3e6, -1e3):
        ref = z.clone()
        ref[0] = away
        r = call(dict(logp=z, old_logp=z, advantage=torch.zeros_like(z), ref_logp=ref, entropy=None, mask=None), kl=0.5)
        assert abs(float(r.dlogp[0]) * size - 0.5) < 1e-6 and (r.dlogp[1:] == 0).all()
        assert abs(float(r.stats[1]) * size / -away - 1) < 1e-2 if away > -math.inf else r.stats[1] == math.inf


def test_gradient_against_differences():
    """Central differences of 2^-9 in 64-bit steps of fp32 inputs: the loss's own rounding of 2^-22 of about 1 over 2^-8
    and a third derivative's 2^-18: 2e-4. Tokens within 2^-8 of a border are passed over."""
    for mean in ('token', 'row'):
        s = inputs((3, 5), seed=3, mask=False)
        s['mask'] = torch.tensor([[1, 1, 1, 0, 0], [0] * 5, [1] * 5], dtype=torch.bool, device='cuda')
        r, d = call(s, mean), 2.0 ** -9
        for key, grad in (('logp', r.dlogp), ('entropy', r.dentropy)):
            for k in range(15):
                delta = float((s['logp'] - s['old_logp']).view(-1)[k])
                if min(abs(delta - math.log1p(HIGH)), abs(delta - math.log1p(-LOW))) < 2.0 ** -8:
                    continue
                moved = []
                for sign in (1, -1):
                    t = s[key].clone()
                    t.view(-1)[k] += sign * d
                    moved.append(float(call(dict(s, **{key: t}), mean).loss))
                assert abs((moved[0] - moved[1]) / (2 * d) - float(grad.view(-1)[k])) < 2e-4


def test_torchs_own_backward_and_no_gradient():
    s = inputs((30, 40))
    want = call(s)
    for lp, h in ((1, 1), (1, 0), (0, 1)):
        leaves = {k: s[k].clone().requires_grad_(bool(n)) for k, n in (('logp', lp), ('entropy', h))}
        r = call(dict(s, **leaves))
        assert r.loss.requires_grad and not (r.stats.requires_grad or r.dlogp.requires_grad)
        (3 * r.loss).backward()
        for k, g in (('logp', want.dlogp), ('entropy', want.dentropy)):
            assert (leaves[k].grad is None) == (not leaves[k].requires_grad)
            assert leaves[k].grad is None or torch.equal(leaves[k].grad, 3 * g)
    r = call(s, gradient=False)
    assert r.dlogp is None and r.dentropy is None and torch.equal(r.loss, want.loss) and torch.equal(r.stats, want.stats)


@pytest.mark.parametrize('shape', [(20, 100), (300, 501)])
def test_graphs_streams_and_the_default_type(shape):
    a, b = inputs(shape, 1), inputs(shape, 2)
    held = {k: v.clone() for k, v in a.items()}
    want = [[t.clone() for t in call(s, 'row')] for s in (a, b)]
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(held, 'row'))
    for k in held:
        held[k].copy_(b[k])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        with torch.cuda.stream(side):
            eager = call(a, 'row')
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want[1]))
    assert all(torch.equal(p, q) for p, q in zip(eager, want[0]))
    torch.set_default_dtype(torch.float64)
    try:
        assert all(torch.equal(p, q) for p, q in zip(call(a, 'row'), want[0]))
    finally:
        torch.set_default_dtype(torch.float32)


def test_with_the_log_probabilities_of_a_policy():
    """token_logprob, the loss and token_logprob's gradient: the logits' gradient is autograd's in 64 bits (1e-4 of the
    largest: a few roundings and approximate exponentials, 2^-22, of 28 terms)."""
    from d1.policy_loss import policy_loss
    from d1.token_logprob import token_logprob, token_logprob_backward
    g = torch.Generator(device='cuda').manual_seed(5)
    logits = torch.randn(64, 50, 28, device='cuda', generator=g)
    tokens = torch.randint(0, 28, (64, 50), device='cuda', generator=g)
    adv, live = torch.randn(64, 50, device='cuda', generator=g), torch.rand(64, 50, device='cuda', generator=g) < 0.8
    old = logits.log_softmax(-1).gather(-1, tokens[..., None])[..., 0] + 0.2 * torch.randn(64, 50, device='cuda', generator=g)
    r = token_logprob(logits, tokens)
    p = policy_loss(r.logp, old, adv, entropy=r.entropy, mask=live, clip=(LOW, HIGH), ent_coef=0.1)
    d = token_logprob_backward(logits, tokens, r.stats, r.entropy, p.dlogp, p.dentropy)
    x = logits.double().requires_grad_()
    lp = x.log_softmax(-1)
    ratio = (lp.gather(-1, tokens[..., None])[..., 0] - old.double()).exp()
    each = -torch.minimum(ratio * adv, ratio.clamp(1 - LOW, 1 + HIGH) * adv) + 0.1 * (lp.exp() * lp).sum(-1)
    loss = each[live].mean()
    loss.backward()
    assert abs(float(p.loss) - float(loss.detach())) < 1e-5 and (d.double() - x.grad).abs().max() <= 1e-4 * x.grad.abs().max()
    own = logits.clone().requires_grad_()
    r = token_logprob(own, tokens)
    policy_loss(r.logp, old, adv, entropy=r.entropy, mask=live, clip=(LOW, HIGH), ent_coef=0.1).loss.backward()
    assert torch.equal(own.grad, d)


def test_rows_without_tokens_in_the_c_entry():
    """More rows than a cluster counts, none of which has a token: everything is 0."""
    from d1._lib import library
    loss, stats = torch.full((), 7.0, device='cuda'), torch.full((5,), 7.0, device='cuda')
    mask = torch.ones(8, dtype=torch.uint8, device='cuda')
    for by_row in (0, 1):
        for m in (None, mask.data_ptr()):
            loss.fill_(7.0), stats.fill_(7.0)
            assert library().d1_policy_loss(None, 0, None, 0, None, 0, 0, None, 0, None, 0, m, 0, 100000, 0, 0.2, 0.2, 0.1, 0.01, by_row,
                                            loss.data_ptr(), stats.data_ptr(), None, None, None, torch.cuda.current_stream().cuda_stream) == 0
            assert loss == 0 and (stats == 0).all()


def test_refusals():
    from d1.policy_loss import policy_loss
    s = inputs((4, 6), mask=False)
    lp, old, adv = s['logp'], s['old_logp'], s['advantage']
    for bad in (lambda: policy_loss(lp.half(), old, adv), lambda: policy_loss(lp, old.double(), adv), lambda: policy_loss(lp, old[:3], adv),
                lambda: policy_loss(lp, old, adv[:, :5]), lambda: policy_loss(lp, old, adv[:3, 0]), lambda: policy_loss(lp, old, adv, mask=lp),
                lambda: policy_loss(lp, old, adv, mask=torch.ones(6, dtype=torch.bool, device='cuda')), lambda: policy_loss(lp.T, old.T, adv.T),
                lambda: policy_loss(lp, old, adv, clip=-0.1), lambda: policy_loss(lp, old, adv, clip=(0.1, float('nan'))),
                lambda: policy_loss(lp, old, adv, mean='sum'), lambda: policy_loss(lp, old.cpu(), adv), lambda: policy_loss(lp[:, :0], old[:, :0], adv[:, :0]),
                lambda: policy_loss(lp, old, adv, ref_logp=old[0]), lambda: policy_loss(lp, old, adv, entropy=old.half())):
        with pytest.raises(ValueError):
            bad()
