"""Token log-probabilities (d1.token_logprob) against the definition in 64 bits.

Tolerances. A log-probability is z - log S with z = (x - max) / T: three fp32
roundings of |z| (2^-24 each) and the error of log S, which is that of S: 2^-22
for each exponential, and one rounding for each term a thread adds in turn
(vocab / 256 for long rows, fewer for short ones) and each join; 2e-5 covers
the vocabularies here. The entropy's error is log S's plus that of the mean of
z, whose weights sum to 1. A gradient's p has the relative error of e^z:
2^-24 |z| twice over, and 2^-22; then one rounding to the output's type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}  # one rounding to nearest
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def unpack(legal, vocab):
    j = torch.arange(vocab, device=legal.device)
    return (legal[:, j >> 3].to(torch.int32) >> (j & 7).to(torch.int32)) & 1 == 1


def definition(logits, tokens, legal, temperature, top):
    """(x masked, z, p, logp, entropy, best values and tokens) in 64 bits."""
    x = logits.double()
    if legal is not None:
        x = torch.where(unpack(legal, x.shape[1]), x, -math.inf)
    m = x.amax(1, keepdim=True)
    z = torch.where(x == -math.inf, -math.inf, (x - m) / temperature)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    p = torch.where(z == -math.inf, 0.0, lp.exp())
    dead = m[:, 0] == -math.inf
    p[dead] = 0
    entropy = torch.where(p > 0, -p * lp, 0.0).sum(1)
    logp = torch.where(dead, -math.inf, lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0])
    logp = torch.where(tokens < 0, 0.0, logp)
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return x, z, p, lp, logp, entropy, order


def check_forward(logits, tokens, legal, temperature, top, got):
    x, z, p, lp, logp, entropy, order = definition(logits, tokens, legal, temperature, top)
    zt = torch.where(tokens < 0, 0.0, z.gather(1, tokens.clamp(min=0)[:, None])[:, 0])
    tol = 2e-5 + 4 * 2.0 ** -24 * torch.where(zt.isfinite(), zt.abs(), 0.0)
    finite = logp.isfinite()
    assert torch.equal(finite, got.logp.isfinite())
    assert torch.equal(got.logp[~finite].double(), logp[~finite])
    assert ((got.logp - logp).abs()[finite] <= tol[finite]).all()
    assert ((got.entropy - entropy).abs() <= 3e-5 * (1 + math.log(logits.shape[1]))).all()
    assert torch.equal(got.stats[:, 0].double(), x.amax(1))
    if top:
        k = min(top, logits.shape[1])
        dead = (x.gather(1, order) == -math.inf)
        want = torch.where(dead, -1, order)
        assert torch.equal(got.top_tokens[:, :k], want)
        assert (got.top_tokens[:, k:] == -1).all() and (got.top_logp[:, k:] == -math.inf).all()
        best = torch.where(dead, -math.inf, lp.gather(1, order))
        assert torch.equal(got.top_logp[:, :k].isfinite(), best.isfinite())
        tol = 2e-5 + 4 * 2.0 ** -24 * z.gather(1, order).abs()
        assert (dead | ((got.top_logp[:, :k] - best).abs() <= tol)).all()


def gradient(logits, tokens, legal, temperature, dlogp, dentropy):
    """(dlogits, its error bound before the last rounding) in 64 bits."""
    x, z, p, lp, logp, entropy, _ = definition(logits, tokens, legal, temperature, 0)
    alive = (tokens >= 0) & logp.isfinite()
    a, b = torch.where(alive, dlogp.double(), 0.0)[:, None], dentropy.double()[:, None]
    lpf = torch.where(p > 0, lp, 0.0)
    d = -p * (a + b * (lpf + entropy[:, None])) / temperature
    size = p * (a.abs() + b.abs() * (lpf.abs() + entropy[:, None])) / temperature
    tol = (2.0 ** -22 * (4 + z.abs().clamp(max=200)) + 4e-5) * size
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], a / temperature)
    return d, tol + 2.0 ** -23 * a.abs() / temperature


def case(rows, vocab, dtype, masked, seed, stride=None):
    g = torch.Generator(device='cuda').manual_seed(seed)
    logits = (3 * torch.randn(rows, stride or vocab, device='cuda', generator=g)).to(dtype)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), device='cuda', generator=g)
    tokens[rows // 2] = -1
    legal = None
    if masked:
        legal = torch.randint(0, 256, (rows, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
        legal[rows - 1] = 0
        # what is left out may hold anything
        out = ~unpack(legal, vocab)
        logits = logits.clone() if stride is None else logits
        logits[out & (torch.rand(out.shape, device='cuda', generator=g) < 0.3)] = math.nan
        logits[out & (torch.rand(out.shape, device='cuda', generator=g) < 0.3)] = math.inf
    return logits, tokens, legal, g


VOCABS = [1, 2, 12, 28, 63, 64, 65, 255, 256, 257, 1000, 1024, 1025, 1031, 2048, 4099, 16384, 33333]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('vocab', VOCABS)
def test_forward_and_gradient(vocab, dtype):
    from d1.token_logprob import token_logprob, token_logprob_backward
    for rows, masked, temperature, top in ((1, False, 1.0, 32), (5, True, 0.7, 20), (67, False, 1.3, 1), (67, True, 1.0, 7)):
        logits, tokens, legal, g = case(rows, vocab, dtype, masked, 7 * vocab + rows)
        got = token_logprob(logits, tokens, legal, temperature, top)
        check_forward(logits, tokens, legal, temperature, top, got)
        dlogp = torch.randn(rows, device='cuda', generator=g)
        dentropy = torch.randn(rows, device='cuda', generator=g)
        d = token_logprob_backward(logits, tokens, got.stats, got.entropy, dlogp, dentropy, legal, temperature)
        want, tol = gradient(logits, tokens, legal, temperature, dlogp, dentropy)
        assert ((d.double() - want).abs() <= tol + EPS[dtype] * (want.abs() + tol) + TINY[dtype]).all()
        if legal is not None:
            assert (d[~unpack(legal, vocab)] == 0).all()
        d = token_logprob_backward(logits, tokens, got.stats, None, dlogp, None, legal, temperature)
        want, tol = gradient(logits, tokens, legal, temperature, dlogp, torch.zeros_like(dentropy))
        assert ((d.double() - want).abs() <= tol + EPS[dtype] * (want.abs() + tol) + TINY[dtype]).all()


@pytest.mark.parametrize('rows, vocab, dtype, masked, top', [
    (1900, 8200, torch.bfloat16, True, 9), (1900, 9001, torch.float32, False, 3), (2500, 12288, torch.float16, True, 0),
    (80003, 70, torch.float16, True, 5), (310003, 5, torch.bfloat16, True, 2), (310003, 64, torch.float32, False, 0)])
def test_more_rows_than_a_grid_holds(rows, vocab, dtype, masked, top):
    from d1.token_logprob import token_logprob, token_logprob_backward
    logits, tokens, legal, g = case(rows, vocab, dtype, masked, rows + vocab)
    got = token_logprob(logits, tokens, legal, 0.9, top)
    check_forward(logits, tokens, legal, 0.9, top, got)
    dlogp, dentropy = torch.randn(rows, device='cuda', generator=g), torch.randn(rows, device='cuda', generator=g)
    d = token_logprob_backward(logits, tokens, got.stats, got.entropy, dlogp, dentropy, legal, 0.9)
    want, tol = gradient(logits, tokens, legal, 0.9, dlogp, dentropy)
    assert ((d.double() - want).abs() <= tol + EPS[dtype] * (want.abs() + tol) + TINY[dtype]).all()


@pytest.mark.parametrize('rows', [1, 2, 9, 40])
def test_few_long_rows_are_split_and_joined(rows):
    from d1.token_logprob import token_logprob
    for vocab in (8192, 65537, 200003):
        for dtype in (torch.bfloat16, torch.float32):
            logits, tokens, legal, _ = case(rows, vocab, dtype, rows % 2 == 0, vocab + rows)
            check_forward(logits, tokens, legal, 1.0, 32, token_logprob(logits, tokens, legal, top=32))


@pytest.mark.parametrize('vocab', [65536, 65544, 70001, 150003])
def test_gradient_of_long_masked_rows(vocab):
    from d1.token_logprob import token_logprob, token_logprob_backward
    for rows, dtype in ((3, torch.bfloat16), (2, torch.float32), (700, torch.bfloat16)):
        if rows == 700 and vocab != 70001:
            continue
        logits, tokens, legal, g = case(rows, vocab, dtype, True, vocab)
        got = token_logprob(logits, tokens, legal)
        dlogp, dentropy = torch.randn(rows, device='cuda', generator=g), torch.randn(rows, device='cuda', generator=g)
        d = token_logprob_backward(logits, tokens, got.stats, got.entropy, dlogp, dentropy, legal)
        for lo in range(0, rows, 50):
            part = slice(lo, lo + 50)
            want, tol = gradient(logits[part], tokens[part], legal[part], 1.0, dlogp[part], dentropy[part])
            assert ((d[part].double() - want).abs() <= tol + EPS[dtype] * (want.abs() + tol) + TINY[dtype]).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('vocab', [28, 300, 3001, 70000])
def test_rows_at_the_edges(vocab, dtype):
    from d1.token_logprob import token_logprob, token_logprob_backward
    low, inf = torch.finfo(dtype).min, math.inf
    x = torch.randn(10, vocab, device='cuda').to(dtype)
    x[0] = low                                 # the type's lowest value everywhere: uniform
    x[1] = -inf                                # nothing left
    x[2], x[2, vocab // 2] = -inf, 3.0         # one token left
    x[3] = 0.0                                 # all equal: the lowest indices come first
    x[4, ::2] = -0.0
    x[4, 1::2] = 0.0                           # equal zeros of both signs
    x[5] = torch.arange(vocab, device='cuda').clamp(max=60000).to(dtype)   # ascending, with ties after rounding
    x[6, vocab // 3] = math.nan
    x[7, vocab // 3] = inf
    x[8, 1:] = low
    x[9, vocab - 1] = torch.finfo(dtype).max
    tokens = torch.full((10,), vocab // 2, device='cuda')
    got = token_logprob(x, tokens, top=20)
    ok = [0, 1, 2, 3, 4, 5, 8, 9]
    check_forward(x[ok], tokens[ok], None, 1.0, 20, type(got)(*(t[ok] for t in got)))
    for r in (6, 7):
        assert got.logp[r].isnan() and got.entropy[r].isnan()
    assert got.top_tokens[6, 0] == vocab // 3 and got.top_tokens[7, 0] == vocab // 3
    assert got.logp[1] == -inf and got.entropy[1] == 0 and (got.top_tokens[1] == -1).all()
    ones = torch.ones(10, device='cuda')
    d = token_logprob_backward(x, tokens, got.stats, got.entropy, ones, ones)
    assert (d[1] == 0).all() and (d[2] == 0).all()
    assert d[6].isnan().all() and d[7].isnan().any()
    assert d[ok].isfinite().all()


def test_shared_and_word_masks_strides_and_shapes():
    from d1.token_logprob import token_logprob, token_logprob_backward
    for vocab in (12, 700, 3000):
        logits, tokens, _, g = case(24, vocab, torch.bfloat16, False, vocab, stride=vocab + 13)
        words = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, (vocab + 31) // 32), device='cuda', generator=g, dtype=torch.int32)
        shared = words.expand(24, -1)
        as_bytes = words.view(torch.uint8).expand(24, -1)
        got = token_logprob(logits, tokens, shared, top=3)
        check_forward(logits, tokens, as_bytes, 1.0, 3, got)
        cube = token_logprob(logits.unflatten(0, (2, 12)), tokens.view(2, 12), shared.unflatten(0, (2, 12)), top=3)
        assert cube.top_tokens.shape == (2, 12, 3) and torch.equal(cube.logp.flatten(), got.logp)
        dlogp = torch.randn(24, device='cuda', generator=g)
        wide = torch.full((24, vocab + 6), 5.0, device='cuda', dtype=torch.bfloat16)
        d = token_logprob_backward(logits, tokens, got.stats, None, dlogp, legal=shared, out=wide[:, 3:3 + vocab])
        assert (wide[:, :3] == 5).all() and (wide[:, 3 + vocab:] == 5).all()
        assert torch.equal(d, token_logprob_backward(logits.contiguous(), tokens, got.stats, None, dlogp, legal=shared))
    legal = torch.tensor([0b101, 0b111111111111, 0], dtype=torch.int16, device='cuda')  # the environments' masks
    logits = torch.randn(3, 12, device='cuda')
    got = token_logprob(logits, torch.tensor([2, 11, 0], device='cuda'), legal, top=12)
    assert sorted(got.top_tokens[0, :2].tolist()) == [0, 2] and (got.top_tokens[0, 2:] == -1).all()
    assert torch.allclose(got.logp[1], logits[1].log_softmax(0)[11], atol=1e-5) and got.logp[2] == -math.inf


def test_tokens_outside_the_vocabulary():
    from d1.token_logprob import token_logprob, token_logprob_backward
    for vocab in (30, 2000):
        logits = torch.randn(3, vocab, device='cuda')
        tokens = torch.tensor([vocab, -7, 2 ** 40], device='cuda')
        got = token_logprob(logits, tokens)
        assert got.logp[0].isnan() and got.logp[1] == 0 and got.logp[2].isnan() and got.entropy.isfinite().all()
        d = token_logprob_backward(logits, tokens, got.stats, None, torch.ones(3, device='cuda'))
        assert d[0].isnan().all() and (d[1] == 0).all() and d[2].isnan().all()


def test_gradient_against_differences():
    """Central differences of the forward pass in fp32: with a step of 2^-6 the truncation is below 2^-12 times the
    third derivative (under 3 for these weights) and the noise 4e-6 / 2^-6: 2e-3 in all."""
    from d1.token_logprob import token_logprob, token_logprob_backward
    g = torch.Generator(device='cuda').manual_seed(5)
    vocab, h = 37, 2.0 ** -6
    x = torch.randn(vocab, device='cuda', generator=g)
    a, b = 0.8, -0.6
    eye = torch.eye(vocab, device='cuda') * h
    tokens = torch.full((vocab,), 11, device='cuda')
    up, down = token_logprob(x + eye, tokens), token_logprob(x - eye, tokens)
    want = ((a * up.logp + b * up.entropy) - (a * down.logp + b * down.entropy)) / (2 * h)
    f = token_logprob(x[None], tokens[:1])
    d = token_logprob_backward(x[None], tokens[:1], f.stats, f.entropy, torch.full((1,), a, device='cuda'),
                               torch.full((1,), b, device='cuda'))
    assert (d[0] - want).abs().max() <= 2e-3


def test_offsets_past_32_bits():
    from d1.token_logprob import token_logprob, token_logprob_backward
    vocab, pitch = 3001, 2 ** 31 + 8
    store = torch.zeros(pitch + vocab, dtype=torch.bfloat16, device='cuda')
    logits = torch.as_strided(store, (2, vocab), (pitch, 1))
    logits.copy_(3 * torch.randn(2, vocab, device='cuda'))
    tokens = torch.tensor([5, 3000], device='cuda')
    got = token_logprob(logits, tokens, top=5)
    check_forward(logits, tokens, None, 1.0, 5, got)
    dlogp = torch.tensor([1.0, -2.0], device='cuda')
    assert torch.equal(token_logprob_backward(logits, tokens, got.stats, None, dlogp),
                       token_logprob_backward(logits.contiguous(), tokens, got.stats, None, dlogp))


def test_another_stream_a_graph_and_the_same_bits():
    from d1.token_logprob import token_logprob
    logits, tokens, legal, _ = case(64, 5000, torch.bfloat16, True, 3)
    want = token_logprob(logits, tokens, legal, top=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprob(logits, tokens, legal, top=8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = token_logprob(logits, tokens, legal, top=8)
    logits[0].fill_(0)
    graph.replay()
    again = token_logprob(logits, tokens, legal, top=8)
    assert all(torch.equal(a, b) for a, b in zip(held, again))


def test_no_rows():
    from d1.token_logprob import token_logprob, token_logprob_backward
    x, t = torch.empty(0, 50, device='cuda'), torch.empty(0, dtype=torch.int64, device='cuda')
    r = token_logprob(x, t, top=2)
    assert r.logp.shape == (0,) and r.top_tokens.shape == (0, 2)
    assert token_logprob_backward(x, t, r.stats, r.entropy, r.logp).shape == (0, 50)


def test_refusals():
    from d1.token_logprob import token_logprob, token_logprob_backward
    x, t = torch.zeros(4, 40, device='cuda'), torch.zeros(4, dtype=torch.int64, device='cuda')
    r = token_logprob(x, t)
    legal = torch.zeros(4, 5, dtype=torch.uint8, device='cuda')
    for bad in (lambda: token_logprob(x.double(), t), lambda: token_logprob(x.T, t[:1]), lambda: token_logprob(x, t[:3]),
                lambda: token_logprob(x, t.int()), lambda: token_logprob(x, t, temperature=0.0),
                lambda: token_logprob(x, t, top=33), lambda: token_logprob(x, t, top=-1),
                lambda: token_logprob(x, t, legal[:, :4]), lambda: token_logprob(x, t, legal.float()),
                lambda: token_logprob(x, t, legal[:3]), lambda: token_logprob(x, t, legal.cpu()),
                lambda: token_logprob(x.cpu(), t.cpu()), lambda: token_logprob(x[:, :0], t),
                lambda: token_logprob(x.expand(3, 4, 40).transpose(0, 1), t.expand(3, 4).T),
                lambda: token_logprob_backward(x, t, r.stats[:3], r.entropy, r.logp),
                lambda: token_logprob_backward(x, t, r.stats, None, r.logp, r.entropy),
                lambda: token_logprob_backward(x, t, r.stats, r.entropy, r.logp, out=x),
                lambda: token_logprob_backward(x, t, r.stats, r.entropy, r.logp, out=x.bfloat16())):
        with pytest.raises(ValueError):
            bad()
