"""AdamW over many tensors (d1.adamw) against the definition in 64 bits.

Tolerances. One step from a given state: m and v are two products and a sum in
fp32 (three roundings of the terms' magnitudes). The update's ratio m / (sqrt(v)
/ c + eps) adds approximate square root and division (2^-21 each) and the
roundings of its operands: 2^-19 of the update in all, and two roundings of p.
An 8-bit m lies within one code of its value: |m| / 8 or, below the smallest
normal code, 2^-9 of the block's scale; v within v / 4 or 2^-16 of the scale.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tensors(sizes, seed, grad_type=torch.float32, offset=0, copies=True):
    g = torch.Generator(device='cuda').manual_seed(seed)
    params, grads, out = [], [], []
    for i, n in enumerate(sizes):
        skip = offset if i % 2 else 0   # every other tensor starts off its alignment
        params.append(torch.randn(n + skip, device='cuda', generator=g)[skip:])
        grads.append((torch.randn(n + skip, device='cuda', generator=g) * 10.0 ** (-(i % 5))).to(grad_type)[skip:])
        out.append(torch.zeros(n + skip, device='cuda', dtype=torch.bfloat16)[skip:] if copies and i % 3 != 2 else None)
    return params, grads, out


def definition(p, g, m, v, t, lr, betas, eps, decay, clip):
    """(p, m, v) after step t, in 64 bits, and the bound on p's error."""
    p, g, m, v = p.double(), g.double() * clip, m.double(), v.double()
    m1 = betas[0] * m + (1 - betas[0]) * g
    v1 = betas[1] * v + (1 - betas[1]) * g * g
    c = math.sqrt(1 - betas[1] ** t)
    update = lr / (1 - betas[0] ** t) * m1 / (v1.sqrt() / c + eps)
    size = lr / (1 - betas[0] ** t) * (betas[0] * m.abs() + (1 - betas[0]) * g.abs()) / (v1.sqrt() / c + eps)
    new = p * (1 - lr * decay) - update
    return new, m1, v1, 4 * U * (p.abs() + new.abs()) + 2.0 ** -19 * update.abs() + 8 * U * size


def check_step(opt, before, grads, decays, clip, lr):
    t = int(opt.step_dev)
    for i, (p0, m0, v0) in enumerate(before):
        if p0.numel() == 0:
            continue
        p, m, v, tol = definition(p0, grads[i], m0, v0, t, lr, opt.betas, opt.eps, decays[i], clip)
        assert ((opt.params[i].double() - p).abs() <= tol).all(), i
        if opt.copies[i] is not None:
            assert torch.equal(opt.copies[i], opt.params[i].bfloat16()), i
        gm, gv = opt.moments(i)
        em = 4 * U * (m0.double().abs() + grads[i].double().abs() * clip)
        ev = 8 * U * v
        if opt.state_bits == 8:
            first = opt.offsets[i] // 128
            blocks = (p0.numel() + 127) // 128
            spread = lambda s: s[first:first + blocks, None].expand(-1, 128).reshape(-1)[:p0.numel()].double()
            em = em + m.abs() / 8 + spread(opt.m_scale) * 2.0 ** -9
            ev = ev + v / 4 + spread(opt.v_scale) * 2.0 ** -16
            assert ((gv > 0) == (v > 0)).all()
        assert ((gm.double() - m).abs() <= em + 1e-38).all(), i
        assert ((gv.double() - v).abs() <= ev + 1e-38).all(), i


SIZES = [1, 127, 128, 129, 5, 0, 1000, 4096, 3, 257, 70001, 40000, 64]


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('grad_type', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('offset', [0, 1])
def test_steps(bits, grad_type, offset):
    from d1.adamw import AdamW
    for max_norm, sizes in ((0.0, SIZES), (0.5, SIZES), (0.0, [2]), (1e9, [513] * 70), (0.1, [300000, 1])):
        params, grads, copies = tensors(sizes, 11 + bits, grad_type, offset)
        decays = [0.1 * (i % 3) for i in range(len(sizes))]
        opt = AdamW(params, grads, lr=1e-2, weight_decay=decays, state_bits=bits, max_norm=max_norm, copies=copies, seed=3)
        for step in range(4):
            before = [(p.clone(), *(x.clone() for x in opt.moments(i))) for i, p in enumerate(params)]
            lr = 1e-2 if step < 3 else 3e-3
            opt.step(lr=None if step < 3 else lr)
            assert int(opt.step_dev) == step + 1
            clip = 1.0
            if max_norm:
                norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
                assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm
                clip = min(1.0, max_norm / (norm + 1e-6))
            check_step(opt, before, grads, decays, clip, lr)
            for g in grads:
                g.mul_(-0.5)


def mix(z):
    """The splitmix64 output function of int64 tensors (products wrap, shifts are logical)."""
    z = z + -7046029254386353131
    z = (z ^ ((z >> 30) & 0x3ffffffff)) * -4658895280553007687
    z = (z ^ ((z >> 27) & 0x1fffffffff)) * -7723592293110705685
    return z ^ ((z >> 31) & 0x1ffffffff)


def test_codes_are_the_formulas_with_every_operation_rounded():
    """m, v, scales and codes bit for bit: products and sums rounded to fp32 one by one, 16 random bits an element."""
    from d1.adamw import AdamW
    n = 1 << 24  # a last bit moves one code in a million
    g = torch.Generator(device='cuda').manual_seed(33)
    p = [torch.randn(n, device='cuda', generator=g)]
    grad = [torch.randn(n, device='cuda', generator=g) * torch.exp(3 * torch.randn(n // 128, 1, device='cuda', generator=g)).expand(-1, 128).reshape(-1)]
    opt = AdamW(p, grad, state_bits=8, seed=5)
    for step in range(1, 4):
        m, v = opt.moments(0)
        m, v = m * 0.9 + grad[0] * (1 - 0.9), v * 0.999 + (grad[0] * grad[0]) * (1 - 0.999)
        opt.step()
        word = mix(mix(mix(torch.tensor(5, device='cuda')) + step) + torch.arange(n // 4, device='cuda'))
        bits = torch.stack([(word >> k) & 0xffff for k in (0, 16, 32, 48)], 1).reshape(-1, 128).to(torch.int32)
        for x, got, scale, field, bias, drop in ((m, opt.m, opt.m_scale, 7, 7, 20), (v, opt.v, opt.v_scale, 14, 15, 21)):
            size = x.abs().view(-1, 128)
            e = ((size.amax(1).view(torch.int32) >> 23) - 127).clamp(min=-100)
            assert torch.equal(scale, ((e - field + 127) << 23).view(torch.float32))
            y = size * ((field - e + 127) << 23).view(torch.float32)[:, None] * 2.0 ** (bias - 127)
            code = (y.view(torch.int32) + (bits << (drop - 16)) + (1 << (drop - 17))) >> drop
            code = torch.maximum(code, (size > 0).to(torch.int32)) if drop == 21 else code | (x.view(-1, 128) < 0).to(torch.int32) << 7
            assert torch.equal(got.view(torch.uint8).view(-1, 128).to(torch.int32), code)


def test_many_tensors_and_large_ones():
    from d1.adamw import AdamW
    for bits in (32, 8):
        sizes = [1 + (i * 7919) % 700 for i in range(1500)] + [3_000_001]
        params, grads, copies = tensors(sizes, 5)
        opt = AdamW(params, grads, state_bits=bits, copies=copies, max_norm=1.0)
        before = [(p.clone(), torch.zeros_like(p), torch.zeros_like(p)) for p in params]
        opt.step()
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        check_step(opt, before, grads, [0.01] * len(sizes), min(1.0, 1.0 / (norm + 1e-6)), 1e-3)


@pytest.mark.parametrize('bits', [32, 8])
def test_tiles_that_are_handed_out(bits):              # four and more for each warp; the counter is left as it was found
    from d1.adamw import AdamW
    sizes = [17_000_003, 700, 1, 4_000_100, 130]
    params, grads, copies = tensors(sizes, 6, torch.bfloat16 if bits == 8 else torch.float32, offset=1)
    opt = AdamW(params, grads, state_bits=bits, copies=copies, max_norm=1.0)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    for step in range(3):
        before = [(p.clone(), *(x.clone() for x in opt.moments(i))) for i, p in enumerate(params)]
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm
        check_step(opt, before, grads, [0.01] * len(sizes), min(1.0, 1.0 / (norm + 1e-6)), 1e-3)


def test_rounding_is_unbiased_and_moments_decay():
    """Elements of one value per block: the decoded mean is the value within five standard errors (at most half a
    code each); and with no gradient v falls as 0.999^t, which rounding to nearest would not let it."""
    from d1.adamw import AdamW
    n = 1 << 16
    p, g = [torch.zeros(n, device='cuda')], [torch.full((n,), 0.37, device='cuda')]
    opt = AdamW(p, g, weight_decay=0.0, state_bits=8)
    opt.step()
    m, v = opt.moments(0)
    for got, want, code in ((m, 0.037, 0.037 / 8), (v, 0.37 ** 2 * 1e-3, 0.37 ** 2 * 1e-3 / 4)):
        assert abs(float(got.double().mean()) - want) <= 5 * code / 2 / math.sqrt(n)
        assert got.unique().numel() == 2
    g[0].zero_()
    for _ in range(1000):
        opt.step()
    m, v = opt.moments(0)
    assert float(m.abs().mean()) < 1e-6
    assert abs(float(v.double().mean()) / (0.37 ** 2 * 1e-3 * 0.999 ** 1000) - 1) < 0.05


def test_a_step_is_a_function_of_seed_and_state():
    from d1.adamw import AdamW
    runs = []
    for seed in (1, 1, 2):
        params, grads, copies = tensors(SIZES, 8)
        opt = AdamW(params, grads, state_bits=8, max_norm=0.3, copies=copies, seed=seed)
        for _ in range(3):
            opt.step()
        runs.append([opt.m.view(torch.uint8).clone(), opt.v.view(torch.uint8).clone()] + [p.clone() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert not torch.equal(runs[0][0], runs[2][0])


@pytest.mark.parametrize('bits', [32, 8])
def test_resume_graph_and_streams(bits):
    from d1.adamw import AdamW
    def fresh():
        params, grads, copies = tensors(SIZES, 21)
        return AdamW(params, grads, state_bits=bits, max_norm=0.7, copies=copies, seed=9)
    a, b, c = fresh(), fresh(), fresh()
    for _ in range(6):
        a.step()
    for _ in range(3):
        b.step()
    saved, params = b.state_dict(), [p.clone() for p in b.params]
    d = fresh()
    d.load_state_dict(saved)
    for p, q in zip(d.params, params):
        p.copy_(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            d.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step()
    for _ in range(6):
        graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(a.params, c.params))
    c.set_grads([torch.zeros_like(g) for g in c.grads])   # the captured step reads them
    a.set_grads([torch.zeros_like(g) for g in a.grads])
    d.set_grads(a.grads)
    graph.replay()
    a.step()
    d.step()
    for other in (d, c):
        assert all(torch.equal(p, q) for p, q in zip(a.params, other.params))
        assert torch.equal(a.m.view(torch.uint8), other.m.view(torch.uint8)) and int(other.step_dev) == 7


def test_other_gradients_and_non_finite_ones():
    from d1.adamw import AdamW
    for bits in (32, 8):
        params, grads, _ = tensors([1000, 300], 4, copies=False)
        other = [torch.zeros_like(g) for g in grads]
        opt = AdamW(params, grads, weight_decay=0.0, state_bits=bits)
        was = [p.clone() for p in params]
        opt.set_grads(other)
        opt.step()
        assert all(torch.equal(p, q) for p, q in zip(params, was))
        other[0][130] = float('nan')
        other[1][0] = float('inf')
        opt.step()
        assert params[0].isnan().nonzero().flatten().tolist() == [130] and params[1].isnan().sum() == 1
        m, v = opt.moments(0)
        bad = v.isnan().nonzero().flatten().tolist()
        assert bad == ([130] if bits == 32 else list(range(128, 256)))
        clipped = AdamW([p.clone().nan_to_num(0) for p in params], other, state_bits=bits, max_norm=1.0)
        clipped.step()
        assert clipped.grad_norm.isnan() and all(p.isnan().all() for p in clipped.params)


def test_extreme_magnitudes():
    from d1.adamw import AdamW
    for bits in (32, 8):
        params, grads, _ = tensors([128] * 7, 6, copies=False)
        for g, scale in zip(grads, (1e-30, 1e-22, 1e-18, 1e-8, 1e4, 1e12, 1e17)):
            g.copy_(torch.randn(128, device='cuda') * scale)
        opt = AdamW(params, grads, lr=1e-2, state_bits=bits)
        for _ in range(3):
            opt.step()
        assert all(p.isfinite().all() for p in params)
        for i in range(2, 7):
            m, v = opt.moments(i)
            assert m.isfinite().all() and v.isfinite().all()
            big = grads[i].abs() > 0.1 * grads[i].abs().max()
            assert torch.equal(m[big].sign(), grads[i][big].sign())


def test_against_torch():
    from d1.adamw import AdamW
    params, grads, _ = tensors([5000, 77], 14, copies=False)
    twins = [p.clone().requires_grad_() for p in params]
    ref = torch.optim.AdamW(twins, lr=3e-3, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.05)
    opt = AdamW(params, grads, lr=3e-3, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.05)
    for _ in range(20):
        for q, g in zip(twins, grads):
            q.grad = g.clone()
        ref.step()
        opt.step()
    for p, q in zip(params, twins):
        assert (p - q).abs().max() <= 20 * 2.0 ** -18 * 3e-3 + 20 * 4 * U * 5


def test_refusals():
    from d1.adamw import AdamW
    p, g = torch.zeros(10, device='cuda'), torch.zeros(10, device='cuda')
    opt = AdamW([p], [g], state_bits=8)
    for bad in (lambda: AdamW([], []), lambda: AdamW([p], []), lambda: AdamW([p], [g[:9]]), lambda: AdamW([p.double()], [g]),
                lambda: AdamW([p], [g.half()]), lambda: AdamW([p.cpu()], [g]), lambda: AdamW([p], [g.cpu()]),
                lambda: AdamW([p[::2]], [g[::2]]), lambda: AdamW([p], [g], state_bits=16),
                lambda: AdamW([p], [g], betas=(1.0, 0.9)), lambda: AdamW([p], [g], eps=-1.0), lambda: AdamW([p], [g], max_norm=-1.0),
                lambda: AdamW([p], [g], copies=[p]), lambda: AdamW([p], [g], copies=[p.bfloat16()[:5]]),
                lambda: AdamW([p], [g], weight_decay=[0.1, 0.2]), lambda: AdamW([p[:0]], [g[:0]]),
                lambda: opt.set_grads([g, g]), lambda: opt.load_state_dict({'step': 1}),
                lambda: opt.load_state_dict(dict(opt.state_dict(), m=torch.zeros(128, device='cuda')))):
        with pytest.raises(ValueError):
            bad()
