"""Muon (d1.muon) against its formulas in 64 bits, and against the same formulas with the fp16 roundings that
it documents.

Tolerances. Rounding to fp16 is off by 2^-11 of an element at most, 2^-12.8 of a matrix's norm for roundings that are
independent. A step rounds X, A and B once; X counts twice in A, A twice in A^2, whose factors b and c and X itself leave
errors of under 8 such roundings, 2^-9.8 of the norm, in directions that X has, and later steps carry them on with factors of about 1: 4e-3
of the result's norm (2^-8) covers several steps' sum. A 16-bit result adds 2^-9 (bf16) or 2^-12 (fp16) of it. Against the
same roundings only the sums' precision differs at first: where it moves an operand over a rounding border it moves by a whole
step, one in some thousands, so that 2^-11 of the norm is ample for two steps. From then on the two go apart: an operand
that is off by 1e-4 crosses a border every fifth time, and the roundings are no longer the same ones (the emulation itself, with
sums in fp32 instead of fp64, moves by 1e-7, 2e-6, 2e-4, 8e-4 and 1.6e-3 in steps one to five of 128 x 128). What is left is that both are within
NS of the exact result: 2 NS.

Matrices with a side of at most 64 take, beside wider ones, products of pairs of fp16: operands of 22 bits, sums in fp32 (a term of 2^-23 for each
of up to 16 partial sums of a long row), under 2^-18 a step, and five steps with factors of at most 4: 2^-12.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315
NS = 2.0 ** -8
SAME = {1: 2.0 ** -11, 2: 2.0 ** -11}  # against the emulation; 2 NS for more steps
OUT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


def exact(u, steps=5):
    x = u.double()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = x / torch.where(norm > 0, norm, 1)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        g = x @ x.mT
        x = A * x + (B * g + C * g @ g) @ x
    return x.mT if tall else x


def emulated(u, steps=5):
    """The same with the documented roundings."""
    f16 = lambda t: (t.float() * 4096).half().double() / 4096
    x = u.double()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = x / torch.where(norm > 0, norm, 1)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        hi = f16(x)
        x = hi + f16(x - hi)
        g = f16(hi @ hi.mT)
        x = A * x + f16(B * g + C * g @ g) @ hi
    return x.mT if tall else x


def distance(got, want):
    """Largest of the matrices' distances over their norms."""
    d = (got.double() - want).square().sum((-2, -1)).sqrt()
    n = want.square().sum((-2, -1)).sqrt()
    assert (d[n == 0] == 0).all()
    return float((d / n.clamp(min=1e-300)).max())


def bound(x):
    return 2.0 ** -12 if min(x.shape[-2:]) <= 64 else NS


def matrix(*shape, kind='full', seed=0, dtype=torch.float32):
    g = torch.Generator(device='cuda').manual_seed(seed + sum(shape))
    new = lambda *s: torch.randn(s, device='cuda', generator=g)
    *lead, m, n = shape
    if kind == 'full':
        return new(*shape).to(dtype)
    k = max(1, min(m, n) // 16)   # of low rank, to the last bit of fp32
    return (new(*lead, m, k) @ new(*lead, k, n)).to(dtype)


SIZES = [(1, 1), (1, 77), (77, 1), (9, 64), (64, 64), (65, 63), (128, 128), (129, 200), (200, 129), (30, 900), (900, 30), (500, 500), (256, 1000),
         (1000, 256), (700, 130)]


@pytest.mark.parametrize('kind', ['full', 'low'])
@pytest.mark.parametrize('size', SIZES)
def test_orthogonalize(size, kind):
    from d1.muon import muon_error, orthogonalize
    for dtype, out in ((torch.float32, torch.float16), (torch.bfloat16, None), (torch.float16, None)):
        x = matrix(*size, kind=kind, dtype=dtype)
        y = orthogonalize(x, out=None if out is None else torch.empty(size, dtype=out, device='cuda'))
        assert y.shape == x.shape and y.dtype == (out or dtype)
        assert distance(y, exact(x)) <= bound(x) + OUT[y.dtype]
        assert distance(y, emulated(x)) <= 2 * NS + OUT[y.dtype]
    assert muon_error() == 0


@pytest.mark.parametrize('steps', [1, 2, 8])
def test_steps(steps):
    from d1.muon import orthogonalize
    x = matrix(130, 70)
    y = orthogonalize(x, steps=steps)
    assert y.dtype == torch.bfloat16 and distance(y, emulated(x, steps)) <= SAME.get(steps, 2 * NS) + OUT[y.dtype]


@pytest.mark.parametrize('batch, size', [(1, (60, 700)), (13, (60, 700)), (14, (60, 700)), (1, (128, 2000)), (20, (2000, 100)), (148, (20, 30)), (149, (20, 30)),
                                         (3, (128, 4100)), (40, (128, 500)), (1, (64, 4000))])
def test_small_ones_together(batch, size):
    """As many as one launch takes through all products, and more; long ones, whose first sum is divided, and too long ones."""
    from d1.muon import muon_error, orthogonalize
    for kind in ('full', 'low'):
        x = matrix(batch, *size, kind=kind)
        y = orthogonalize(x)
        assert distance(y, exact(x)) <= bound(x) + OUT[y.dtype]
        assert all(torch.equal(orthogonalize(x), y) for _ in range(2))
    assert muon_error() == 0


@pytest.mark.parametrize('steps', [1, 2, 5, 7])
@pytest.mark.parametrize('batch, size', [(1, (1, 8)), (1, (64, 520)), (3, (7, 513)), (17, (64, 1100)), (1, (40, 20001)), (2, (16500, 33)), (300, (24, 48)), (5, (600, 64)),
                                         (2, (8, 9)), (50, (60, 500)), (40, (30, 700)), (1, (9, 1024)), (1, (1025, 10)), (30, (64, 4096))])
def test_narrow_ones(batch, size, steps):
    """A side of at most 64. Between the sums and the result all is fp64 (11.9 a step on 2^-53 is nothing); Q X is fp32: 64 terms' rounding, 2^-21 if
    all were alike, of |Q| |X|, which is at most 3.44 a step (485) times the result where X hardly has a direction: 2^-12. Up to 7 steps (5,700)
    the matrices of full rank here have no such direction, and those of low rank have it in fp32's last bits only, 2^-24 each."""
    from d1.muon import orthogonalize
    for kind in ('full', 'low') if steps <= 5 else ('full',):
        x = matrix(batch, *size, kind=kind)
        y = orthogonalize(x, steps=steps, out=torch.empty(x.shape, dtype=torch.float16, device='cuda'))
        assert distance(y, exact(x, steps)) <= 2.0 ** -12 + OUT[y.dtype]
        assert torch.equal(orthogonalize(x, steps=steps, out=torch.empty_like(y)), y)


@pytest.mark.parametrize('scale', [1e-38, 1e-20, 1e19, 1e38])
def test_scales_of_narrow_ones(scale):
    from d1.muon import orthogonalize
    for size in ((30, 150), (1000, 30)):
        x = matrix(*size).clamp(-3, 3)
        assert distance(orthogonalize(x * scale), exact((x * scale).double())) <= 2.0 ** -12 + OUT[torch.bfloat16]


def test_zeros_and_infinities_in_narrow_ones():
    from d1.muon import orthogonalize
    for size in ((60, 90), (900, 60)):
        x = matrix(4, *size)
        x[0] = 0
        x[1, 3, 4] = float('nan')
        x[2, 5, 6] = float('inf')
        y = orthogonalize(x)
        assert (y[0] == 0).all() and y[1].isnan().any() and y[2].isnan().any() and torch.equal(y[3], orthogonalize(x[3]))


def test_stacks_and_pitches_of_narrow_ones():
    from d1.muon import orthogonalize
    for size in ((20, 1100), (1100, 20), (33, 70)):
        m, n = size
        x = matrix(2, 3, *size)
        y = orthogonalize(x)
        assert distance(y, exact(x)) <= 2.0 ** -12 + OUT[y.dtype]
        for i in range(2):
            for j in range(3):
                assert torch.equal(y[i, j], orthogonalize(x[i, j]))
        wide = torch.zeros(2, 3, m + 10, n + 31, device='cuda')
        wide[..., 5:5 + m, 3:3 + n] = x
        assert torch.equal(orthogonalize(wide[..., 5:5 + m, 3:3 + n]), y)
        assert torch.equal(orthogonalize(x[:1, :1].expand(2, 3, m, n)), y[:1, :1].expand(2, 3, m, n))


def test_unaligned_narrow_tensors():
    from d1.muon import Muon, orthogonalize
    for size in ((12, 40), (60, 8), (16, 1200), (1200, 16), (64, 64)):
        n = size[0] * size[1]
        mk = lambda dtype, k: torch.zeros(n + 8, device='cuda', dtype=dtype)[k:k + n].view(size)
        p, g, c = mk(torch.float32, 1), mk(torch.bfloat16, 3), mk(torch.bfloat16, 1)
        q, h, d = (t.clone() for t in (p, g, c))
        for t in (p, q):
            t.copy_(matrix(*size))
        for t in (g, h):
            t.copy_(matrix(*size, seed=3))
        for args in ((p, g, c), (q, h, d)):
            Muon([args[0]], [args[1]], copies=[args[2]], lr=0.1).step()
        assert torch.equal(p, q) and torch.equal(c, d) and torch.equal(c, p.to(torch.bfloat16))
        assert torch.equal(orthogonalize(g, out=c), orthogonalize(h))


def test_graphs_and_streams_of_narrow_ones():
    from d1.muon import orthogonalize
    for shapes in ([(28, 512), (12, 90), (64, 64)], [(28, 2512), (12, 90)]):   # one launch, three
        a, pa, ga, ca = optimizer(shapes, lr=0.01)
        b, pb, gb, cb = optimizer(shapes, lr=0.01)
        a.step(), b.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.step()
        for k in range(3):
            for g, h in zip(ga, gb):
                g.mul_(0.9).add_(1e-4 * k)
                h.copy_(g)
            graph.replay()
            b.step()
        assert all(torch.equal(p, q) for p, q in zip(pa + ca, pb + cb)) and torch.equal(a.momentum, b.momentum)
    for size in ((30, 200), (2000, 30)):
        x, z = matrix(*size), matrix(*size, seed=4)
        want, wanted = orthogonalize(x), orthogonalize(z)
        held, graphs, outs = z.clone(), [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(orthogonalize(held))
        held.copy_(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for g in graphs:
                g.replay()
            with torch.cuda.stream(side):
                eager = orthogonalize(z)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs) and torch.equal(eager, wanted)


NARROW = [(32, 90), (64, 288), (900, 12), (3, 28, 700), (1, 50), (50, 1), (5, 5), (1300, 61)]  # all taken without X


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('grad', [torch.float32, torch.bfloat16])
def test_step_of_narrow_ones(grad, nesterov):
    test_step(grad, nesterov, NARROW)


@pytest.mark.parametrize('size', [(2048, 2500), (2500, 2048), (1300, 5000)])
def test_large(size):
    """Sizes that pairs of CTAs take together, whole tiles and ragged ones."""
    from d1.muon import orthogonalize
    for kind in ('full', 'low'):
        x = matrix(*size, kind=kind)
        assert distance(orthogonalize(x), exact(x)) <= NS + OUT[torch.bfloat16]


def test_stacks_and_pitches():
    from d1.muon import orthogonalize
    x = matrix(3, 4, 70, 90)
    y = orthogonalize(x)
    for i in range(3):
        for j in range(4):
            assert torch.equal(y[i, j], orthogonalize(x[i, j]))
    wide = torch.zeros(3, 4, 80, 200, device='cuda')
    wide[..., 5:75, 100:190] = x
    assert torch.equal(orthogonalize(wide[..., 5:75, 100:190]), y)
    assert torch.equal(orthogonalize(x[:1, :1].expand(2, 3, 70, 90)), y[:1, :1].expand(2, 3, 70, 90))
    many = matrix(40, 300, 260)
    y = orthogonalize(many)      # enough for pairs of CTAs
    assert distance(y, exact(many)) <= NS + OUT[y.dtype]
    assert orthogonalize(matrix(0, 5, 5)).shape == (0, 5, 5)


@pytest.mark.parametrize('scale', [1e-38, 1e-20, 1e19, 1e38])
def test_scales(scale):
    """The norm is one of fp64: gradients whose squares pass fp32 on either side."""
    from d1.muon import orthogonalize
    x = matrix(100, 150).clamp(-3, 3)
    assert distance(orthogonalize(x * scale), exact(x.double() * scale)) <= NS + OUT[torch.bfloat16] + (1e-6 if scale > 1e-30 else 1e-2)


def test_zeros_and_infinities():
    from d1.muon import orthogonalize
    x = matrix(3, 70, 90)
    x[0] = 0
    x[1, 3, 4] = float('nan')
    y = orthogonalize(x)
    assert (y[0] == 0).all() and y[1].isnan().any() and torch.equal(y[2], orthogonalize(x[2]))


SHAPES = [(32, 90), (64, 288), (512, 700), (700, 300), (28, 512), (2, 3, 20, 33), (1, 50), (50, 1), (5, 5)]


def optimizer(shapes, grad=torch.float32, copies=True, seed=0, **more):
    from d1.muon import Muon
    params = [0.05 * matrix(*s, seed=seed + 1) for s in shapes]
    grads = [(1e-3 * matrix(*s, seed=seed + 2)).to(grad) for s in shapes]
    c = [p.to(torch.bfloat16) for p in params] if copies else None
    return Muon(params, grads, copies=c, **more), params, grads, c


SMALL = [(32, 90), (64, 288), (100, 120), (120, 900), (3, 28, 300), (1, 50), (50, 1), (5, 5)]  # one launch for all products


@pytest.mark.parametrize('shapes', [SHAPES, SMALL])
@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('grad', [torch.float32, torch.bfloat16])
def test_step(grad, nesterov, shapes):
    """Three steps; the update is taken from the parameters' change at a rate at which their rounding (2^-24 of 0.05) is far below it."""
    opt, params, grads, copies = optimizer(shapes, grad, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=[0.1 * (i % 3) for i in range(len(shapes))])
    m = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    for step in range(3):
        before = [p.double() for p in params]
        for i, g in enumerate(grads):
            g.copy_(1e-3 * matrix(*shapes[i], seed=50 * step + i, kind='full' if i % 2 else 'low'))
        opt.step()
        for i, (p, g) in enumerate(zip(params, grads)):
            was = m[i]
            m[i] = 0.9 * was + g.double()
            mag = 0.9 * was.abs() + g.double().abs()
            assert ((opt.momentum_of(i).double() - m[i]).abs() <= (step + 2) * 2.0 ** -23 * mag + 1e-40).all()
            m[i] = opt.momentum_of(i).double()
            u = g.double() + 0.9 * m[i] if nesterov else m[i]
            rate = 0.05 * 0.2 * max(p.shape[-2:]) ** 0.5
            x = (before[i] * (1 - 0.05 * opt.decay[i]) - p.double()) / rate
            slack = 2.0 ** -22 * 0.3 / (rate * max(p.shape[-2:]) ** -0.5)  # of the parameters' own rounding, per element of X's size
            assert distance(x, exact(u)) <= bound(x) + slack, i
            assert torch.equal(copies[i], p.to(torch.bfloat16))


def test_step_of_large_layers():
    shapes = [(1024, 1024)] * 6 + [(2048, 512), (512, 2100)]
    opt, params, grads, _ = optimizer(shapes, torch.bfloat16, copies=False, lr=0.05, weight_decay=0.0)
    before = [p.double() for p in params]
    opt.step()
    for p, b, g, s in zip(params, before, grads, shapes):
        u = g.double() * (1 + 0.95)
        assert distance((b - p.double()) / (0.05 * 0.2 * max(s) ** 0.5), exact(u)) <= NS + 1e-4


def test_unaligned_tensors():
    """Parameters, gradients and copies that start at odd elements of a larger buffer."""
    from d1.muon import Muon
    for size in ((40, 30), (33, 65), (128, 130)):
        n = size[0] * size[1]
        mk = lambda dtype, k: torch.zeros(n + 8, device='cuda', dtype=dtype)[k:k + n].view(size)
        p, g, c = mk(torch.float32, 1), mk(torch.bfloat16, 3), mk(torch.bfloat16, 1)
        q, h, d = (t.clone() for t in (p, g, c))
        for t in (p, q):
            t.copy_(matrix(*size))
        for t in (g, h):
            t.copy_(matrix(*size, seed=3))
        for args in ((p, g, c), (q, h, d)):
            Muon([args[0]], [args[1]], copies=[args[2]], lr=0.1).step()
        assert torch.equal(p, q) and torch.equal(c, d)


def test_state_and_new_gradients():
    a, pa, ga, _ = optimizer(SHAPES, lr=0.01)
    a.step()
    b, pb, gb, _ = optimizer(SHAPES, lr=0.01, seed=9)
    for p, q in zip(pb, pa):
        p.copy_(q)
    b.load_state_dict(a.state_dict())
    other = [g * 2 - 1e-4 for g in ga]
    a.set_grads(other)
    b.set_grads([g.clone() for g in other])
    a.step()
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(pa, pb)) and torch.equal(a.momentum, b.momentum)
    a.step(lr=0.0)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))
    with pytest.raises(ValueError):
        a.load_state_dict({'momentum': a.momentum[:-1]})
    with pytest.raises(ValueError):
        a.load_state_dict({'m': a.momentum})


def test_graphs_and_streams():
    """A captured step reads the gradients as they are at its replay, and goes on from the eager steps' state; two
    orthogonalisations captured into two graphs and an eager one on another stream do not disturb one another."""
    from d1.muon import orthogonalize
    a, pa, ga, ca = optimizer(SHAPES, lr=0.01)
    b, pb, gb, cb = optimizer(SHAPES, lr=0.01)
    a.step(), b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(3):
        for g, h in zip(ga, gb):
            g.mul_(0.9).add_(1e-4 * k)
            h.copy_(g)
        graph.replay()
        b.step()
    assert all(torch.equal(p, q) for p, q in zip(pa + ca, pb + cb)) and torch.equal(a.momentum, b.momentum)
    x, z = matrix(300, 200), matrix(300, 200, seed=4)
    want, wanted = orthogonalize(x), orthogonalize(z)
    held, graphs, outs = z.clone(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(orthogonalize(held))
    held.copy_(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            eager = orthogonalize(z)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and torch.equal(eager, wanted)


def test_the_same_bits_each_time():
    from d1.muon import orthogonalize
    x = matrix(700, 1000)
    y = orthogonalize(x)
    assert all(torch.equal(orthogonalize(x), y) for _ in range(3))


def test_leaves_are_marked():
    from d1.muon import Muon
    w = matrix(20, 30).requires_grad_()
    x = matrix(5, 20).requires_grad_()     # its gradient takes w, so that the graph keeps it
    opt = Muon([w], [torch.ones_like(w)])
    loss = (x @ w).square().sum()
    opt.step()
    with pytest.raises(RuntimeError):      # the step has overwritten what the graph kept
        loss.backward()


def test_refusals():
    from d1.muon import Muon, orthogonalize
    p, g = matrix(8, 16), matrix(8, 16, seed=1)
    flat = torch.zeros(2000, device='cuda')
    for bad in (lambda: Muon([], []), lambda: Muon([p], []), lambda: Muon([p], [g[:4]]), lambda: Muon([p], [g.half()]), lambda: Muon([p.half()], [g]),
                lambda: Muon([p.T], [g.T]), lambda: Muon([p[0]], [g[0]]), lambda: Muon([p], [p]), lambda: Muon([p, p], [g, g]),
                lambda: Muon([p], [g], lr=-1.0), lambda: Muon([p], [g], momentum=1.0), lambda: Muon([p], [g], steps=0), lambda: Muon([p], [g], steps=65),
                lambda: Muon([p], [g], copies=[p]), lambda: Muon([p], [g], copies=[]), lambda: Muon([p], [g.cpu()]), lambda: Muon([p[:0]], [g[:0]]),
                lambda: Muon([p], [g], weight_decay=[0.1, 0.1]), lambda: Muon([flat[:100].view(10, 10), flat[50:150].view(10, 10)], [g, g]),
                lambda: orthogonalize(p[0]), lambda: orthogonalize(p.double()), lambda: orthogonalize(p.T), lambda: orthogonalize(p, steps=0),
                lambda: orthogonalize(p, out=torch.empty(8, 16, device='cuda')), lambda: orthogonalize(p[:, :0]),
                lambda: orthogonalize(p, out=torch.empty(8, 15, device='cuda', dtype=torch.float16)),
                lambda: orthogonalize(matrix(2, 3, 4, 8)[:, :2])):
        with pytest.raises(ValueError):
            bad()
    half = p.half()
    from d1._lib import D1Error
    with pytest.raises(D1Error):
        orthogonalize(half, out=half)
