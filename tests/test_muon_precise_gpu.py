"""Newton-Schulz products of pairs of fp16 (`precise`, and fp16 results) where both sides are above 64.

Tolerances. A pair holds 22 bits and a product leaves lo lo out: 2^-21 of each operand. A product adds up its sum 16 elements and a term
at a time in fp32; were all of those truncated alike, a sum over 512 elements (96 of them) would be off by 96 * 2^-23. A error e of A moves
F X by |A (b + 2 c A)| e < 1.5 e of it, F's and X's own sums by e each: 3.5 e = 2^-14.6 a step, and 2^-12.3 in five, whose own factor is at
most 1 in directions that X has. In those that it hardly has (low rank) 2^-21 grows by 3.44 a step, 485 in all: 2^-12.1. Both: 2^-11. Sums of 1,800
elements are off by 3.5 times as much: 2^-10.4 and 2^-12.1, under 2^-10. A 16-bit result adds 2^-9 (bf16) or 2^-12 (fp16).
"""
import pytest
import torch

from test_muon_gpu import OUT, distance, exact, matrix, optimizer

pytestmark = pytest.mark.gpu


def near(x):
    return 2.0 ** -11 if max(x.shape[-2:]) <= 520 else 2.0 ** -10


SIZES = [(65, 65), (65, 129), (128, 128), (129, 65), (200, 129), (256, 512), (512, 130), (500, 500), (1003, 1777), (1300, 700)]


@pytest.mark.parametrize('kind', ['full', 'low'])
@pytest.mark.parametrize('size', SIZES)
def test_half_results_have_the_bits_of_their_type(size, kind):
    from d1.muon import muon_error, orthogonalize
    for dtype in (torch.float16, torch.float32):
        x = matrix(*size, kind=kind, dtype=dtype)
        y = orthogonalize(x, out=torch.empty(size, dtype=torch.float16, device='cuda'))
        assert distance(y, exact(x)) <= near(x) + OUT[y.dtype]
        assert torch.equal(orthogonalize(x, out=torch.empty_like(y), precise=True), y)
        y = orthogonalize(x, out=torch.empty(size, dtype=torch.bfloat16, device='cuda'), precise=True)
        assert distance(y, exact(x)) <= near(x) + OUT[y.dtype]
    assert muon_error() == 0


def test_the_choice():
    """bf16 results, and whoever asks for it, take single products."""
    from d1.muon import orthogonalize
    x = matrix(200, 300)
    single, half = orthogonalize(x, precise=False), torch.empty(200, 300, dtype=torch.float16, device='cuda')
    assert torch.equal(orthogonalize(x), single)
    assert distance(orthogonalize(x, out=half, precise=False), exact(x)) <= 2.0 ** -8 + OUT[torch.float16]
    assert not torch.equal(orthogonalize(x, precise=True), single)


@pytest.mark.parametrize('batch, size', [(1, (128, 2000)), (14, (100, 700)), (40, (128, 500)), (70, (70, 90)), (40, (300, 260)), (3, (128, 4100))])
def test_stacks(batch, size):
    """Small ones in one launch (their long sums divided), and in the products' launches by single CTAs and by pairs."""
    from d1.muon import muon_error, orthogonalize
    x = matrix(batch, *size)
    half = lambda: torch.empty(x.shape, dtype=torch.float16, device='cuda')
    y = orthogonalize(x, out=half())
    # long sums once more: of 4,100 elements eight times those of 512, 2^-9.3
    assert distance(y, exact(x)) <= max(near(x), max(size) / 512 * 2.0 ** -12.3) + OUT[y.dtype]
    assert all(torch.equal(orthogonalize(x, out=half()), y) for _ in range(2))
    assert muon_error() == 0


@pytest.mark.parametrize('size', [(2048, 2500), (2500, 2048)])
def test_large(size):
    """By pairs of CTAs; truncated sums of 2,500 elements: 2^-10."""
    from d1.muon import orthogonalize
    for kind in ('full', 'low'):
        x = matrix(*size, kind=kind)
        assert distance(orthogonalize(x, out=torch.empty(size, dtype=torch.float16, device='cuda')), exact(x)) <= 2.0 ** -10 + OUT[torch.float16]


def test_zeros_nan_and_pitches():
    from d1.muon import orthogonalize
    x = matrix(3, 170, 90)
    x[0] = 0
    x[1, 3, 4] = float('nan')
    wide = torch.zeros(3, 180, 200, device='cuda')
    wide[:, 5:175, 100:190] = x
    y = orthogonalize(x, precise=True)
    assert (y[0] == 0).all() and y[1].isnan().any() and torch.equal(y[2], orthogonalize(x[2], precise=True))
    assert torch.equal(orthogonalize(wide[:, 5:175, 100:190], precise=True)[::2], y[::2])


@pytest.mark.parametrize('shapes', [[(512, 500), (500, 300), (64, 288), (3, 70, 130), (1, 50)], [(100, 120), (120, 500), (30, 90)], [(32, 90), (64, 64)]])
def test_steps_of_the_optimizer(shapes):
    """X is taken from the parameters' change; their rounding as in the test of single products."""
    opt, params, grads, copies = optimizer(shapes, lr=0.05, momentum=0.9, weight_decay=0.0, precise=True)
    for step in range(2):
        before = [p.double() for p in params]
        for i, g in enumerate(grads):
            g.copy_(1e-3 * matrix(*shapes[i], seed=50 * step + i, kind='full' if i % 2 else 'low'))
        opt.step()
        for i, (p, g) in enumerate(zip(params, grads)):
            rate = 0.05 * 0.2 * max(p.shape[-2:]) ** 0.5
            slack = 2.0 ** -22 * 0.3 / (rate * max(p.shape[-2:]) ** -0.5)
            u = g.double() + 0.9 * opt.momentum_of(i).double()
            assert distance((before[i] - p.double()) / rate, exact(u)) <= near(p) + slack, i
            assert torch.equal(copies[i], p.to(torch.bfloat16))


def test_graphs():
    """Captured with single products beside it: each has a work buffer of its own size."""
    from d1.muon import orthogonalize
    x, z = matrix(300, 200), matrix(300, 200, seed=4)
    want = [orthogonalize(x, precise=p) for p in (True, False)]
    held, graphs, outs = z.clone(), [], []
    for p in (True, False):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(orthogonalize(held, precise=p))
    held.copy_(x)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
