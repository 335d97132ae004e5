"""Newton-Schulz steps up to the most that are accepted, on matrices of low rank too: there the steps amplify what rounding leaves in the
directions that the matrix does not have, until those have singular values of their own. Every singular value then is one of the polynomial's, which
maps [0, 1.21] into itself; its largest value there is 1.2025. Products round by under 2^-8 of it (single ones, where both sides are above 64), a bf16
result by 2^-9: all stay below 1.22."""
import pytest
import torch

from test_muon_gpu import OUT, distance, exact, matrix, optimizer

pytestmark = pytest.mark.gpu
MOST = 1.22
STEPS = [6, 8, 16, 20, 32, 64]
# one launch or three with five steps, tall and wide, stacks
SIZES = [(64, 512), (28, 512), (512, 28), (64, 64), (7, 3000), (3000, 33), (64, 8192), (3, 50, 60), (40, 16, 24), (20, 64, 1100), (130, 170), (2, 300, 100)]


def of_kind(size, kind):
    x = matrix(*size, kind='full')
    if kind == 'low':
        return matrix(*size, kind='low')
    if kind == 'one':        # rank 1
        return x[..., :1] @ x[..., :1, :]
    if kind == 'twice':      # every row twice
        return x[..., :(size[-2] + 1) // 2, :].repeat_interleave(2, -2)[..., :size[-2], :].contiguous()
    return x


@pytest.mark.parametrize('kind', ['low', 'one', 'twice', 'full'])
@pytest.mark.parametrize('size', SIZES)
def test_singular_values_stay(size, kind):
    from d1.muon import muon_error, orthogonalize
    x = of_kind(size, kind)
    for steps in STEPS:
        for precise in (False, True):
            y = orthogonalize(x, steps=steps, precise=precise)
            assert y.isfinite().all(), steps
            assert torch.linalg.matrix_norm(y.double(), ord=2).max() <= MOST, steps
    assert muon_error() == 0


@pytest.mark.parametrize('size', [(64, 512), (28, 512), (3000, 33), (3, 50, 60)])
def test_more_steps_of_full_rank(size):
    """Pairs of fp16: under 2^-18 a step, whose own factor is about 1 by then; at most 4 in each of the first five: 2^-12."""
    from d1.muon import orthogonalize
    x = matrix(*size)
    for steps in (6, 8, 12):
        y = orthogonalize(x, steps=steps, out=torch.empty(x.shape, dtype=torch.float16, device='cuda'))
        assert distance(y, exact(x, steps)) <= 2.0 ** -12 + OUT[y.dtype], steps


@pytest.mark.parametrize('steps', [6, 20, 64])
def test_the_optimizer(steps):
    """Narrow ones alone and beside a wide one: neither leaves a NaN."""
    for shapes in ([(32, 90), (64, 288), (3, 28, 300), (1, 50)], [(28, 3000), (64, 64)], [(32, 90), (200, 300)]):
        opt, params, grads, copies = optimizer(shapes, steps=steps, lr=0.05)
        for g in grads:
            g.copy_(1e-3 * of_kind(tuple(g.shape), 'one'))
        before = [p.clone() for p in params]
        for _ in range(3):
            opt.step()
        for p, b, c in zip(params, before, copies):
            rate = 0.05 * 0.2 * max(p.shape[-2:]) ** 0.5
            assert p.isfinite().all() and torch.equal(c, p.to(torch.bfloat16))
            assert torch.linalg.matrix_norm((p - b).double(), ord=2).max() <= 3 * (MOST * rate + 0.05 * 0.01 * 0.05 * 100)
