"""Layer norm (d1.layer_norm) against the definition in 64 bits.

Tolerances. A row's mean is a sum of n terms in fp32: at most n / threads + 10
additions in turn, 2^-24 of the row's largest magnitude each; 64 of them cover
every size here (a thread adds at most 32 terms of a held row, n / 1024 of a
longer one). rstd then has that relative error of x - mean against the row's
spread, and xhat, dx and the products a few roundings more. Column sums add at
most rows / parts + 37 terms in turn. Results of 16 bits add half a unit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (x - mean) * rstd
    return xhat * (1 if w is None else w.double()) + (0 if b is None else b.double()), mean, rstd, xhat


def gradients(dy, xhat, rstd, w):
    dy = dy.double()
    g = dy if w is None else dy * w.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0), g


def check_forward(x, w, b, eps, got):
    y, mean, rstd = got
    want, mu, rs, xhat = definition(x, w, b, eps)
    size = x.double().abs().amax(-1, keepdim=True)
    dm = 64 * U * size                                 # of the mean, and of each x - mean
    assert ((mean.double() - mu[..., 0]).abs() <= dm[..., 0]).all()
    rel = 64 * U + dm * rs                             # of rstd
    assert ((rstd.double() - rs[..., 0]).abs() <= (rel * rs)[..., 0]).all()
    scale = 1 if w is None else w.double().abs()
    tol = (xhat.abs() * (rel + 4 * U) + dm * rs) * scale + 4 * U * want.abs() + (0 if b is None else 2 * U * b.double().abs())
    assert ((y.double() - want).abs() <= tol + HALF[x.dtype] * (want.abs() + tol) + 2.0 ** -25).all()


def check_backward(dy, x, w, eps, got, stats):
    dx, dw, db = got
    mu, rs = stats[0].double()[:, None], stats[1].double()[:, None]
    xhat = (x.double() - mu) * rs                      # of the statistics that the call was given
    want, sw, sb, g = gradients(dy, xhat, rs, w)
    top, n = g.abs().amax(1, keepdim=True), x.shape[1]
    err = 3 * U * (xhat.abs() + (x.double() * rs).abs())   # of xhat
    worst = (xhat.abs() + err).amax(1, keepdim=True)
    tol = rs * (8 * U * g.abs() + 64 * U * top + (err + 4 * U * xhat.abs()) * (g * xhat).mean(1, keepdim=True).abs()
                + xhat.abs() * top * (64 * U * worst + err.mean(1, keepdim=True)))
    assert ((dx.double() - want).abs() <= tol + HALF[x.dtype] * (want.abs() + tol) + 2.0 ** -25).all()
    terms = (x.shape[0] + 100) * U
    tw = terms * (dy.double() * xhat).abs().sum(0) + (dy.double().abs() * err).sum(0)
    assert ((dw.double() - sw).abs() <= tw + 1e-30).all()
    assert ((db.double() - sb).abs() <= terms * dy.double().abs().sum(0) + 1e-30).all()


def data(rows, n, dtype, seed, pitch=None, offset=0):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def make(scale, shift):
        flat = scale * torch.randn(rows * (pitch or n) + offset, device='cuda', generator=g) + shift
        return flat.to(dtype)[offset:].view(rows, pitch or n)[:, :n]
    x, dy = make(2.0, 0.7), make(0.3, 0.05)
    w, b = 1 + 0.2 * torch.randn(n, device='cuda', generator=g), torch.randn(n, device='cuda', generator=g)
    return x, dy, w, b


SIZES = [1, 2, 7, 8, 63, 64, 65, 255, 256, 264, 511, 512, 513, 1000, 1024, 1025, 1111, 2048, 2050, 4096, 5001, 8192,
         8193, 12288, 16384, 20000, 32768, 33001]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', SIZES)
def test_against_the_definition(n, dtype):
    from d1.layer_norm import layer_norm, layer_norm_backward
    for rows in (1, 3, 45) + ((700,) if n <= 1111 else ()):
        x, dy, w, b = data(rows, n, dtype, 31 * n + rows)
        got = layer_norm(x, w, b)
        check_forward(x, w, b, 1e-5, got)
        check_backward(dy, x, w, 1e-5, layer_norm_backward(dy, x, got[1], got[2], w), got[1:])
        got = layer_norm(x, eps=0.1)
        check_forward(x, None, None, 0.1, got)
        check_backward(dy, x, None, 0.1, layer_norm_backward(dy, x, got[1], got[2]), got[1:])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [1500, 2050, 4096, 5001, 8192, 8200, 12033, 16384])
def test_many_long_rows(n, dtype):                     # a block's rows follow one another through shared memory
    from d1.layer_norm import layer_norm, layer_norm_backward
    x, dy, w, b = data(700, n, dtype, 17 * n)
    y, mean, rstd = layer_norm(x, w, b)
    check_forward(x, w, b, 1e-5, (y, mean, rstd))
    check_backward(dy, x, w, 1e-5, layer_norm_backward(dy, x, mean, rstd, w), (mean, rstd))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [3, 16, 33, 64, 65, 72, 100, 128, 130, 200, 256, 279, 384, 521, 767])
def test_thousands_of_short_rows(n, dtype):            # in the teams that many rows have, the last one not full
    from d1.layer_norm import layer_norm, layer_norm_backward
    x, dy, w, b = data(5003, n, dtype, 19 * n)
    y, mean, rstd = layer_norm(x, w, b)
    check_forward(x, w, b, 1e-5, (y, mean, rstd))
    check_backward(dy, x, w, 1e-5, layer_norm_backward(dy, x, mean, rstd, w), (mean, rstd))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [8, 500, 512, 1024, 4096, 9000])
def test_pitches_and_alignments(n, dtype):
    from d1.layer_norm import layer_norm, layer_norm_backward
    for pitch, offset in ((n + 8, 0), (n + 1, 0), (n, 1), (n + 16, 8)):
        x, dy, w, b = data(37, n, dtype, n, pitch, offset)
        got = layer_norm(x, w, b)
        check_forward(x, w, b, 1e-5, got)
        wide = torch.full((37, n + 5), 9.0, device='cuda', dtype=dtype)
        dx, dw, db = layer_norm_backward(dy, x, got[1], got[2], w, out=wide[:, 2:2 + n])
        assert (wide[:, :2] == 9).all() and (wide[:, 2 + n:] == 9).all()
        check_backward(dy, x, w, 1e-5, (dx, dw, db), got[1:])
        same = x.clone()
        layer_norm(same, w, b, out=same)
        assert torch.equal(same, layer_norm(x.clone(), w, b)[0])
    one = torch.randn(1, n, device='cuda').to(dtype).expand(5, n)   # one row, read five times
    check_forward(one, None, None, 1e-5, layer_norm(one))


def test_many_rows_and_the_same_bits():
    from d1.layer_norm import layer_norm, layer_norm_backward
    for rows, n in ((20011, 48), (9001, 512), (3001, 2048), (1500, 6000)):
        x, dy, w, b = data(rows, n, torch.bfloat16, n)
        got = layer_norm(x, w, b)
        check_forward(x, w, b, 1e-5, got)
        grads = layer_norm_backward(dy, x, got[1], got[2], w)
        check_backward(dy, x, w, 1e-5, grads, got[1:])
        assert all(torch.equal(a, b) for a, b in zip(grads, layer_norm_backward(dy, x, got[1], got[2], w)))


def test_shapes_streams_and_graphs():
    from d1.layer_norm import layer_norm, layer_norm_backward
    x, dy, w, b = data(24, 512, torch.bfloat16, 4)
    want = layer_norm(x, w, b)
    cube = layer_norm(x.view(2, 3, 4, 512), w, b)
    assert cube[0].shape == (2, 3, 4, 512) and cube[1].shape == (2, 3, 4) and torch.equal(cube[0].view(24, 512), want[0])
    line = layer_norm(x[3], w, b)
    assert line[1].shape == () and torch.equal(line[0], want[0][3])
    grads = layer_norm_backward(dy, x, want[1], want[2], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm(x, w, b) + layer_norm_backward(dy, x, want[1], want[2], w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want + grads))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer_norm(x, w, b)
        held += layer_norm_backward(dy, x, held[1], held[2], w)
    x.mul_(0.5)
    graph.replay()
    again = layer_norm(x, w, b)
    again += layer_norm_backward(dy, x, again[1], again[2], w)
    assert all(torch.equal(a, c) for a, c in zip(held, again))


def test_edges():
    from d1.layer_norm import layer_norm, layer_norm_backward
    for n in (1, 40, 512, 3000, 40000):
        const = torch.full((4, n), 3.0, device='cuda')
        y, mean, rstd = layer_norm(const)
        assert (y == 0).all() and (mean == 3).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))
        big = torch.randn(4, n, device='cuda') + 1e4   # a mean far above the spread
        check_forward(big, None, None, 1e-5, layer_norm(big))
        bad = torch.randn(4, n, device='cuda')
        bad[1, n // 2], bad[2, 0] = float('nan'), float('inf')
        y = layer_norm(bad)[0]
        assert y[0].isfinite().all() and y[3].isfinite().all() and y[1].isnan().all() and y[2].isnan().any()
        none = torch.empty(0, n, device='cuda')
        y, mean, rstd = layer_norm(none)
        assert y.shape == (0, n) and mean.shape == (0,)
        dx, dw, db = layer_norm_backward(none, none, mean, rstd)
        assert dx.shape == (0, n) and (dw == 0).all() and (db == 0).all()


def test_gradient_against_differences():
    """Central differences in the forward pass: with a step of 2^-5 of unit inputs the truncation is below
    2^-10 / 6 times the third derivative (under 6 for these weights) and the noise 64 * 2^-24 * 4 * 40 / 2^-4."""
    from d1.layer_norm import layer_norm, layer_norm_backward
    g = torch.Generator(device='cuda').manual_seed(9)
    n, h = 40, 2.0 ** -5
    x, c = torch.randn(n, device='cuda', generator=g), torch.randn(n, device='cuda', generator=g)
    w, b = torch.rand(n, device='cuda', generator=g) + 0.5, torch.randn(n, device='cuda', generator=g)
    eye = torch.eye(n, device='cuda') * h
    loss = lambda *a: (layer_norm(*a)[0].double() * c).sum(-1)
    y, mean, rstd = layer_norm(x[None], w, b)
    dx, dw, db = layer_norm_backward(c[None].contiguous(), x[None], mean, rstd, w)
    assert (dx[0] - (loss(x + eye, w, b) - loss(x - eye, w, b)) / (2 * h)).abs().max() <= 1e-2
    for k in range(0, n, 7):
        for grad, at in ((dw, (w + eye[k], b, w - eye[k], b)), (db, (w, b + eye[k], w, b - eye[k]))):
            want = (loss(x, *at[:2]) - loss(x, *at[2:])) / (2 * h)
            assert (grad[k] - want).abs() <= 1e-2


def test_offsets_past_32_bits():
    from d1.layer_norm import layer_norm, layer_norm_backward
    pitch = 2 ** 31 + 8
    store = torch.zeros(pitch + 512, dtype=torch.bfloat16, device='cuda')
    x = torch.as_strided(store, (2, 512), (pitch, 1))
    x.copy_(torch.randn(2, 512, device='cuda'))
    got = layer_norm(x)
    check_forward(x, None, None, 1e-5, got)
    dy = torch.randn(2, 512, device='cuda').bfloat16()
    a, b = layer_norm_backward(dy, x, got[1], got[2]), layer_norm_backward(dy, x.contiguous(), got[1], got[2])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals():
    from d1.layer_norm import layer_norm, layer_norm_backward
    x, w = torch.randn(4, 40, device='cuda'), torch.ones(40, device='cuda')
    y, mean, rstd = layer_norm(x)
    for bad in (lambda: layer_norm(x.double()), lambda: layer_norm(x.T), lambda: layer_norm(x.cpu()),
                lambda: layer_norm(x, w[:39]), lambda: layer_norm(x, w.bfloat16()), lambda: layer_norm(x, w, w.cpu()),
                lambda: layer_norm(x, eps=-1.0), lambda: layer_norm(x, out=x[:2]), lambda: layer_norm(x[:, :0]),
                lambda: layer_norm(torch.tensor(1.0, device='cuda')), lambda: layer_norm(x, out=y.bfloat16()),
                lambda: layer_norm_backward(y[:3], x, mean, rstd), lambda: layer_norm_backward(y, x, mean[:3], rstd),
                lambda: layer_norm_backward(y, x, mean, rstd.double()),
                lambda: layer_norm_backward(y, x, mean, rstd, out=x),
                lambda: layer_norm_backward(y, x, mean, rstd, out=y)):
        with pytest.raises(ValueError):
            bad()
