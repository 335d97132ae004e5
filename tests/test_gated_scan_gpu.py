"""The gated recurrence (d1.gated_scan) against the steps themselves in 64 bits.

Tolerances. A decay is e^-|g| (expf: 1 ulp), 1 + e, a reciprocal and a product: under 6 half steps
(2^-24 each) of a and of 1 - a; the state's and the input's products and sums add 3 more. Such an
error of the terms at step t, 10 * 2^-24 of their magnitude mag_t = a_t mag_{t-1} + |b_t|, is carried on like
the state itself, so that tol_t = a_t tol_{t-1} + 10 * 2^-24 mag_t bounds all of them; composing chunks
multiplies the same decays in another order, at most twice the roundings. A result is rounded once more to its type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 20 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rounding(value, dtype):
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps


def factors(gate, form):
    g = gate.double()
    return (torch.sigmoid(g), torch.sigmoid(-g)) if form == 'average' else (g.exp(), torch.ones_like(g))


def forward(x, gate, h0, reset, form):
    a, w = factors(gate, form)
    h = torch.zeros(x.shape[1:], dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    mag, tol, y, tols = h.abs(), torch.zeros_like(h), [], []
    for t in range(x.shape[0]):
        cut = torch.zeros_like(h, dtype=torch.bool) if reset is None else (reset[t] != 0).unsqueeze(-1).expand_as(h)
        b = w[t] * x[t].double()
        h, mag, tol = (torch.where(cut, 0.0, v) for v in (h, mag, tol))
        h, mag = a[t] * h + b, a[t] * mag + b.abs()
        tol = a[t] * tol + U * mag
        y.append(h)
        tols.append(tol)
    return torch.stack(y), torch.stack(tols)


def backward(dy, x, gate, y, h0, reset, dlast, form):
    a, w = factors(gate, form)
    e = torch.zeros(x.shape[1:], dtype=torch.float64, device=x.device) if dlast is None else dlast.double()
    mag, tol = e.abs(), torch.zeros_like(e)
    start = torch.zeros_like(e) if h0 is None else h0.double()
    out = []
    for t in reversed(range(x.shape[0])):
        cut = torch.zeros_like(e, dtype=torch.bool) if reset is None else (reset[t] != 0).unsqueeze(-1).expand_as(e)
        D, mag = dy[t].double() + e, dy[t].double().abs() + mag
        tol = tol + U * mag
        h = torch.where(cut, 0.0, y[t - 1].double() if t else start)
        # the two terms of dg are rounded apart, so that their magnitudes count
        inner, size = (h - x[t].double(), h.abs() + x[t].double().abs()) if form == 'average' else (h, h.abs())
        part = a[t] * w[t]
        out.append((D * w[t], (tol + U * mag) * w[t], D * inner * part, (tol * inner.abs() + U * mag * size) * part))
        e, mag, tol = (torch.where(cut, 0.0, a[t] * v) for v in (D, mag, tol))
    dx, tdx, dg, tdg = (torch.stack(v[::-1]) for v in zip(*out))
    return dx, tdx, dg, tdg, e, tol + U * mag


def inputs(shape, dtype, form='average', seed=0, rate=0.1):
    g = torch.Generator(device='cuda').manual_seed(seed + sum(shape))
    new = lambda *s: torch.randn(s, device='cuda', generator=g)
    gate = new(*shape) * 2 + 1 if form == 'average' else -(new(*shape) - 2).exp()
    reset = torch.rand(shape[:-1], device='cuda', generator=g) < rate
    return new(*shape).to(dtype), gate.to(dtype), new(*shape[1:]), reset, new(*shape).to(dtype), new(*shape[1:])


def check(x, gate, h0, reset, dy, dlast, form):
    from d1.gated_scan import gated_scan, gated_scan_backward
    y, last = gated_scan(x, gate, h0, reset=reset, form=form)
    want, tol = forward(x, gate, h0, reset, form)
    assert y.dtype == x.dtype and y.shape == x.shape and last.dtype == torch.float32 and last.shape == x.shape[1:]
    assert ((y.double() - want).abs() <= tol + rounding(want, x.dtype)).all()
    assert ((last.double() - want[-1]).abs() <= tol[-1] + rounding(want[-1], torch.float32)).all()
    dx, dgate, dh0 = gated_scan_backward(dy, x, gate, y, h0, reset=reset, dlast=dlast, form=form)
    wx, tx, wg, tg, w0, t0 = backward(dy, x, gate, y, h0, reset, dlast, form)
    assert ((dx.double() - wx).abs() <= tx + rounding(wx, x.dtype)).all()
    assert ((dgate.double() - wg).abs() <= tg + rounding(wg, x.dtype)).all()
    assert ((dh0.double() - w0).abs() <= t0 + rounding(w0, torch.float32)).all()


SHAPES = [(1, 1, 1), (1, 64, 256), (2, 3, 7), (7, 5, 33), (8, 4, 64), (9, 2, 34), (31, 130, 12), (33, 1, 2), (64, 3, 50),
          (127, 1, 1), (300, 2, 66), (1025, 1, 40), (2000, 3, 5), (63, 700, 520)]


@pytest.mark.parametrize('form', ['average', 'sum'])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_against_the_steps(shape, dtype, form):
    x, gate, h0, reset, dy, dlast = inputs(shape, dtype, form)
    check(x, gate, h0, reset, dy, dlast, form)


@pytest.mark.parametrize('shape', [(5, 3, 8), (700, 2, 20)])
def test_without_state_or_resets(shape):
    x, gate, h0, reset, dy, dlast = inputs(shape, torch.float32)
    check(x, gate, None, None, dy, None, 'average')
    check(x, gate, h0, None, dy, None, 'sum' if shape[0] < 10 else 'average')
    check(x, gate, None, reset, dy, dlast, 'average')
    check(x, gate, h0, torch.ones_like(reset), dy, dlast, 'average')          # every step begins an episode
    check(x, gate, h0, reset.to(torch.uint8) * 7, dy, dlast, 'average')       # any byte but 0 is one


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [12, 24, 33])
def test_strides(dtype, D):
    """Columns of one projection, sequences stored one after the other, more leading dimensions, odd starts."""
    from d1.gated_scan import gated_scan
    x, gate, h0, reset, dy, dlast = inputs((40, 6, D), dtype)
    both = torch.cat((gate, x), 2)
    check(both[..., D:], both[..., :D], h0, reset, dy, dlast, 'average')
    flip = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    check(flip(x), flip(gate), h0, flip(reset), flip(dy), dlast, 'average')
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)
    check(odd(x), odd(gate), h0, reset, odd(dy), dlast, 'average')
    shape = (40, 2, 3, D)
    y, last = gated_scan(x.view(shape), gate.view(shape), h0.view(shape[1:]), reset=reset.view(shape[:-1]))
    want = gated_scan(x, gate, h0, reset=reset)
    assert torch.equal(y.view(x.shape), want[0]) and torch.equal(last.view(h0.shape), want[1])
    wide = x[:, :1].expand(40, 6, D)                                           # one sequence for all
    check(wide, gate, h0, reset[:, :1].expand(40, 6), dy, dlast, 'average')


def test_time_and_channels_alone():
    from d1.gated_scan import gated_scan
    x, gate, h0, reset, _, _ = inputs((50, 1, 10), torch.float32)
    y, last = gated_scan(x[:, 0], gate[:, 0], h0[0], reset=reset[:, 0])
    want = gated_scan(x, gate, h0, reset=reset)
    assert torch.equal(y, want[0][:, 0]) and torch.equal(last, want[1][0])


def test_no_steps_and_no_sequences():
    from d1.gated_scan import gated_scan, gated_scan_backward
    h0 = torch.randn(3, 4, device='cuda')
    x = torch.zeros(0, 3, 4, device='cuda')
    y, last = gated_scan(x, x, h0)
    assert y.shape == x.shape and torch.equal(last, h0)
    assert (gated_scan(x, x)[1] == 0).all()
    dx, dg, dh0 = gated_scan_backward(x, x, x, x, h0, dlast=2 * h0)
    assert dx.shape == x.shape and torch.equal(dh0, 2 * h0) and (gated_scan_backward(x, x, x, x, h0)[2] == 0).all()
    x = torch.zeros(5, 0, 4, device='cuda')
    y, last = gated_scan(x, x)
    assert y.shape == (5, 0, 4) and last.shape == (0, 4)
    assert gated_scan_backward(x, x, x, x)[0].shape == x.shape


def test_steps_one_by_one_are_the_rollout():
    """A decision at a time from the state that the last one left: the same bits as the walk over the rollout
    where one thread has a channel's whole time."""
    from d1.gated_scan import gated_scan
    x, gate, h0, reset, _, _ = inputs((9, 300, 512), torch.bfloat16)
    y, last = gated_scan(x, gate, h0, reset=reset)
    h = h0
    for t in range(9):
        yt, h = gated_scan(x[t:t + 1], gate[t:t + 1], h, reset=reset[t:t + 1])
        assert torch.equal(yt[0], y[t])
    assert torch.equal(h, last)


@pytest.mark.parametrize('T, B, D', [(12, 2, 6), (900, 2, 6)])
def test_a_reset_stops_infinities(T, B, D):
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, _, dy, dlast = inputs((T, B, D), torch.float32)
    cut = T // 2
    reset = torch.zeros(T, B, dtype=torch.bool, device='cuda')
    reset[cut] = True
    x2, dy2 = x.clone(), dy.clone()
    x2[cut - 1, 0], x2[cut - 1, 1, 0], dy2[cut, 0] = float('inf'), float('nan'), float('nan')
    h2 = torch.full_like(h0, float('nan'))
    y, last = gated_scan(x, gate, h0, reset=reset)
    y2, last2 = gated_scan(x2, gate, h2, reset=reset)
    assert torch.equal(y[cut:], y2[cut:]) and torch.equal(last, last2)
    assert y2[cut - 1, 0].isnan().all() or y2[cut - 1, 0].isinf().any()
    g = gated_scan_backward(dy, x, gate, y, h0, reset=reset, dlast=dlast)
    g2 = gated_scan_backward(dy2, x, gate, y, h0, reset=reset, dlast=dlast)
    assert all(torch.equal(p[:cut], q[:cut]) for p, q in zip(g[:2], g2[:2])) and torch.equal(g[2], g2[2])


@pytest.mark.parametrize('dtype', TYPES)
def test_gates_at_their_ends(dtype):
    """Gates of the type's largest magnitudes and infinities: the state is held or replaced, no NaN."""
    from d1.gated_scan import gated_scan
    big = torch.finfo(dtype).max
    gate = torch.tensor([float('inf'), big, -big, float('-inf')], device='cuda', dtype=dtype).view(1, 1, 4).expand(3, 2, 4)
    x, h0 = torch.full((3, 2, 4), 2.0, device='cuda', dtype=dtype), torch.full((2, 4), 5.0, device='cuda')
    y, last = gated_scan(x, gate, h0)
    want = torch.tensor([5.0, 5.0, 2.0, 2.0], device='cuda')
    assert (y.float() == want).all() and (last == want).all()
    y, _ = gated_scan(x, gate.clamp(max=0), h0, form='sum')
    assert (y[0].float() == torch.tensor([7.0, 7.0, 2.0, 2.0], device='cuda')).all()


@pytest.mark.parametrize('form', ['average', 'sum'])
def test_gradient_against_differences(form):
    """Central differences of 2^-7 of sums of about 60 terms of unit size in fp32: the third derivative's term, under
    2^-14 * 5 terms of 1, and roundings of 60 * 2^-22 / 2^-6: 2e-3."""
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, reset, dy, dlast = inputs((5, 2, 3), torch.float32, form, rate=0.2)

    def value(*args):
        y, last = gated_scan(*args, reset=reset, form=form)
        return float((y * dy).double().sum() + (last * dlast).double().sum())
    y, _ = gated_scan(x, gate, h0, reset=reset, form=form)
    grads = gated_scan_backward(dy, x, gate, y, h0, reset=reset, dlast=dlast, form=form)
    args, d = [x, gate, h0], 2.0 ** -7
    for i, g in enumerate(grads):
        for k in range(g.numel()):
            moved = []
            for sign in (1, -1):
                other = [t.clone() for t in args]
                other[i].view(-1)[k] += sign * d
                moved.append(value(*other))
            assert abs((moved[0] - moved[1]) / (2 * d) - float(g.reshape(-1)[k])) < 2e-3 * (1 + abs(float(g.reshape(-1)[k])))


def test_torchs_own_backward():
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, reset, dy, dlast = inputs((20, 3, 8), torch.float32)
    for need in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, gate, h0))]
        y, last = gated_scan(*leaves, reset=reset)
        ((y * dy).sum() + (last * dlast).sum()).backward()
        want = gated_scan_backward(dy, x, gate, y.detach(), h0, reset=reset, dlast=dlast)
        for t, w in zip(leaves, want):
            assert (t.grad is None) == (not t.requires_grad) and (t.grad is None or torch.equal(t.grad, w))
    x = x.clone().requires_grad_()
    gated_scan(x, gate)[1].sum().backward()      # the last state alone, expanded; no first state
    assert torch.equal(x.grad, gated_scan_backward(torch.zeros_like(dy), x.detach(), gate, gated_scan(x.detach(), gate)[0],
                                                   dlast=torch.ones_like(h0))[0])


def test_a_flat_first_state_has_a_flat_gradient():
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, reset, dy, _ = inputs((9, 3, 8), torch.float32)
    leaf = h0.reshape(-1).clone().requires_grad_()
    y, _ = gated_scan(x, gate, leaf, reset=reset)
    (y * dy).sum().backward()
    assert leaf.grad.shape == leaf.shape
    assert torch.equal(leaf.grad.view(h0.shape), gated_scan_backward(dy, x, gate, y.detach(), h0, reset=reset)[2])


def test_graphs_streams_and_the_default_type():
    """Captured calls of two graphs and an eager one on another stream, with new inputs: none disturbs the others."""
    from d1.gated_scan import gated_scan, gated_scan_backward
    a, b = inputs((800, 2, 16), torch.bfloat16, seed=1), inputs((800, 2, 16), torch.bfloat16, seed=2)
    held = [t.clone() for t in a]

    def both(s):
        y, last = gated_scan(s[0], s[1], s[2], reset=s[3])
        return (y, last, *gated_scan_backward(s[4], s[0], s[1], y, s[2], reset=s[3], dlast=s[5]))
    want = [[t.clone() for t in both(s)] for s in (a, b)]
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both(held))
    for t, n in zip(held, b):
        t.copy_(n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        with torch.cuda.stream(side):
            eager = both(a)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want[1]))
    assert all(torch.equal(p, q) for p, q in zip(eager, want[0]))
    torch.set_default_dtype(torch.float64)
    try:
        assert all(torch.equal(p, q) for p, q in zip(both(a), want[0]))
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize('T', [3, 900])
def test_the_state_in_place(T):
    """The C entries with last in place of h0, and dh0 in place of dlast: the same bits."""
    from d1._lib import check as ok, library, stream_of
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, reset, dy, dlast = inputs((T, 2, 48), torch.bfloat16, rate=0.001)
    y, last = gated_scan(x, gate, h0, reset=reset)
    want = gated_scan_backward(dy, x, gate, y, h0, reset=reset, dlast=dlast)
    lib, at = library(), lambda t: t.data_ptr()
    work = torch.empty(max(8, lib.d1_gated_scan_work_bytes(T, 2, 48)), dtype=torch.uint8, device='cuda')
    state, grad, out, dx, dg = h0.clone(), dlast.clone(), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ok(lib.d1_gated_scan(at(x), 96, 48, at(gate), 96, 48, 1, 0, T, 2, 48, at(state), at(reset), 2, 1, at(out), at(state), at(work), stream_of(x)))
    assert torch.equal(out, y) and torch.equal(state, last)
    ok(lib.d1_gated_scan_backward(at(dy), 96, 48, at(x), 96, 48, at(gate), 96, 48, at(y), 96, 48, 1, 0, T, 2, 48, at(h0), at(grad), at(reset), 2, 1,
                                  at(dx), at(dg), at(grad), at(work), stream_of(x)))
    assert torch.equal(dx, want[0]) and torch.equal(dg, want[1]) and torch.equal(grad, want[2])


def test_nan_gates_show():
    from d1.gated_scan import gated_scan
    x, gate, h0, _, _, _ = inputs((40, 2, 16), torch.bfloat16)
    gate[20, 1, 3] = float('nan')
    for form in ('average', 'sum'):
        y, last = gated_scan(x, gate.clamp(max=0) if form == 'sum' else gate, h0, form=form)
        assert y[20:, 1, 3].isnan().all() and last[1, 3].isnan() and int(y.isnan().sum()) == 20


def test_refusals():
    from d1.gated_scan import gated_scan, gated_scan_backward
    x, gate, h0, reset, dy, dlast = inputs((4, 3, 8), torch.float32)
    y, _ = gated_scan(x, gate, h0)
    for bad in (lambda: gated_scan(x, gate[:3]), lambda: gated_scan(x, gate.half()), lambda: gated_scan(x, gate, h0.half()),
                lambda: gated_scan(x, gate, h0[:2]), lambda: gated_scan(x, gate, reset=reset[:, :2]),
                lambda: gated_scan(x, gate, reset=reset.float()), lambda: gated_scan(x, gate, form='mean'),
                lambda: gated_scan(x.transpose(1, 2), gate.transpose(1, 2)), lambda: gated_scan(x.double(), gate.double()),
                lambda: gated_scan(x[0, 0], gate[0, 0]), lambda: gated_scan(x, gate.cpu()), lambda: gated_scan(x[..., :0], gate[..., :0]),
                lambda: gated_scan_backward(dy[:2], x, gate, y), lambda: gated_scan_backward(dy, x, gate, y, dlast=dlast[0]),
                lambda: gated_scan_backward(dy, x, gate, y.half()), lambda: gated_scan_backward(dy, x, gate, y, h0.T)):
        with pytest.raises(ValueError):
            bad()


def test_far_offsets():
    """Steps that lie more than 2^31 elements apart from the first."""
    from d1.gated_scan import gated_scan
    rows, pitch = 5, 2 ** 29 + 4096
    room = torch.empty(4 * pitch + 64, dtype=torch.bfloat16, device='cuda')
    x, gate, h0, reset, _, _ = inputs((rows, 2, 32), torch.bfloat16)
    far = torch.as_strided(room, (rows, 2, 32), (pitch, 32, 1))
    far.copy_(x)
    y, last = gated_scan(far, gate, h0, reset=reset)
    want = gated_scan(x, gate, h0, reset=reset)
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
