"""The C entries of the gated recurrence refuse bad arguments before any CUDA call (checked without a
GPU), and the Python calls refuse tensors that are not on one."""
import pytest
import torch

BAD = 9002
P = 1 << 20  # an aligned address that is never read


@pytest.fixture(scope='module')
def lib():
    from d1 import _lib
    return _lib.library()


def forward(**change):
    good = dict(x=P, xt=16, xb=8, gate=2 * P, gt=16, gb=8, type=1, form=0, T=3, B=2, D=8, h0=P, reset=P, rt=2, rb=1, y=4 * P, last=P,
                work=None, s=None)
    return dict(good, **change).values()


def backward(**change):
    good = dict(dy=P, dt=16, db=8, x=P, xt=16, xb=8, gate=2 * P, gt=16, gb=8, y=3 * P, yt=16, yb=8, type=0, form=1, T=3, B=2, D=8, h0=P,
                dlast=P, reset=None, rt=0, rb=0, dx=4 * P, dgate=5 * P, dh0=P, work=None, s=None)
    return dict(good, **change).values()


def test_forward(lib):
    for k, v in dict(x=None, gate=None, y=None, type=3, form=2, T=-1, B=-1, D=0, xt=-1, xb=-8, gt=-1, gb=-1, rt=-1, rb=-1, h0=P + 2,
                     last=P + 1).items():
        assert lib.d1_gated_scan(*forward(**{k: v})) == BAD, k
    for k in ('x', 'gate', 'y'):
        assert lib.d1_gated_scan(*forward(**{k: 6 * P + 1})) == BAD, k
    for y in (P, P + 30, 2 * P, P - 2 * 3 * 16 + 2):           # the range of x or of gate
        assert lib.d1_gated_scan(*forward(y=y)) == BAD, y
    assert lib.d1_gated_scan(*forward(T=1 << 41)) == BAD and lib.d1_gated_scan(*forward(B=1 << 41)) == BAD
    assert lib.d1_gated_scan(*forward(T=1000, y=64 * P)) == BAD     # needs its work buffer
    assert lib.d1_gated_scan(*forward(T=1000, y=64 * P, work=P + 4)) == BAD
    assert lib.d1_gated_scan(*forward(B=0)) == 0
    assert lib.d1_gated_scan(*forward(T=0, x=None, gate=None, y=None, last=None)) == 0


def test_backward(lib):
    for k, v in dict(dy=None, x=None, gate=None, y=None, dx=None, dgate=None, type=-1, form=-1, T=-1, D=0, dt=-1, db=-1, yt=-1, yb=-1,
                     dh0=P + 2, dlast=P + 2).items():
        assert lib.d1_gated_scan_backward(*backward(**{k: v})) == BAD, k
    for k in ('dx', 'dgate'):
        for at in (P, 2 * P, 3 * P + 4 * 47, 4 * P + 4, 5 * P + 4):   # an input's range, or the other gradient's
            if at // P != {'dx': 4, 'dgate': 5}[k]:
                assert lib.d1_gated_scan_backward(*backward(**{k: at})) == BAD, (k, at)
    assert lib.d1_gated_scan_backward(*backward(T=0, dh0=None)) == 0


def test_work_bytes(lib):
    size = lib.d1_gated_scan_work_bytes
    assert size(-1, 1, 1) == size(1, -1, 1) == size(1, 1, 0) == size(1 << 41, 1, 1) == -1
    assert size(0, 0, 1) == size(1, 64, 256) == size(128, 4096, 512) == 0
    assert 0 < size(131072, 1, 256) <= 1 << 24
    for T in (1, 31, 32, 33, 1000, 10 ** 7):
        for C in (1, 7, 512, 10 ** 5):
            assert size(T, 1, C) == size(T, C, 1) and size(T, 1, C) % (8 * C) == 0


def test_host_tensors_are_refused():
    from d1.gated_scan import gated_scan, gated_scan_backward
    x = torch.zeros(4, 2, 8)
    with pytest.raises(ValueError):
        gated_scan(x, x)
    with pytest.raises(ValueError):
        gated_scan_backward(x, x, x, x)


def test_pitches():
    from d1.gated_scan import _pitch, _steps
    t = torch.zeros(5, 4, 3, 8)
    assert _steps(t, 'x')[1:] == (96, 8) and _steps(t[:, :, :, 2:], 'x')[1:] == (96, 8)
    assert _steps(t[:, :1], 'x')[1:] == (96, 8) and _steps(t[:, :, :1], 'x')[1:] == (96, 24)
    assert _steps(t[:, 0, 0], 'x')[1:] == (96, 0) and _pitch((), (), 'x') == 0
    assert _steps(torch.zeros(4, 5, 8).transpose(0, 1), 'x')[1:] == (8, 40)
    assert _steps(torch.zeros(5, 1, 1, 8).expand(5, 4, 3, 8), 'x')[1:] == (8, 0)
    with pytest.raises(ValueError):
        _steps(t[:, :, :2], 'x')
    with pytest.raises(ValueError):
        _steps(torch.zeros(8), 'x')
