"""Which memory the results of the gated recurrence's C entries may share, and strides out of range; checked before any CUDA call, without a
GPU. B = 0 and T = 0 calls that are allowed return before any too."""
import pytest

from test_gated_scan_host import BAD, P, backward, forward, lib  # noqa: F401

FAR = dict(x=P, gate=2 * P, h0=5 * P, reset=6 * P, last=7 * P, y=4 * P)
BACK = dict(dy=P, x=2 * P, gate=3 * P, y=4 * P, h0=5 * P, dlast=6 * P, reset=7 * P, rt=2, rb=1, dx=8 * P, dgate=9 * P, dh0=10 * P)


def test_forward(lib):  # noqa: F811
    call = lambda **k: lib.d1_gated_scan(*forward(**dict(FAR, **k)))
    # y is 3 * 2 * 8 elements of 2 bytes, h0 and last 2 * 8 of 4, the resets' last byte is 2 * 2 + 1 on
    for at in (P, 2 * P, 5 * P, 6 * P, 7 * P):
        assert call(y=at) == BAD and call(y=at - 94) == BAD, at
    for at in (5 * P + 62, 6 * P + 4, 7 * P + 62):
        assert call(y=at) == BAD, at
    for at in (P, 2 * P, 6 * P, P + 76, 6 * P - 60, 5 * P + 4, 5 * P - 60):
        assert call(last=at) == BAD, at
    # T = 0: nothing of x, gate, y; last is h0 or apart from it
    assert call(T=0, last=5 * P, h0=5 * P) == 0 and call(T=0, last=5 * P + 4) == BAD


def test_backward(lib):  # noqa: F811
    call = lambda **k: lib.d1_gated_scan_backward(*backward(**dict(BACK, **k)))
    for k in ('dx', 'dgate'):    # fp32: 192 bytes
        for at in [i * P for i in range(1, 11) if i * P != BACK[k]] + [5 * P + 60, 6 * P + 60, 7 * P + 4, 10 * P + 60, 5 * P - 188]:
            assert call(**{k: at}) == BAD, (k, at)
    for at in [i * P for i in (1, 2, 3, 4, 5, 7, 8, 9)] + [5 * P + 60, 6 * P + 4, 6 * P - 4, 8 * P + 188]:
        assert call(dh0=at) == BAD, at
    assert call(T=0, dh0=6 * P) == 0 and call(T=0, dh0=6 * P + 4) == BAD


def test_strides(lib):  # noqa: F811
    """(T - 1) * stride past 64 bits is refused, not wrapped around; one step or sequence has none."""
    T = 1 << 39
    for k in ('xt', 'gt', 'rt'):
        for s in ((1 << 42), (1 << 25) + (1 << 20), (1 << 62)):
            assert lib.d1_gated_scan(*forward(**dict(FAR, T=T, B=1, D=1, y=1 << 50, work=8 * P, **{k: s}))) == BAD, (k, s)
    for k in ('dt', 'xt', 'gt', 'yt', 'rt'):
        assert lib.d1_gated_scan_backward(*backward(**dict(BACK, T=T, B=1, D=1, dx=1 << 50, dgate=1 << 52, work=11 * P, **{k: 1 << 42}))) == BAD, k
    for k in ('xb', 'gb', 'rb'):
        assert lib.d1_gated_scan(*forward(**dict(FAR, T=1, B=T, D=1, y=1 << 50, **{k: 1 << 42}))) == BAD, k


def test_strides_of_one_step(lib):  # noqa: F811
    """Where there is one step or sequence its stride is not used, but one past 59 bits is refused all the same."""
    for k in ('xt', 'gt', 'rt'):
        assert lib.d1_gated_scan(*forward(**dict(FAR, T=1, **{k: 1 << 62}))) == BAD, k
    for k in ('xb', 'gb', 'rb'):
        assert lib.d1_gated_scan(*forward(**dict(FAR, B=1, **{k: 1 << 62}))) == BAD, k
