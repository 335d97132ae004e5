"""Layer norm's weight gradients, tightly: every row counts once, whichever block, team
and part it falls to.

dbias of small whole numbers is exact. dweight has the error of its additions, rows /
parts of them in turn and at most 100 in the joins, of 2^-24 of the sum of magnitudes;
its terms are given xhat to a few roundings (3 2^-24 of |xhat| + |x rstd|).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows, n', [(1, 64), (7, 513), (20011, 48), (5003, 64), (5003, 65), (3001, 130), (3001, 256), (2003, 300),
                                     (2003, 512), (1501, 783), (1501, 1024), (901, 2050), (901, 4096), (300, 8200), (300, 12033),
                                     (90, 16384), (70, 20000), (149, 9000)])
def test_every_row_once(rows, n, dtype):
    from d1._lib import library
    from d1.layer_norm import layer_norm, layer_norm_backward
    g = torch.Generator(device='cuda').manual_seed(rows + n)
    x = (torch.randn(rows, n, device='cuda', generator=g) + 0.5).to(dtype)
    dy = torch.randint(-3, 4, (rows, n), device='cuda', generator=g).to(dtype)
    _, mean, rstd = layer_norm(x)
    _, dweight, dbias = layer_norm_backward(dy, x, mean, rstd)
    assert torch.equal(dbias.double(), dy.double().sum(0))
    mu, rs = mean.double()[:, None], rstd.double()[:, None]
    xhat = (x.double() - mu) * rs
    parts = max(1, min(rows, library().d1_layer_norm_parts(rows, n)))
    if n > 8192:                       # the plain passes have 16 at most
        parts = min(parts, 16)
    err = 3 * U * (xhat.abs() + (x.double() * rs).abs())
    tol = (rows / parts + 100) * U * (dy.double() * xhat).abs().sum(0) + (dy.double().abs() * err).sum(0)
    assert ((dweight.double() - (dy.double() * xhat).sum(0)).abs() <= tol + 1e-30).all()
    last = torch.zeros_like(dy)
    for r in {0, rows // 2, rows - 1}:  # one row alone
        last.zero_()
        last[r] = 1
        _, dweight, dbias = layer_norm_backward(last, x, mean, rstd)
        assert (dbias == 1).all()
        assert ((dweight.double() - xhat[r]).abs() <= err[r] + 2 * U * xhat[r].abs()).all()
