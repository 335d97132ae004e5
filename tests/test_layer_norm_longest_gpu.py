"""Layer norm of a row whose two column sums together pass 31 bits.

The row alternates between 1 and -1 and dy is 1, so that the mean, db and the sums of
g and g xhat are exact: a thread sees one sign, and as many threads see the other. The
sum of squares, 2^30 and some, is rounded: 2^-23 of rstd.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_row_of_a_billion_columns():
    from d1.layer_norm import layer_norm, layer_norm_backward
    n = 2 ** 30 + 40
    x = torch.ones(1, n, device='cuda', dtype=torch.float16)
    x[0, 1::2] = -1
    y, mean, rstd = layer_norm(x)
    assert float(mean) == 0 and abs(float(rstd) * (1 + 1e-5) ** 0.5 - 1) <= 2.0 ** -21
    assert torch.equal(y, x)                                   # rstd is 1 to half a unit of fp16
    del y
    dy = torch.ones_like(x)
    dx, dweight, dbias = layer_norm_backward(dy, x, mean, rstd)
    assert float(dbias.min()) == 1 and float(dbias.max()) == 1
    for part in (slice(0, 10 ** 6), slice(n // 2, n // 2 + 10 ** 6), slice(n - 10 ** 6, n)):
        assert torch.equal(dweight[part], x[0, part].float() * rstd)
        assert (dx[0, part].abs() <= 1e-6).all()
