"""Layer norm's output over its input, beside it, and the overlaps that are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('n', [24, 513, 1111, 1536])
def test_out_is_x_or_apart_from_it(n):
    from d1.layer_norm import layer_norm
    buf = torch.randn(71, 2 * n, device='cuda').bfloat16()
    x, beside = buf[:, :n], buf[:, n:]
    want = layer_norm(x)
    got = layer_norm(x, out=beside)
    assert got[0].data_ptr() == beside.data_ptr() and torch.equal(got[1], want[1])
    assert ((got[0] - want[0]).abs() <= 2.0 ** -7 * (1 + want[0].abs())).all()   # one rounding to bf16 on either side
    dense = buf[:, :n].clone()
    for bad in (dense[1:], dense.view(-1)[n:], dense[:-1]):
        rows = dense[:-1] if bad.data_ptr() != dense.data_ptr() else dense[1:]
        with pytest.raises(ValueError):
            layer_norm(rows, out=bad.view(-1, n))
    with pytest.raises(ValueError):
        layer_norm(x, out=buf[:, 1:n + 1])
    with pytest.raises(ValueError):
        layer_norm(x[:10], out=torch.as_strided(buf, (10, n), (4 * n, 1)))
    want = layer_norm(dense)
    got = layer_norm(dense, out=dense)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
