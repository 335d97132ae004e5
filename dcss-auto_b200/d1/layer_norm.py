"""Layer norm over the last dimension and its gradients (d1_layer_norm).

    y, mean, rstd = layer_norm(x, weight, bias)
    dx, dweight, dbias = layer_norm_backward(dy, x, mean, rstd, weight)

x is float32, bfloat16 or float16 of any shape whose leading dimensions have
one row pitch (a slice of columns will do); weight and bias are float32, as the
policies' masters are, or None. Sums are held in 32 bits, y and dx are rounded
once. The calls launch on the current stream of x's device and can be captured
in a CUDA graph.
"""
import torch

from ._lib import check, library, stream_of
from ._rows import apart, empty_f32, empty_like, like, matrix, on_gpu, type_of, vector


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """(y, mean, rstd): y as x (or written to `out`, which may be x), mean and
    rstd float32 of x's leading shape, which the backward pass takes."""
    dev, kind, m = on_gpu(x, 'x'), type_of(x, 'x'), matrix(x, 'x')
    rows, n = m.shape
    if not eps >= 0:
        raise ValueError('eps must not be negative')
    w, b = vector(weight, n, torch.float32, dev, 'weight'), vector(bias, n, torch.float32, dev, 'bias')
    if out is None:
        y = out = empty_like(x)
        ldy = n
    else:
        y = like(out, x, 'out')
        ldy = y.stride(0)
    lead = rows if x.dim() == 2 else x.shape[:-1]
    mean, rstd = empty_f32(dev, lead), empty_f32(dev, lead)
    check(library().d1_layer_norm(m.data_ptr(), m.stride(0), kind, rows, n, w, b, eps, y.data_ptr(), ldy,
                                  mean.data_ptr(), rstd.data_ptr(), stream_of(x)), 'd1_layer_norm')
    return out, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, out=None):
    """(dx, dweight, dbias) of layer_norm from dy (x's shape and type). dx is
    written to `out` when given, which overlaps no input; dweight and dbias are
    float32 [n]. The sums over the rows are taken in a fixed order."""
    dev, kind, m = on_gpu(x, 'x'), type_of(x, 'x'), matrix(x, 'x')
    rows, n = m.shape
    d = like(dy, x, 'dy')
    w = vector(weight, n, torch.float32, dev, 'weight')
    mu, rs = vector(mean, rows, torch.float32, dev, 'mean'), vector(rstd, rows, torch.float32, dev, 'rstd')
    if out is None:
        dx = out = empty_like(x)
        lddx = n
    else:
        dx = like(out, x, 'out')
        lddx = dx.stride(0)
        apart(dx, m, 'out', 'x')
        apart(dx, d, 'out', 'dy')
    lib = library()
    dweight, dbias = empty_f32(dev, n), empty_f32(dev, n)
    work = empty_f32(dev, lib.d1_layer_norm_parts(rows, n) * 2 * n)
    check(lib.d1_layer_norm_backward(d.data_ptr(), d.stride(0), m.data_ptr(), m.stride(0), kind, rows, n, w, mu, rs,
                                     dx.data_ptr(), lddx, dweight.data_ptr(), dbias.data_ptr(), work.data_ptr(),
                                     stream_of(x)), 'd1_layer_norm_backward')
    return out, dweight, dbias
