"""Layer norm over the last dimension and its gradients (d1_layer_norm).

    y, mean, rstd = layer_norm(x, weight, bias)
    dx, dweight, dbias = layer_norm_backward(dy, x, mean, rstd, weight)

x is float32, bfloat16 or float16 of any shape whose leading dimensions have
one row pitch (a slice of columns will do); weight and bias are float32, as the
policies' masters are, or None. Sums are held in 32 bits, y and dx are rounded
once. The calls launch on the current stream of x's device and can be captured
in a CUDA graph. Where torch records gradients of x, weight or bias, y has its
(first) gradient; mean and rstd have none.
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import check, library, stream_of
from ._rows import apart, empty_f32, empty_like, like, matrix, recorded, type_of, vector

F32 = torch.float32


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.mark_non_differentiable(mean, rstd)
        ctx.shapes = [None if t is None else t.shape for t in (weight, bias)]
        return y, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dmean, drstd):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, *sums = layer_norm_backward(dy.contiguous(), x, mean, rstd, weight)
        need = ctx.needs_input_grad
        return (dx if need[0] else None, *(g.view(shape) if n else None for g, shape, n in zip(sums, ctx.shapes, need[1:3])), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """(y, mean, rstd): y as x (or written to `out`, which may be x but shares no
    memory with it otherwise), mean and rstd float32 of x's leading shape, which
    the backward pass takes."""
    if recorded(x, weight, bias):
        if out is not None:
            raise ValueError('out has no gradient: call under torch.no_grad(), or without out')
        return _LayerNorm.apply(x, weight, bias, eps)
    return _layer_norm(x, weight, bias, eps, out)


def _layer_norm(x, weight, bias, eps, out=None):
    kind, dev = type_of(x, 'x'), x.device
    px, rows, n, ldx = mx = matrix(x, 'x')
    if not eps >= 0:
        raise ValueError('eps must not be negative')
    w, b = vector(weight, n, F32, dev, 'weight'), vector(bias, n, F32, dev, 'bias')
    if out is None:
        out = empty_like(x)
        py, ldy = out.data_ptr(), n
    else:
        py, _, _, ldy = mo = like(out, x, 'out')
        if py != px or (ldy != ldx and rows > 1):
            apart(mo, mx, x.element_size(), 'out', 'x')
    lead = rows if x.dim() == 2 else x.shape[:-1]
    mean, rstd = empty_f32(dev, lead), empty_f32(dev, lead)
    check(library().d1_layer_norm(px, ldx, kind, rows, n, w, b, eps, py, ldy, mean.data_ptr(), rstd.data_ptr(),
                                  stream_of(x)), 'd1_layer_norm')
    return out, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, out=None):
    """(dx, dweight, dbias) of layer_norm from dy (x's shape and type). dx is
    written to `out` when given, which overlaps no input; dweight and dbias are
    float32 [n]. The sums over the rows are taken in a fixed order."""
    kind, dev = type_of(x, 'x'), x.device
    px, rows, n, ldx = mx = matrix(x, 'x')
    pd, _, _, ldd = md = like(dy, x, 'dy')
    w = vector(weight, n, F32, dev, 'weight')
    mu, rs = vector(mean, rows, F32, dev, 'mean'), vector(rstd, rows, F32, dev, 'rstd')
    if out is None:
        out = empty_like(x)
        po, ldo = out.data_ptr(), n
    else:
        po, _, _, ldo = mo = like(out, x, 'out')
        apart(mo, mx, x.element_size(), 'out', 'x')
        apart(mo, md, x.element_size(), 'out', 'dy')
    lib = library()
    dweight, dbias = empty_f32(dev, n), empty_f32(dev, n)
    work = empty_f32(dev, lib.d1_layer_norm_parts(rows, n) * 2 * n)
    check(lib.d1_layer_norm_backward(pd, ldd, px, ldx, kind, rows, n, w, mu, rs, po, ldo, dweight.data_ptr(),
                                     dbias.data_ptr(), work.data_ptr(), stream_of(x)), 'd1_layer_norm_backward')
    return out, dweight, dbias
