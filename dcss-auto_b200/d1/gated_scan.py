"""A gated linear recurrence over time (the memory of a policy) and its gradients (d1_gated_scan).

    y, last = gated_scan(x, gate, h0, reset=reset)            # a rollout: x, gate [T, B, D]
    y, h = gated_scan(x[None], gate[None], h)                 # one decision: T = 1
    dx, dgate, dh0 = gated_scan_backward(dy, x, gate, y, h0, reset=reset, dlast=dlast)

Each of the D channels of each of the B sequences has a state of its own:

    form 'average':  a = sigmoid(gate)   h_t = a_t h_{t-1} + (1 - a_t) x_t
    form 'sum':      a = exp(gate)       h_t = a_t h_{t-1} + x_t     (a is float32: infinite for gates above 88.7)

x and gate are float32, bfloat16 or float16 [T, ..., D], time first as the
rollouts are, with contiguous channels and one pitch between sequences (a slice
of a projection's columns will do, and so will x.transpose(0, 1) of sequences
stored one after the other). reset (bool or uint8 [T, ...]) marks the steps at
which an episode begins: the state before them counts for nothing, so that
sequences packed behind one another are resets too. h0 and last are the float32
states [..., D] before and after. States and their gradients are held in 32
bits; y, dx and dgate are rounded once to x's type. The gradient reads the
states as y has them.

The calls launch on the current stream of x's device, allocate through torch and
can be captured in a CUDA graph. Where torch records gradients of x, gate or h0, y
and last lead back to them (first derivatives).
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import check, library, stream_of
from ._rows import empty_f32, empty_like, type_of, vector

F32 = torch.float32
FORMS = {'average': 0, 'sum': 1}  # D1_SCAN_* of d1.h
_FLAGS = (torch.bool, torch.uint8)


def _steps(t, name):
    """(address, step pitch, sequence pitch) of t as [T, B, D] with contiguous channels; nothing is copied."""
    strides = t.stride()
    if len(strides) == 3:
        st, sb, sd = strides
        if sd != 1 and t.shape[2] > 1:
            raise ValueError(f'{name}: the last dimension must be contiguous')
        return t.data_ptr(), st, sb
    if t.dim() < 2:
        raise ValueError(f'{name} needs a time and a channel dimension, not {tuple(t.shape)}')
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')
    return t.data_ptr(), t.stride(0), _pitch(t.shape[1:-1], t.stride()[1:-1], name)


def _pitch(shape, strides, name):
    """The one pitch between the sequences of these leading dimensions."""
    pitch, count = 0, 1
    for n, s in zip(reversed(shape), reversed(strides)):
        if n == 1:
            continue
        if count == 1:
            pitch = s
        elif s != pitch * count:
            raise ValueError(f'{name}: sequences of shape {tuple(shape)} with strides {tuple(strides)} have no single pitch')
        count *= n
    return pitch


def _flags(reset, shape, dev):
    """(address, step pitch, sequence pitch) of the resets."""
    if reset is None:
        return None, 0, 0
    flags = shape[:-1]
    if reset.dtype not in _FLAGS or reset.shape != flags or reset.device != dev:
        raise ValueError(f'reset must be a bool or uint8 tensor {tuple(flags)} on {dev}, not '
                         f'{reset.dtype} {tuple(reset.shape)} on {reset.device}')
    if len(flags) == 2:
        return reset.data_ptr(), *reset.stride()
    return reset.data_ptr(), reset.stride(0), _pitch(flags[1:], reset.stride()[1:], 'reset')


def _same(t, shape, dtype, dev, name):
    if t.shape != shape or t.dtype is not dtype or t.device != dev:
        raise ValueError(f'{name} must be {dtype} {tuple(shape)} on {dev}, not {t.dtype} {tuple(t.shape)} on {t.device}')
    return _steps(t, name)


def _sizes(x, form):
    """(type, form, x's address and pitches, (T, B, D), (shape, dtype, device))."""
    kind, code = type_of(x, 'x'), FORMS.get(form)
    if code is None:
        raise ValueError(f"form must be 'average' or 'sum', not {form!r}")
    ax, shape = _steps(x, 'x'), x.shape
    D = shape[-1]
    if D < 1 or D > 2 ** 31 - 1:
        raise ValueError(f'x has {D} channels')
    sizes = tuple(shape) if len(shape) == 3 else (shape[0], shape[1:-1].numel(), D)
    return kind, code, ax, sizes, (shape, x.dtype, x.device)


def _work(sizes, device):
    T, B, D = sizes
    if T <= 32:  # not cut into chunks
        return None
    size = library().d1_gated_scan_work_bytes(T, B, D)
    if size < 0:
        raise ValueError(f'{T} steps of {B} sequences of {D} channels are out of range')
    return empty_f32(device, size // 4) if size else None


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, reset, form):
        y, last = _gated_scan(x, gate, h0, reset, form)
        ctx.save_for_backward(x, gate, y, h0, reset)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return (None,) * 5
        x, gate, y, h0, reset = ctx.saved_tensors
        dy = torch.zeros_like(y) if dy is None else dy.contiguous()
        dx, dgate, dh0 = gated_scan_backward(dy, x, gate, y, h0, reset, None if dlast is None else dlast.contiguous(), ctx.form)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dgate if need[1] else None, dh0.view(h0.shape) if need[2] else None, None, None


def gated_scan(x, gate, h0=None, reset=None, form='average'):
    """(y, last): the states of every step in x's type, and the last one in float32."""
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, h0, reset, form)
    return _gated_scan(x, gate, h0, reset, form)


def _gated_scan(x, gate, h0, reset, form):
    kind, code, ax, sizes, as_x = _sizes(x, form)
    shape, _, dev = as_x
    ag, start, flags = _same(gate, *as_x, 'gate'), vector(h0, sizes[1] * sizes[2], F32, dev, 'h0'), _flags(reset, shape, dev)
    y = empty_like(x)
    last = torch.empty_like(h0) if h0 is not None and h0.shape == shape[1:] else empty_f32(dev, *shape[1:])
    work = _work(sizes, dev)
    check(library().d1_gated_scan(*ax, *ag, kind, code, *sizes, start, *flags, y.data_ptr(), last.data_ptr(),
                                  None if work is None else work.data_ptr(), stream_of(x)), 'd1_gated_scan')
    return y, last


def gated_scan_backward(dy, x, gate, y, h0=None, reset=None, dlast=None, form='average'):
    """(dx, dgate, dh0) of gated_scan from the gradients of y (x's shape and type) and of
    last (float32, None: zeros). h0, reset and form are the forward pass's."""
    kind, code, ax, sizes, as_x = _sizes(x, form)
    shape, _, dev = as_x
    ag, ay, ad = _same(gate, *as_x, 'gate'), _same(y, *as_x, 'y'), _same(dy, *as_x, 'dy')
    first, end = vector(h0, sizes[1] * sizes[2], F32, dev, 'h0'), vector(dlast, sizes[1] * sizes[2], F32, dev, 'dlast')
    flags = _flags(reset, shape, dev)
    dx, dgate, dh0 = empty_like(x), empty_like(x), empty_f32(dev, *shape[1:])
    work = _work(sizes, dev)
    check(library().d1_gated_scan_backward(*ad, *ax, *ag, *ay, kind, code, *sizes, first, end, *flags, dx.data_ptr(),
                                           dgate.data_ptr(), dh0.data_ptr(), None if work is None else work.data_ptr(),
                                           stream_of(x)), 'd1_gated_scan_backward')
    return dx, dgate, dh0
