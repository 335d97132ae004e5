"""What the row operators (layer norm, token log-probabilities) ask of their tensors."""
import torch

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # D1_TYPE_* of d1.h


def type_of(t, name):
    code = TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f'{name} must be float32, bfloat16 or float16, not {t.dtype}')
    return code


def matrix(t, name):
    """t as [rows, n] with one row pitch and contiguous rows (a view: nothing is copied)."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f'{name} needs at least one dimension')
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(-1, t.shape[-1])
        except RuntimeError:
            raise ValueError(f'{name}: the leading dimensions of shape {tuple(t.shape)} with strides {t.stride()} '
                             'have no single row pitch') from None
    if t.shape[1] < 1:
        raise ValueError(f'{name}: rows are empty')
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')
    return t


def vector(t, count, dtype, device, name):
    """A contiguous tensor of `count` elements, or None; its address."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != count or t.device != device or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous {dtype} tensor of {count} elements on {device}, not '
                         f'{t.dtype} {tuple(t.shape)} on {t.device}')
    return t.data_ptr()


def like(t, of, name):
    """An output (or second input) of the shape, type and device of `of`, as a matrix."""
    if t.shape != of.shape or t.dtype != of.dtype or t.device != of.device:
        raise ValueError(f'{name} must be {of.dtype} {tuple(of.shape)} on {of.device}, not {t.dtype} '
                         f'{tuple(t.shape)} on {t.device}')
    return matrix(t, name)


_F32 = {}


def empty_f32(device, *shape):
    """torch.empty of float32 on `device`, by the cheapest route: new_empty of a kept
    tensor, with the sizes as numbers (half the cost of torch.empty with a shape)."""
    kept = _F32.get(device)
    if kept is None:
        kept = _F32[device] = torch.empty(0, device=device)
    return kept.new_empty(*shape) if shape else kept.new_empty(())


def empty_like(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def on_gpu(t, name):
    if not t.is_cuda:
        raise ValueError(f'{name} must be on a CUDA device (there is no CPU path)')
    return t.device


def apart(a, b, name, other):
    """Refuses two matrices whose spans of memory overlap."""
    ends = []
    for t in (a, b):
        span = ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() if t.shape[0] else 0
        ends.append((t.data_ptr(), t.data_ptr() + span))
    if ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]:
        raise ValueError(f'{name} overlaps {other}')
