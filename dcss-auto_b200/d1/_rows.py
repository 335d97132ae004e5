"""What the row operators (layer norm, token log-probabilities) ask of their tensors.

They are called on batches of a few microseconds of GPU work, so that the checks
are written for few Python and torch calls."""
import torch

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # D1_TYPE_* of d1.h
MAX_COLUMNS = 2 ** 31 - 1


def recorded(x, weight=None, bias=None):
    """Whether torch records gradients of one of them."""
    return torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                        (bias is not None and bias.requires_grad))


def type_of(t, name):
    """D1_TYPE_* of a tensor on a GPU."""
    code = TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f'{name} must be float32, bfloat16 or float16, not {t.dtype}')
    if not t.is_cuda:
        raise ValueError(f'{name} must be on a CUDA device (there is no CPU path)')
    return code


def matrix(t, name):
    """(address, rows, n, row pitch) of t as [rows, n] with contiguous rows; nothing is copied."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f'{name} needs at least one dimension')
        if t.shape[-1] == 0:
            raise ValueError(f'{name}: rows are empty')
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(-1, t.shape[-1])
        except RuntimeError:
            raise ValueError(f'{name}: the leading dimensions of shape {tuple(t.shape)} with strides {t.stride()} '
                             'have no single row pitch') from None
    rows, n = t.shape
    pitch, step = t.stride()
    if n < 1:
        raise ValueError(f'{name}: rows are empty')
    if n > MAX_COLUMNS:  # the C entries take it as an int, and ctypes would cut it off without a word
        raise ValueError(f'{name}: rows of {n} elements are longer than {MAX_COLUMNS}')
    if step != 1 and n > 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')
    return t.data_ptr(), rows, n, pitch


def vector(t, count, dtype, device, name):
    """The address of a contiguous tensor of `count` elements, or None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != count or t.device != device or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous {dtype} tensor of {count} elements on {device}, not '
                         f'{t.dtype} {tuple(t.shape)} on {t.device}')
    return t.data_ptr()


def like(t, of, name):
    """An output (or second input) of the shape, type and device of `of`, as a matrix."""
    if t.shape != of.shape or t.dtype is not of.dtype or t.device != of.device:
        raise ValueError(f'{name} must be {of.dtype} {tuple(of.shape)} on {of.device}, not {t.dtype} '
                         f'{tuple(t.shape)} on {t.device}')
    return matrix(t, name)


_F32 = {}


def empty_f32(device, *shape):
    """torch.empty of float32 on `device`, by the cheapest route: new_empty of a kept
    tensor, with the sizes as numbers (half the cost of torch.empty with a shape).
    The type is named: the kernels write 4 bytes an element whatever torch's default is."""
    kept = _F32.get(device)
    if kept is None:
        kept = _F32[device] = torch.empty(0, dtype=torch.float32, device=device)
    return kept.new_empty(*shape) if shape else kept.new_empty(())


def empty_like(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def rows_meet(p, rows, width, pitch, q, rows_q, width_q, pitch_q):
    """Whether `rows` rows of `width` bytes from p on, `pitch` apart, share a byte with
    those from q on. Exact: column slices of one buffer lie between one another."""
    if not pitch:
        rows = min(rows, 1)
    if not pitch_q:
        rows_q = min(rows_q, 1)
    if not (rows and rows_q and p < q + (rows_q - 1) * pitch_q + width_q and q < p + (rows - 1) * pitch + width):
        return False
    if rows == 1:
        pitch = pitch_q
    if rows_q == 1:
        pitch_q = pitch
    if rows == rows_q == 1:
        return True
    if pitch != pitch_q:  # row by row of the one that has fewer
        if rows <= rows_q:
            return any(rows_meet(p + i * pitch, 1, width, 0, q, rows_q, width_q, pitch_q) for i in range(rows))
        return any(rows_meet(p, rows, width, pitch, q + i * pitch_q, 1, width_q, 0) for i in range(rows_q))
    # rows i and j meet where q - p - width < k pitch < q - p + width_q with k = i - j
    k = max((q - p - width) // pitch + 1, 1 - rows_q)
    return k < rows and k * pitch < q - p + width_q


def apart(a, b, size, name, other):
    """Refuses two matrices of elements of `size` bytes that share memory."""
    (p, rows, n, pitch), (q, rows_q, n_q, step) = a, b
    if rows_meet(p, rows, n * size, pitch * size, q, rows_q, n_q * size, step * size):
        raise ValueError(f'{name} overlaps {other}')
