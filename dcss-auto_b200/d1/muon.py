"""Muon over many weight matrices (d1_muon), and its orthogonalisation by itself (d1_orthogonalize).

    opt = Muon(params, grads, lr=3e-4, momentum=0.95, weight_decay=0.01, copies=bf16_copies)
    opt.step()                       # reads grads, updates params, momentum and bf16 copies in place
    y = orthogonalize(x)             # x [..., m, n]: the same directions, singular values near 1

    m = momentum m + grad       u = grad + momentum m (nesterov) or m
    X = u / |u|_F, then `steps` times X = 3.4445 X - 4.7750 (X X^T) X + 2.0315 (X X^T)^2 X
    p = p (1 - lr decay) - lr 0.2 sqrt(max(rows, cols)) X

With that factor an update is as large as AdamW's at the same rate (0.2 of lr an element), so
that one rate serves both: the matrices' here, vectors' and embeddings' in d1.adamw.
params are contiguous float32 tensors (masters) of two or more dimensions, [..., rows,
cols]: leading dimensions are a stack of matrices. grads are float32 or bfloat16 of the same
shapes; each step reads whatever they then hold. copies (bfloat16, or None for a tensor that
has none) are refreshed by the step. weight_decay and copies may differ by tensor. No
parameter or copy shares memory with another one or with a gradient, and each keeps
its storage for the optimizer's life (the step has their addresses).

The products are fp16 with fp32 sums and X is held to 22 bits between them, so that a
gradient of low rank comes out as exact as one of full rank (in five steps to 3e-3 of the result's norm; matrices with a
side of at most 64 to 2e-4). precise=True takes products as good as fp32 ones, up to three times their time: X to 2e-4 for
any size. Each further step makes the directions that a gradient does not have 3.4 times as large: from some twelve on a gradient of low
rank has them too, as in any arithmetic of 32 bits. The momentum is float32, flat over the tensors, each starting at a multiple of 128 elements
(`offsets`); momentum_of(i) gives a tensor's in its shape. A step may be captured in a CUDA graph.
Steps of one optimizer share its work buffer: run them on one stream, or ordered. A step that failed is seen by the next
one, which raises, or by check().
"""
import ctypes as C

import torch

from ._lib import D1Error, check, library, stream_of
from ._rows import type_of
from .adamw import GRAD_TYPES, _outside, _spans
from .gated_scan import _pitch

F32, BF16 = torch.float32, torch.bfloat16
MAX_STEPS = 64


class _Tensor(C.Structure):
    _fields_ = [('param', C.c_void_p), ('grad', C.c_void_p), ('copy', C.c_void_p), ('count', C.c_int64), ('rows', C.c_int64),
                ('cols', C.c_int64), ('decay', C.c_double), ('grad_type', C.c_int), ('precise', C.c_int)]


_told = None   # a pinned int that a failed call sets, looked at before the next one


def _watch():
    """Raises if a call before this one is known to have failed."""
    global _told
    if _told is None:
        if torch.cuda.is_current_stream_capturing():   # (no time to allocate)
            return
        flag = torch.zeros(1, dtype=torch.int32, device='cpu', pin_memory=True)
        check(library().d1_muon_error_flag(flag.data_ptr()), 'd1_muon_error_flag')
        _told = C.c_int.from_address(flag.data_ptr()), flag
    if _told[0].value:
        raise D1Error(f'a wait of an earlier Muon step or orthogonalisation ran out (error {_told[0].value}): what it wrote is incomplete, '
                      'the parameters of a step may be too. muon_error() clears it')


def _steps_ok(steps):
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f'steps must be between 1 and {MAX_STEPS}')


class Muon:
    def __init__(self, params, grads, lr=3e-4, momentum=0.95, nesterov=True, weight_decay=0.01, steps=5, copies=None, precise=False):
        params, grads = list(params), list(grads)
        if not params or len(grads) != len(params):
            raise ValueError(f'{len(params)} parameters and {len(grads)} gradients')
        if not (0 <= momentum < 1 and lr >= 0):
            raise ValueError('lr must not be negative and momentum lie in [0, 1)')
        _steps_ok(steps)
        copies = [None] * len(params) if copies is None else list(copies)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(params)
        if len(copies) != len(params) or len(decay) != len(params):
            raise ValueError('copies and weight_decay must have one entry for each parameter')
        self.device = params[0].device
        if self.device.type != 'cuda':
            raise ValueError('params[0] must be on a CUDA device (there is no CPU path)')
        for i, (p, c) in enumerate(zip(params, copies)):
            if p.dtype != F32 or p.device != self.device or not p.is_contiguous() or p.dim() < 2 or not p.numel():
                raise ValueError(f'params[{i}] must be a contiguous float32 tensor [..., rows, cols] on {self.device}')
            if c is not None and (c.dtype != BF16 or c.shape != p.shape or c.device != self.device or not c.is_contiguous()):
                raise ValueError(f'copies[{i}] must be a contiguous bfloat16 tensor of shape {tuple(p.shape)}')
        self._written = _spans([(f'params[{i}]', p) for i, p in enumerate(params)] +
                               [(f'copies[{i}]', c) for i, c in enumerate(copies) if c is not None])
        self.params, self.copies, self.decay = params, copies, decay
        self._leaves = [p for p in params if p.requires_grad]
        self.lr, self.mu, self.nesterov, self.steps, self.precise = lr, momentum, nesterov, steps, bool(precise)
        padded = [(p.numel() + 127) // 128 * 128 for p in params]
        self.offsets = [sum(padded[:i]) for i in range(len(padded))]
        self.momentum = torch.zeros(sum(padded), dtype=F32, device=self.device)
        self.lib = library()
        self._plan = self._work = None
        self.set_grads(grads)

    def set_grads(self, grads):
        """Read the gradients from other tensors from now on (a captured step too). The plan
        is copied on the current stream: the steps', or one that is ordered with it."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f'{len(self.params)} parameters and {len(grads)} gradients')
        table = (_Tensor * len(grads))()
        for i, (p, g, c) in enumerate(zip(self.params, grads, self.copies)):
            kind = GRAD_TYPES.get(g.dtype)
            if kind is None or g.shape != p.shape or g.device != self.device or not g.is_contiguous():
                raise ValueError(f'grads[{i}] must be a contiguous float32 or bfloat16 tensor of shape {tuple(p.shape)} on {self.device}')
            _outside(g, i, self._written)
            rows, cols = p.shape[-2:]
            table[i] = _Tensor(p.data_ptr(), g.data_ptr(), None if c is None else c.data_ptr(), p.numel() // (rows * cols), rows, cols,
                               self.decay[i], kind, self.precise)
        size = self.lib.d1_muon_plan_bytes(table, len(grads))
        if size < 0:
            raise ValueError('the parameters are out of range (2^21 rows or columns, 2^36 elements of work)')
        host = (C.c_uint64 * ((size + 7) // 8))()
        check(self.lib.d1_muon_plan(table, len(grads), self.momentum.data_ptr(), host, C.sizeof(host)), 'd1_muon_plan')
        if self._plan is None:
            self._plan = torch.empty(C.sizeof(host), dtype=torch.uint8, device=self.device)
            self._work = torch.empty(self.lib.d1_muon_work_bytes(table, len(grads)), dtype=torch.uint8, device=self.device)
        self.grads, self._host = grads, host
        self._plan.copy_(torch.frombuffer(bytearray(host), dtype=torch.uint8))

    def step(self, lr=None):
        """One step, in place. lr: this step's learning rate (default: self.lr). Raises D1Error where an earlier step is
        known to have failed (see check())."""
        _watch()
        check(self.lib.d1_muon(self._host, self._plan.data_ptr(), self.lr if lr is None else lr, self.mu, int(self.nesterov),
                               self.steps, self._work.data_ptr(), stream_of(self.momentum)), 'd1_muon')
        if self._leaves:  # torch then refuses a backward pass through what the step has overwritten
            torch.autograd.graph.increment_version(self._leaves)

    def check(self):
        """Raise if a wait inside the steps so far ran out (a GPU that others held for seconds): such a step leaves
        the matrices that go through the products as they were, but for those it had already updated. Synchronises the
        device and clears the error."""
        torch.cuda.synchronize(self.device)
        with torch.cuda.device(self.device):
            code = muon_error()
        if code:
            raise D1Error(f'a wait inside Muon ran out (error {code}): the parameters may be updated in part')

    def momentum_of(self, i):
        """The momentum of parameter i in its shape (a view)."""
        p = self.params[i]
        return self.momentum[self.offsets[i]:self.offsets[i] + p.numel()].view(p.shape)

    def state_dict(self):
        """A copy of the momentum: a run that loads it, with the same parameters, rates and gradients,
        goes on bit for bit."""
        return {'momentum': self.momentum.clone()}

    def load_state_dict(self, state):
        """Takes over a state_dict()."""
        if set(state) != {'momentum'}:
            raise ValueError(f"the state has {sorted(state)}, not ['momentum']")
        m = state['momentum']
        if m.dtype != F32 or m.shape != self.momentum.shape:
            raise ValueError(f'momentum is {m.dtype} {tuple(m.shape)}, not {F32} {tuple(self.momentum.shape)}')
        self.momentum.copy_(m)


def orthogonalize(x, steps=5, out=None, precise=None):
    """x's directions with singular values brought near 1, matrix by matrix of [..., m, n]: bfloat16 or
    float16 as x is, bfloat16 of a float32 one (the products have 16 bits). Rows are contiguous, of one pitch, and
    the matrices of a stack one pitch apart. `out`: a contiguous tensor for the result (bfloat16 or float16), which
    shares no memory with x. precise: products as good as fp32 ones, up to three times their time; None: for a float16 result, whose
    own rounding the others' error (up to 3e-3 of the norm, a bfloat16 result's rounding) would pass. The result has no
    gradient."""
    kind, dev = type_of(x, 'x'), x.device
    if x.dim() < 2:
        raise ValueError(f'x needs two dimensions, not {tuple(x.shape)}')
    _steps_ok(steps)
    rows, cols = x.shape[-2:]
    if rows < 1 or cols < 1:
        raise ValueError('x: the matrices are empty')
    if x.stride(-1) != 1 and cols > 1:
        raise ValueError('x: the last dimension must be contiguous')
    count = x.shape[:-2].numel()
    between = _pitch(x.shape[:-2], x.stride()[:-2], 'x')
    if out is None:
        out = torch.empty(x.shape, dtype=BF16 if x.dtype is F32 else x.dtype, device=dev)
    elif out.dtype not in (BF16, torch.float16) or out.shape != x.shape or out.device != dev or not out.is_contiguous():
        raise ValueError(f'out must be a contiguous bfloat16 or float16 tensor {tuple(x.shape)} on {dev}')
    lib = library()
    _watch()
    if precise is None:
        precise = out.dtype is torch.float16
    call, room = ((lib.d1_orthogonalize_precise, lib.d1_orthogonalize_precise_work_bytes) if precise else
                  (lib.d1_orthogonalize, lib.d1_orthogonalize_work_bytes))
    size = room(count, rows, cols)
    if size < 0:
        raise ValueError(f'{count} matrices of {rows} x {cols} are out of range')
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    check(call(x.data_ptr(), x.stride(-2), between, kind, count, rows, cols, out.data_ptr(), type_of(out, 'out'), steps, work.data_ptr(),
               stream_of(x)), 'd1_orthogonalize')
    return out


def muon_error():
    """The last error of a wait that ran out, on the current device (0: none); clears it."""
    return library().d1_muon_error()
