"""AdamW over many parameter tensors in one launch (d1_adamw).

    opt = AdamW(params, grads, lr=3e-4, weight_decay=0.01, state_bits=8, max_norm=0.5)
    opt.step()          # reads grads, updates params, moments, step count and bf16 copies in place

params are contiguous float32 tensors (masters) of any size and alignment,
grads float32 or bfloat16 of the same shapes; each step reads whatever the
gradient tensors then hold. copies (bfloat16, or None for a tensor that has
none) are refreshed by the step. weight_decay and copies may differ by tensor.
No parameter or copy shares memory with another one or with a gradient, and each
keeps its storage for the optimizer's life (the step has their addresses).
An eps below 2^-63 counts as 2^-63.

Moments are held in 32 bits, or in 8: m as float8_e4m3fn and v as float8_e5m2
codes with a power-of-two scale for each block of 128 elements, 2.06 bytes a
parameter in place of 8. They are flat over the tensors, each padded to whole
blocks (`offsets` says where a tensor starts); moments(i) gives a tensor's as
float32. The step count is on the device, so a captured step stays correct.
Steps of one optimizer share its work buffer: run them on one stream, or
ordered.
"""
import bisect
import ctypes as C

import torch

from ._lib import check, library, stream_of

BLOCK = 128
GRAD_TYPES = {torch.float32: 0, torch.bfloat16: 1}  # D1_TYPE_* of d1.h


class _Tensor(C.Structure):
    _fields_ = [('param', C.c_void_p), ('grad', C.c_void_p), ('copy', C.c_void_p), ('count', C.c_int64),
                ('first_block', C.c_int64), ('decay', C.c_double), ('grad_type', C.c_int), ('reserved', C.c_int)]


def _spans(named):
    """(first addresses, ends, names) in order of the (name, tensor) pairs that a step
    writes, which may share no memory: two warps would write the same elements."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), name) for name, t in named if t.numel())
    for (_, end, name), (at, _, other) in zip(spans, spans[1:]):
        if at < end:
            raise ValueError(f'{name} and {other} share memory')
    return tuple(zip(*spans)) or ((), (), ())


def _outside(t, i, spans):
    """Refuses gradient i, which a step reads, if it writes one of the spans over it."""
    starts, ends, names = spans
    at = t.data_ptr()
    end = at + t.nbytes
    near = bisect.bisect_left(starts, end) - 1  # the last span that begins before its end
    if near >= 0 and ends[near] > at < end:
        raise ValueError(f'grads[{i}] shares memory with {names[near]}')


class AdamW:
    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 max_norm=0.0, copies=None, seed=0):
        params, grads = list(params), list(grads)
        if not params or len(grads) != len(params):
            raise ValueError(f'{len(params)} parameters and {len(grads)} gradients')
        if state_bits not in (8, 32):
            raise ValueError('state_bits must be 8 or 32')
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and lr >= 0 and max_norm >= 0):
            raise ValueError('lr, eps and max_norm must not be negative and the betas lie in [0, 1)')
        copies = [None] * len(params) if copies is None else list(copies)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(params)
        if len(copies) != len(params) or len(decay) != len(params):
            raise ValueError('copies and weight_decay must have one entry for each parameter')
        self.device = params[0].device
        if self.device.type != 'cuda':
            raise ValueError('params[0] must be on a CUDA device (there is no CPU path)')
        for i, (p, c) in enumerate(zip(params, copies)):
            if p.dtype != torch.float32 or p.device != self.device or not p.is_contiguous():
                raise ValueError(f'params[{i}] must be a contiguous float32 tensor on {self.device}')
            if c is not None and (c.dtype != torch.bfloat16 or c.shape != p.shape or c.device != self.device or
                                  not c.is_contiguous()):
                raise ValueError(f'copies[{i}] must be a contiguous bfloat16 tensor of shape {tuple(p.shape)}')
        self._written = _spans([(f'params[{i}]', p) for i, p in enumerate(params)] +
                               [(f'copies[{i}]', c) for i, c in enumerate(copies) if c is not None])
        self.params, self.copies, self.decay = params, copies, decay
        self._leaves = [p for p in params if p.requires_grad]
        self.lr, self.betas, self.eps, self.max_norm = lr, betas, eps, max_norm
        self.state_bits, self.seed = state_bits, seed
        blocks = [(p.numel() + BLOCK - 1) // BLOCK for p in params]
        self._first = [sum(blocks[:i]) for i in range(len(blocks))]
        self.offsets = [b * BLOCK for b in self._first]
        self.nblocks = sum(blocks)
        if not self.nblocks:
            raise ValueError('the parameters hold no elements')
        n, dev = self.nblocks * BLOCK, self.device
        f32 = dict(dtype=torch.float32, device=dev)
        if state_bits == 32:
            self.m, self.v = torch.zeros(n, **f32), torch.zeros(n, **f32)
            self.m_scale = self.v_scale = None
        else:
            self.m = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
            self.v = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e5m2)
            self.m_scale, self.v_scale = torch.ones(self.nblocks, **f32), torch.ones(self.nblocks, **f32)
        self.lib = library()
        self.step_dev = torch.zeros(1, dtype=torch.int64, device=dev)
        self.grad_norm = torch.zeros(1, **f32)  # the last step's, when it clips
        self._work = torch.zeros(self.lib.d1_adamw_work_bytes(), dtype=torch.uint8, device=dev)
        self._table = torch.empty(len(params) * C.sizeof(_Tensor), dtype=torch.uint8, device=dev)
        at = lambda t: None if t is None else t.data_ptr()
        self._state_args = (self._table.data_ptr(), len(params), self.nblocks, state_bits, at(self.m), at(self.v),
                            at(self.m_scale), at(self.v_scale))
        self._step_dev, self._step_args = self.step_dev.data_ptr(), (self._work.data_ptr(), self.grad_norm.data_ptr())
        self.set_grads(grads)

    def set_grads(self, grads):
        """Read the gradients from other tensors from now on (a captured step too). The tensors'
        list is copied on the current stream: the steps', or one that is ordered with it."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f'{len(self.params)} parameters and {len(grads)} gradients')
        table = (_Tensor * len(grads))()
        for i, (p, g, c) in enumerate(zip(self.params, grads, self.copies)):
            kind = GRAD_TYPES.get(g.dtype)
            if kind is None or g.shape != p.shape or g.device != self.device or not g.is_contiguous():
                raise ValueError(f'grads[{i}] must be a contiguous float32 or bfloat16 tensor of shape '
                                 f'{tuple(p.shape)} on {self.device}')
            _outside(g, i, self._written)
            table[i] = _Tensor(p.data_ptr(), g.data_ptr(), None if c is None else c.data_ptr(), p.numel(),
                               self._first[i], self.decay[i], kind, 0)
        self.grads = grads
        self._table.copy_(torch.frombuffer(bytearray(table), dtype=torch.uint8))

    def step(self, lr=None):
        """One step, in place. lr: this step's learning rate (default: self.lr)."""
        check(self.lib.d1_adamw(*self._state_args, self.lr if lr is None else lr, self.betas[0], self.betas[1], self.eps,
                                self.max_norm, self._step_dev, self.seed, *self._step_args, stream_of(self.m)), 'd1_adamw')
        if self._leaves:  # torch then refuses a backward pass through what the step has overwritten
            torch.autograd.graph.increment_version(self._leaves)

    def moments(self, i):
        """(m, v) of parameter i as float32 in its shape (decoded copies where the state is in 8 bits)."""
        p, first = self.params[i], self._first[i]
        blocks = slice(first, first + (p.numel() + BLOCK - 1) // BLOCK)
        out = []
        for x, scale in ((self.m, self.m_scale), (self.v, self.v_scale)):
            x = x.view(-1, BLOCK)[blocks].float()
            if scale is not None:
                x = x * scale[blocks, None]
            out.append(x.reshape(-1)[:p.numel()].view(p.shape))
        return tuple(out)

    def _state(self):
        return {k: getattr(self, k) for k in ('m', 'v', 'm_scale', 'v_scale') if getattr(self, k) is not None}

    def state_dict(self):
        """Copies of the moments, the step count and the seed of the 8-bit rounding: a run that
        loads them, with the same parameters, rates and gradients, goes on bit for bit."""
        return dict({k: t.clone() for k, t in self._state().items()}, step=int(self.step_dev.item()), seed=self.seed)

    def load_state_dict(self, state):
        """Takes over a state_dict() (one without a seed leaves the seed as it is)."""
        own = self._state()
        if set(state) - {'seed'} != set(own) | {'step'}:
            raise ValueError(f'the state has {sorted(state)}, not {sorted(own) + ["step"]}')
        for k, t in own.items():
            if state[k].dtype != t.dtype or state[k].shape != t.shape:
                raise ValueError(f'{k} is {state[k].dtype} {tuple(state[k].shape)}, not {t.dtype} {tuple(t.shape)}')
        for k, t in own.items():
            t.copy_(state[k])
        self.step_dev.fill_(state['step'])
        self.seed = state.get('seed', self.seed)
