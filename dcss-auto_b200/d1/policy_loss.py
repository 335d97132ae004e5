"""The clipped policy loss with KL and entropy terms, and its gradient (d1_policy_loss).

    r = token_logprob(logits, tokens, legal=legal)
    p = policy_loss(r.logp, old_logp, advantage, ref_logp=ref, entropy=r.entropy, mask=live,
                    clip=(0.2, 0.28), kl_coef=0.05, ent_coef=0.01)
    dlogits = token_logprob_backward(logits, tokens, r.stats, r.entropy, p.dlogp, p.dentropy, legal=legal)

    loss = mean( -min(ratio A, clip(ratio) A) + kl_coef (e^d - d - 1) - ent_coef H )
    ratio = e^(logp - old_logp), clip to [1 - low, 1 + high], d = ref_logp - logp

logp, old_logp, ref_logp and entropy are float32 [..., length] whose leading
dimensions have one row pitch; advantage has that shape, or one number for each row
[...]. mask (bool or uint8) marks the tokens that count: the others are never looked
at, whatever they hold. mean='token' takes the mean over all tokens that count,
'row' over the rows that have any of each row's mean. A batch without a token that
counts has a loss of 0 and gradients of 0. ratio and e^d are float32, infinite past a
difference of 88.7; beside one an advantage or a coefficient of 0 still takes no part. The log-probabilities are float32
because their differences are close to 0, where 16 bits would leave no ratio.

The gradient comes with the loss, in one pass: each token's needs nothing that the
loss has not read. The calls launch on the current stream of logp's device and
can be captured in a CUDA graph. Where torch records gradients of logp or entropy,
loss leads back to them (first derivatives); old_logp, advantage and ref_logp have none.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import check, library, stream_of
from ._rows import empty_f32, matrix

MEANS = {'token': 0, 'row': 1}


class PolicyLoss(NamedTuple):
    loss: torch.Tensor             # float32 []
    stats: torch.Tensor            # float32 [5]: means of the clipped term, of e^d - d - 1, of the entropy, of the
                                   # tokens that were clipped (their share) and of ratio - 1 - log ratio
    dlogp: torch.Tensor = None     # float32, the loss's gradient by logp
    dentropy: torch.Tensor = None  # float32, by entropy


def _floats(t, like, ld, shape, device, name):
    """(address, row pitch) of t, whose rows lie as those of `like` (ld) more often than not."""
    if t is None:
        return None, 0
    if t.dtype is torch.float32 and t.device == device and t.shape == shape:
        if t.stride() == like:
            return t.data_ptr(), ld
    else:
        raise ValueError(f'{name} must be float32 {tuple(shape)} on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}')
    p, _, _, ld = matrix(t, name)
    return p, ld


def _advantage(t, like, ld, shape, device):
    """(address, row pitch, whether it is one number a row)."""
    if t.shape == shape or t.dim() != len(shape) - 1:
        return *_floats(t, like, ld, shape, device, 'advantage'), 0
    p, ld = _floats(t.unsqueeze(-1), None, 0, (*shape[:-1], 1), device, 'advantage')
    return p, ld, 1


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, entropy, *others):
        r = _policy_loss(logp, entropy, *others)
        ctx.save_for_backward(r.dlogp, r.dentropy)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in r[1:] if t is not None))
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *others):
        dlogp, dentropy = ctx.saved_tensors
        need = ctx.needs_input_grad
        out = [d * dloss if dloss is not None and n else None for d, n in zip((dlogp, dentropy), need)]
        return (*out, *(None for _ in need[2:]))


def policy_loss(logp, old_logp, advantage, ref_logp=None, entropy=None, mask=None, clip=0.2, kl_coef=0.0,
                ent_coef=0.0, mean='token', gradient=True):
    """PolicyLoss of these tokens. clip: one number, or (low, high). gradient=False leaves the
    gradients out (None) where torch records none."""
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (low >= 0 and high >= 0):
        raise ValueError('clip must not be negative')
    if mean not in MEANS:
        raise ValueError(f"mean must be 'token' or 'row', not {mean!r}")
    args = (old_logp, advantage, ref_logp, mask, low, high, kl_coef, ent_coef, MEANS[mean])
    if torch.is_grad_enabled() and (logp.requires_grad or (entropy is not None and entropy.requires_grad)):
        return PolicyLoss(*_PolicyLoss.apply(logp, entropy, *args, True))
    return _policy_loss(logp, entropy, *args, gradient)


def _policy_loss(logp, entropy, old_logp, advantage, ref_logp, mask, low, high, kl_coef, ent_coef, by_row, gradient):
    if logp.dtype is not torch.float32 or not logp.is_cuda:
        raise ValueError(f'logp must be float32 on a CUDA device (there is no CPU path), not {logp.dtype} on {logp.device}')
    shape, dev = logp.shape, logp.device
    px, rows, length, ld = matrix(logp, 'logp')
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.shape != shape or mask.device != dev:
            raise ValueError(f'mask must be a bool or uint8 tensor {tuple(shape)} on {dev}, not {mask.dtype} '
                             f'{tuple(mask.shape)} on {mask.device}')
        pm, _, _, ldm = matrix(mask, 'mask')
    else:
        pm, ldm = None, 0
    as_logp = logp.stride(), ld, shape, dev
    old, adv = _floats(old_logp, *as_logp, 'old_logp'), _advantage(advantage, *as_logp)
    ref, ent = _floats(ref_logp, *as_logp, 'ref_logp'), _floats(entropy, *as_logp, 'entropy')
    lib = library()
    size = 0 if rows * length <= 2048 else lib.d1_policy_loss_work_bytes(rows, length)  # (a small batch needs none)
    if size < 0 or (mask is not None and rows * length > 2 ** 31 - 1):
        raise ValueError(f'{rows} rows of {length} tokens are out of range')
    work = empty_f32(dev, (size + 3) // 4) if size else None
    loss, stats = empty_f32(dev), empty_f32(dev, 5)
    dlogp = empty_f32(dev, *shape) if gradient else None
    dentropy = empty_f32(dev, *shape) if gradient and entropy is not None else None
    at = lambda t: None if t is None else t.data_ptr()
    check(lib.d1_policy_loss(px, ld, *old, *adv, *ref, *ent, pm, ldm, rows, length, low, high, kl_coef, ent_coef, by_row,
                             loss.data_ptr(), stats.data_ptr(), at(dlogp), at(dentropy), at(work), stream_of(logp)),
          'd1_policy_loss')
    return PolicyLoss(loss, stats, dlogp, dentropy)
