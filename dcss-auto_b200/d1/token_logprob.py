"""Log-probabilities of given tokens (actions), with the distribution's entropy
and its likeliest alternatives, and their gradient (d1_token_logprob).

    r = token_logprob(logits, tokens, legal=legal, top=8)
    dlogits = token_logprob_backward(logits, tokens, r.stats, r.entropy, dlogp, dentropy, legal=legal)

logits are float32, bfloat16 or float16 [..., vocab] with one row pitch; tokens
int64 [...], negative where a row has none. `legal` holds a bit per token, as
the environments' legal masks do: an integer tensor [...] or [..., words], bit
j of a row (counted from its lowest byte) for token j; a mask shared by all
rows may be expanded. A token whose bit is clear counts for nothing, whatever
its logit holds. The calls launch on the current stream of the logits' device
and can be captured in a CUDA graph. Where torch records gradients of the
logits, logp and entropy have their (first) gradient; the others have none.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import check, library, stream_of
from ._rows import apart, empty_f32, empty_like, like, matrix, recorded, type_of, vector

MAX_TOP = 32
LEAST, MOST = 2.0 ** -126, 3.4028234663852886e38  # temperatures: fp32 numbers with a finite reciprocal


class TokenLogprob(NamedTuple):
    logp: torch.Tensor                 # float32 [...]; 0 where a row has no token, -inf where it is left out
    entropy: torch.Tensor              # float32 [...]
    stats: torch.Tensor                # float32 [..., 2], for the backward pass
    top_tokens: torch.Tensor = None    # int64 [..., top], likeliest first, -1 where no token is left
    top_logp: torch.Tensor = None      # float32 [..., top]


_BITS = {torch.uint8: 1, torch.int8: 1, torch.int16: 2, torch.int32: 4, torch.int64: 8}  # bytes of a mask's words


def _legal(legal, lead, vocab, device):
    """(address, row pitch in bytes) of the mask."""
    if legal is None:
        return None, 0
    size = _BITS.get(legal.dtype)
    if size is None:
        raise ValueError(f'legal must be an integer tensor of bits, not {legal.dtype}')
    if legal.shape == lead:
        legal = legal.unsqueeze(-1)
    if legal.shape[:-1] != lead or legal.device != device:
        raise ValueError(f'legal {tuple(legal.shape)} on {legal.device} does not match rows {tuple(lead)} on {device}')
    p, _, words, pitch = matrix(legal, 'legal')
    if words * size * 8 < vocab:
        raise ValueError(f'legal has {words * size * 8} bits a row for {vocab} tokens')
    return p, pitch * size


def _common(logits, tokens, legal, temperature):
    kind, dev, m = type_of(logits, 'logits'), logits.device, matrix(logits, 'logits')
    if not LEAST <= temperature <= MOST:
        raise ValueError(f'temperature must be between {LEAST} and {MOST}')
    lead = logits.shape[:-1]
    if tokens.shape != lead:
        raise ValueError(f'tokens {tuple(tokens.shape)} do not match rows {tuple(lead)}')
    t = vector(tokens, m[1], torch.int64, dev, 'tokens')
    return dev, kind, m, lead, t, _legal(legal, lead, m[2], dev)


class _TokenLogprob(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, legal, temperature, top):
        r = _token_logprob(logits, tokens, legal, temperature, top)
        ctx.save_for_backward(logits, tokens, legal, r.stats, r.entropy)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in r[2:] if t is not None))
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, *others):
        if dlogp is None and dentropy is None:
            return (None,) * 5
        logits, tokens, legal, stats, entropy = ctx.saved_tensors
        dlogp, dentropy = (None if g is None else g.contiguous() for g in (dlogp, dentropy))
        return token_logprob_backward(logits, tokens, stats, entropy, dlogp, dentropy, legal, ctx.temperature), None, None, None, None


def token_logprob(logits, tokens, legal=None, temperature=1.0, top=0):
    """TokenLogprob of softmax(logits / temperature) over the legal tokens."""
    if recorded(logits):
        return TokenLogprob(*_TokenLogprob.apply(logits, tokens, legal, temperature, top))
    return _token_logprob(logits, tokens, legal, temperature, top)


def _token_logprob(logits, tokens, legal, temperature, top):
    dev, kind, (px, rows, vocab, ld), lead, t, (bits, pitch) = _common(logits, tokens, legal, temperature)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f'top must be between 0 and {MAX_TOP}')
    shape = (rows,) if len(lead) == 1 else lead
    logp, entropy, stats = empty_f32(dev, *shape), empty_f32(dev, *shape), empty_f32(dev, *shape, 2)
    top_tokens = top_logp = tt = tl = None
    if top:
        top_tokens, top_logp = tokens.new_empty((*shape, top)), empty_f32(dev, *shape, top)
        tt, tl = top_tokens.data_ptr(), top_logp.data_ptr()
    check(library().d1_token_logprob(px, ld, kind, rows, vocab, t, bits, pitch, temperature, top, logp.data_ptr(),
                                     entropy.data_ptr(), stats.data_ptr(), tt, tl, stream_of(logits)),
          'd1_token_logprob')
    return TokenLogprob(logp, entropy, stats, top_tokens, top_logp)


def token_logprob_backward(logits, tokens, stats, entropy, dlogp, dentropy=None, legal=None, temperature=1.0,
                           out=None):
    """dlogits (the logits' shape and type) from the gradients of logp and of the
    entropy (float32 of the rows' shape; either may be None: zero), written to `out` when given,
    which overlaps no input."""
    dev, kind, m, _, t, (bits, pitch) = _common(logits, tokens, legal, temperature)
    px, rows, vocab, ld = m
    f32 = torch.float32
    s = vector(stats, 2 * rows, f32, dev, 'stats')
    if dentropy is not None and entropy is None:
        raise ValueError('dentropy needs the entropy')
    h, dl = vector(entropy, rows, f32, dev, 'entropy'), vector(dlogp, rows, f32, dev, 'dlogp')
    dh = vector(dentropy, rows, f32, dev, 'dentropy')
    if out is None:
        out = empty_like(logits)
        po, ldo = out.data_ptr(), vocab
    else:
        po, _, _, ldo = d = like(out, logits, 'out')
        apart(d, m, logits.element_size(), 'out', 'logits')
    check(library().d1_token_logprob_backward(px, ld, kind, rows, vocab, t, bits, pitch, temperature, s, h, dl, dh, po,
                                              ldo, stream_of(logits)), 'd1_token_logprob_backward')
    return out
