"""The C entries of layer norm, token log-probabilities and AdamW refuse bad
arguments before any CUDA call (checked without a GPU), and the Python calls
refuse tensors that are not on one."""
import ctypes as C

import pytest
import torch

BAD, LARGE = 9002, 9003
P = 4096  # an aligned address that is never read


@pytest.fixture(scope='module')
def lib():
    from d1 import _lib
    return _lib.library()


def test_layer_norm(lib):
    good = dict(x=P, ldx=8, type=1, rows=2, n=8, w=P, b=P, eps=1e-5, y=P, ldy=8, mean=P, rstd=P, s=None)
    for k, v in dict(type=3, rows=-1, n=0, x=None, y=None, eps=-1.0, ldx=-1, ldy=7).items():
        assert lib.d1_layer_norm(*dict(good, **{k: v}).values()) == BAD, k
    assert lib.d1_layer_norm(*dict(good, x=P + 1).values()) == BAD
    assert lib.d1_layer_norm(*dict(good, eps=float('nan')).values()) == BAD
    assert lib.d1_layer_norm(*dict(good, rows=0).values()) == 0
    good = dict(dy=P, lddy=8, x=P, ldx=8, type=0, rows=2, n=8, w=None, mean=P, rstd=P, dx=P, lddx=8, dw=P, db=P, work=P, s=None)
    for k, v in dict(type=-1, rows=-1, n=0, x=None, dy=None, mean=None, rstd=None, lddx=7, work=None, lddy=-1).items():
        assert lib.d1_layer_norm_backward(*dict(good, **{k: v}).values()) == BAD, k
    assert lib.d1_layer_norm_backward(*dict(good, dx=P + 2).values()) == BAD
    for rows, n in ((-1, 8), (4, 0)):
        assert lib.d1_layer_norm_parts(rows, n) == BAD
    for rows in (0, 1, 7, 100000):
        for n in (1, 64, 512, 4096, 8193, 50000):
            assert 1 <= lib.d1_layer_norm_parts(rows, n) <= 148 * 32


def test_token_logprob(lib):
    good = dict(x=P, ld=40, type=1, rows=2, vocab=40, tokens=P, legal=P, ldl=5, t=1.0, top=2, logp=P, ent=P, stats=P, tt=P, tl=P, s=None)
    for k, v in dict(type=9, rows=-1, vocab=0, x=None, tokens=None, ldl=-1, t=0.0, top=-1, tt=None, tl=None, ld=-1).items():
        assert lib.d1_token_logprob(*dict(good, **{k: v}).values()) == BAD, k
    assert lib.d1_token_logprob(*dict(good, t=float('nan')).values()) == BAD
    assert lib.d1_token_logprob(*dict(good, x=P + 1).values()) == BAD
    assert lib.d1_token_logprob(*dict(good, top=33).values()) == LARGE
    assert lib.d1_token_logprob(*dict(good, rows=0).values()) == 0
    good = dict(x=P, ld=40, type=1, rows=2, vocab=40, tokens=P, legal=None, ldl=0, t=1.0, stats=P, ent=P, dl=P, dh=P, d=P, ldd=40, s=None)
    for k, v in dict(type=9, rows=-1, vocab=0, x=None, stats=None, d=None, tokens=None, ent=None, ldd=39, t=-1.0).items():
        assert lib.d1_token_logprob_backward(*dict(good, **{k: v}).values()) == BAD, k


def test_adamw(lib):
    good = dict(tensors=P, n=1, blocks=1, bits=8, m=P, v=P, ms=P, vs=P, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, clip=0.0, step=P, seed=0,
                work=P, norm=None, s=None)
    for k, v in dict(tensors=None, n=0, blocks=0, bits=16, m=None, v=None, ms=None, vs=None, b1=1.0, b2=-0.1, eps=-1.0, step=None,
                     work=None).items():
        assert lib.d1_adamw(*dict(good, **{k: v}).values()) == BAD, k
    assert lib.d1_adamw(*dict(good, m=P + 4).values()) == BAD
    assert lib.d1_adamw(*dict(good, blocks=2 ** 31).values()) == LARGE
    assert lib.d1_adamw_work_bytes() >= 16


def test_host_tensors_are_refused():
    from d1.adamw import AdamW, _Tensor
    from d1.layer_norm import layer_norm
    from d1.token_logprob import token_logprob
    x = torch.zeros(4, 8)
    for bad in (lambda: layer_norm(x), lambda: token_logprob(x, torch.zeros(4, dtype=torch.int64)), lambda: AdamW([x], [x])):
        with pytest.raises(ValueError):
            bad()
    assert C.sizeof(_Tensor) == 56  # D1AdamWTensor
