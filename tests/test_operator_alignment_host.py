"""The C entries of layer norm, token log-probabilities and AdamW refuse pointers that are
no multiple of what they point to, which on the GPU would be a misaligned access
(checked before any CUDA call, so without a GPU)."""
import pytest

BAD = 9002
P = 1 << 20  # an aligned address that is never read; the matrices are 1 Mi apart


@pytest.fixture(scope='module')
def lib():
    from d1 import _lib
    return _lib.library()


def refused(f, good, **off):
    for name, by in off.items():
        bad = dict(good)
        assert bad[name] is not None, name
        bad[name] += by
        assert f(*bad.values()) == BAD, name


def test_layer_norm(lib):
    good = dict(x=P, ldx=8, type=1, rows=2, n=8, w=P, b=P, eps=1e-5, y=2 * P, ldy=8, mean=P, rstd=P, s=None)
    refused(lib.d1_layer_norm, good, x=1, y=1, w=2, b=1, mean=2, rstd=3)
    good = dict(dy=P, lddy=8, x=2 * P, ldx=8, type=0, rows=2, n=8, w=P, mean=P, rstd=P, dx=3 * P, lddx=8, dw=P, db=P, work=P, s=None)
    refused(lib.d1_layer_norm_backward, good, dy=2, x=2, dx=2, w=1, mean=2, rstd=2, dw=2, db=2, work=8)


def test_token_logprob(lib):
    good = dict(x=P, ld=40, type=1, rows=2, vocab=40, tokens=P, legal=P, ldl=5, t=1.0, top=2, logp=P, ent=P, stats=P, tt=P, tl=P, s=None)
    refused(lib.d1_token_logprob, good, x=1, tokens=4, logp=2, ent=2, stats=2, tt=4, tl=2)
    good = dict(x=P, ld=40, type=1, rows=2, vocab=40, tokens=P, legal=P + 1, ldl=5, t=1.0, stats=P, ent=P, dl=P, dh=P, d=2 * P, ldd=40, s=None)
    refused(lib.d1_token_logprob_backward, good, x=1, d=1, tokens=4, stats=2, ent=2, dl=2, dh=1)


def test_adamw(lib):
    good = dict(tensors=P, n=1, blocks=1, bits=8, m=P, v=P, ms=P, vs=P, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, clip=1.0, step=P, seed=0,
                work=P, norm=P, s=None)
    refused(lib.d1_adamw, good, tensors=4, m=8, v=8, ms=2, vs=2, step=4, work=8, norm=2)
