"""The C entries of layer norm and token log-probabilities without some of their outputs
(NULL): what is wanted has the bits that it has with all of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def at(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize('n', [48, 257, 1000, 1536, 4096, 9000, 20000, 40000])
def test_layer_norm(n):
    from d1._lib import check, library, stream_of
    lib, rows = library(), 37
    g = torch.Generator(device='cuda').manual_seed(n)
    new = lambda *shape: torch.randn(*shape, device='cuda', generator=g)
    for dtype, kind in ((torch.float32, 0), (torch.bfloat16, 1)):
        x, dy, w, b = new(rows, n).to(dtype), new(rows, n).to(dtype), new(n), new(n)

        def forward(mean, rstd):
            y = torch.empty_like(x)
            check(lib.d1_layer_norm(at(x), n, kind, rows, n, at(w), at(b), 1e-5, at(y), n, at(mean), at(rstd), stream_of(x)))
            return y

        def backward(dx, dw, db):
            work = new(lib.d1_layer_norm_parts(rows, n) * 2 * n) if dw is not None or db is not None else None
            check(lib.d1_layer_norm_backward(at(dy), n, at(x), n, kind, rows, n, at(w), at(mean), at(rstd), at(dx), n, at(dw), at(db),
                                             at(work), stream_of(x)))
        mean, rstd = new(rows), new(rows)
        y, only = forward(mean, rstd), new(rows)
        assert torch.equal(forward(None, None), y) and torch.equal(forward(only, None), y) and torch.equal(only, mean)
        assert torch.equal(forward(None, only), y) and torch.equal(only, rstd)
        want = torch.empty_like(x), new(n), new(n)
        backward(*want)
        for keep in range(8):
            got = [torch.full_like(t, 7) if keep >> i & 1 else None for i, t in enumerate(want)]
            backward(*got)
            assert all(t is None or torch.equal(t, r) for t, r in zip(got, want)), keep


@pytest.mark.parametrize('rows, vocab', [(37, 28), (37, 1000), (400, 9000), (2, 70000)])
def test_token_logprob(rows, vocab):
    from d1._lib import check, library, stream_of
    lib = library()
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = torch.randn(rows, vocab, device='cuda', generator=g)
    tokens = torch.randint(0, vocab, (rows,), device='cuda', generator=g)
    new = lambda *shape: torch.full(shape, 7.0, device='cuda')

    def forward(logp, entropy, stats, top, top_tokens, top_logp, tokens=tokens):
        check(lib.d1_token_logprob(at(x), vocab, 0, rows, vocab, at(tokens), None, 0, 0.9, top, at(logp), at(entropy), at(stats),
                                   at(top_tokens), at(top_logp), stream_of(x)))
    want = new(rows), new(rows), new(rows, 2)
    tt, tl = torch.zeros(rows, 5, dtype=torch.int64, device='cuda'), new(rows, 5)
    forward(*want, 5, tt, tl)
    for keep in range(8):
        got = [torch.zeros_like(t) if keep >> i & 1 else None for i, t in enumerate(want)]
        for top in (0, 5):
            a, b = (torch.zeros_like(tt), torch.zeros_like(tl)) if top else (None, None)
            forward(*got, top, a, b, tokens if keep & 1 else None)
            assert all(t is None or torch.equal(t, r) for t, r in zip(got, want)), keep
            assert not top or (torch.equal(a, tt) and torch.equal(b, tl))

    def backward(dlogp, dentropy, entropy, tokens):
        d = new(rows, vocab)
        check(lib.d1_token_logprob_backward(at(x), vocab, 0, rows, vocab, at(tokens), None, 0, 0.9, at(want[2]), at(entropy), at(dlogp),
                                            at(dentropy), at(d), vocab, stream_of(x)))
        return d
    some, zero = torch.randn(rows, device='cuda', generator=g), torch.zeros(rows, device='cuda')
    assert torch.equal(backward(some, None, None, tokens), backward(some, zero, want[1], tokens))
    assert torch.equal(backward(None, some, want[1], None), backward(zero, some, want[1], tokens))
    assert (backward(None, None, None, None) == 0).all()
