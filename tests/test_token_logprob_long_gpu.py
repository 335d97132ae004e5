"""Rows of more than 8,192 tokens in numbers that give each a whole block (from 296 rows
on): the edge rows, equal logits in great numbers, cells of one and of several batches.
Tolerances are those of test_token_logprob_gpu."""
import math

import pytest
import torch
from test_token_logprob_gpu import check_forward, unpack

pytestmark = pytest.mark.gpu


def edge_rows(vocab, dtype):
    low, inf = torch.finfo(dtype).min, math.inf
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = torch.randn(14, vocab, device='cuda', generator=g).to(dtype)
    x[0] = low
    x[1] = -inf
    x[2], x[2, vocab // 2] = -inf, 3.0
    x[3] = 0.0
    x[4, ::2], x[4, 1::2] = -0.0, 0.0
    x[5] = torch.arange(vocab, device='cuda').clamp(max=60000).to(dtype)
    x[6, vocab // 3] = math.nan
    x[7, vocab // 3] = inf
    x[8, 1:] = low
    x[9, vocab - 1] = torch.finfo(dtype).max
    x[10], x[10, [7, 100, vocab - 1]] = -1e4, torch.tensor([0.5, 2.0, 1.0], device='cuda', dtype=dtype)  # masked by a finite number
    x[11] = -1.5                                                                                         # equal and negative
    x[12] = -torch.arange(vocab, device='cuda').div(700, rounding_mode='floor').clamp(max=90).to(dtype)  # hundreds of each
    x[13] = x[12].flip(0)
    return x


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('vocab, rows', [(9001, 700), (20011, 602), (100003, 602), (230007, 406), (2500, 700)])
def test_edge_rows(vocab, rows, masked, dtype):
    from d1.token_logprob import token_logprob
    x = edge_rows(vocab, dtype)
    pitch = (vocab + 15) // 16 * 16                  # every copy of a row has the same alignment, so the same bits
    logits = torch.zeros(rows, pitch, device='cuda', dtype=dtype)[:, :vocab]
    logits.copy_(x.repeat(rows // 14, 1))
    legal = None
    if masked:
        g = torch.Generator(device='cuda').manual_seed(1)
        legal = torch.randint(0, 256, (14, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
        at, bit = vocab // 3 // 8, 1 << (vocab // 3 % 8)
        legal[6, at] |= bit                          # the NaN is in, the +inf is left out
        legal[7, at] &= 255 - bit
    tokens = torch.full((rows,), vocab // 2, device='cuda')
    got = token_logprob(logits, tokens, None if legal is None else legal.repeat(rows // 14, 1), top=20)
    for t in got:
        tiles = t.view(rows // 14, 14, -1)
        tiles = tiles.view(torch.int32) if t.dtype is torch.float32 else tiles   # bits, for NaN
        assert (tiles == tiles[:1]).all()
    bad = [6] if masked else [6, 7]
    ok = [r for r in range(14) if r not in bad]
    check_forward(x[ok], tokens[ok], None if legal is None else legal[ok], 1.0, 20, type(got)(*(t[ok] for t in got)))
    for r in bad:
        taken = legal is None or bool(unpack(legal, vocab)[r, vocab // 2])   # a token that is left out has -inf in any row
        assert got.logp[r].isnan() if taken else got.logp[r] == -math.inf
        assert got.entropy[r].isnan() and got.top_tokens[r, 0] == vocab // 3
    if not masked:
        assert got.top_tokens[11].tolist() == list(range(20)) == got.top_tokens[0].tolist()
        assert got.top_tokens[10, :4].tolist() == [100, vocab - 1, 7, 0]
    else:
        first = unpack(legal, vocab)[11].nonzero()[:20, 0]
        assert torch.equal(got.top_tokens[11], first)


@pytest.mark.parametrize('vocab', [4096, 32768])
def test_negative_ties_cost_what_positive_ones_do(vocab):
    """Equal logits in great numbers take one more pass over the row; negative ones of 16 bits used to take one for
    each alternative (10 times as long with 20). A factor of four is far from either."""
    from d1.token_logprob import token_logprob
    tokens = torch.zeros(600, dtype=torch.int64, device='cuda')
    took = []
    for value in (1.5, -1.5):
        x = torch.full((600, vocab), value, device='cuda', dtype=torch.bfloat16)
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                token_logprob(x, tokens, top=20)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    assert took[1] < 4 * took[0], took
