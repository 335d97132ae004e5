"""Cases, plain forms and 64-bit values of the training operators for policies with named parameter
tensors: layer norm (forward and backward), log-probabilities of given tokens with entropy and top
alternatives (forward and backward), and the AdamW step over many tensors (states in 32 and in 8 bits).

A case is a dict of plain values; prepare() makes its inputs on the GPU from a seed, run() makes one call
of the operator (with `own`, through the package; else in elementary torch operations in 32 bits), exact()
computes the same outputs in 64 bits, and work() counts the bytes and operations no implementation can do
without.
"""
import math
import pathlib
import sys

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-5
BLOCK = 128  # elements of one scale of an 8-bit optimizer state
LR, BETAS, ADAM_EPS, DECAY = 3e-4, (0.9, 0.999), 1e-8, 0.01
AGE = 100    # steps the optimizer has taken before the measured one
MAX_CASE_BYTES = 3_500_000_000


def listed():
    return [
        # the 256-wide hidden layer of the policy for one small batch of environments: latency
        {'name': 'ln_fwd_small', 'op': 'ln', 'pass': 'fwd', 'rows': 64, 'n': 256, 'dtype': 'bf16'},
        # the 512-wide features of 65,536 environments
        {'name': 'ln_fwd_512', 'op': 'ln', 'pass': 'fwd', 'rows': 65536, 'n': 512, 'dtype': 'bf16'},
        # a training minibatch of 16,384 rows through a wide layer
        {'name': 'ln_bwd_4096', 'op': 'ln', 'pass': 'bwd', 'rows': 16384, 'n': 4096, 'dtype': 'bf16'},
        # odd sizes, in 32 bits
        {'name': 'ln_bwd_odd', 'op': 'ln', 'pass': 'bwd', 'rows': 5003, 'n': 1111, 'dtype': 'f32'},
        # the 28 joint actions (verb and target) of a small batch, with legal bits and 4 alternatives
        {'name': 'lp_joint', 'op': 'lp', 'pass': 'fwd', 'rows': 4096, 'vocab': 28, 'dtype': 'f32', 'legal': True,
         'top': 4, 'temperature': 1.0},
        # a minibatch over a word-sized vocabulary, with 8 alternatives
        {'name': 'lp_fwd_32k', 'op': 'lp', 'pass': 'fwd', 'rows': 4096, 'vocab': 32768, 'dtype': 'bf16',
         'legal': False, 'top': 8, 'temperature': 1.0},
        # scoring single tokens of a few sequences over a large vocabulary: few long rows
        {'name': 'lp_decode', 'op': 'lp', 'pass': 'fwd', 'rows': 4, 'vocab': 131072, 'dtype': 'bf16', 'legal': True,
         'top': 20, 'temperature': 0.7},
        # the gradient of log-probability and entropy over an odd vocabulary (rows start unaligned)
        {'name': 'lp_bwd_odd', 'op': 'lp', 'pass': 'bwd', 'rows': 4096, 'vocab': 50021, 'dtype': 'bf16',
         'legal': True, 'top': 0, 'temperature': 1.0},
        # the 17 parameter tensors of the conv policy, clipped as the PPO update clips, with bf16 copies
        {'name': 'adamw_policy', 'op': 'adamw', 'bits': 32, 'sizes': 'policy', 'total': 0, 'tensors': 17,
         'grad': 'f32', 'copies': True, 'clip': 0.5},
        # 128 Mi parameters in 48 tensors, states in 32 bits
        {'name': 'adamw_128m', 'op': 'adamw', 'bits': 32, 'sizes': 'spread', 'total': 128 << 20, 'tensors': 48,
         'grad': 'f32', 'copies': False, 'clip': 0.0},
        # the same with states in 8 bits, bf16 gradients and bf16 compute copies
        {'name': 'adamw8_128m', 'op': 'adamw', 'bits': 8, 'sizes': 'spread', 'total': 128 << 20, 'tensors': 48,
         'grad': 'bf16', 'copies': True, 'clip': 0.0},
        # many small tensors of odd sizes, states in 8 bits, clipped
        {'name': 'adamw8_many', 'op': 'adamw', 'bits': 8, 'sizes': 'spread', 'total': 1_000_003, 'tensors': 300,
         'grad': 'f32', 'copies': False, 'clip': 1.0},
    ]


def _log_int(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['ln', 'lp', 'adamw'])
    if op == 'ln':
        case = {'op': 'ln', 'pass': rng.choice(['fwd', 'bwd']), 'rows': _log_int(rng, 1, 65536),
                'n': _log_int(rng, 8, 16384), 'dtype': rng.choice(['f32', 'bf16', 'f16'])}
        case['rows'] = max(1, min(case['rows'], 16384 * 4096 // case['n']))
        return case
    if op == 'lp':
        vocab = _log_int(rng, 2, 262144)
        return {'op': 'lp', 'pass': rng.choice(['fwd', 'bwd']),
                'rows': max(1, min(_log_int(rng, 1, 65536), 4096 * 40000 // vocab)), 'vocab': vocab,
                'dtype': rng.choice(['f32', 'bf16', 'f16']), 'legal': rng.random() < 0.5,
                'top': min(vocab, rng.choice([0, 0, 1, 5, 20, 32])), 'temperature': rng.choice([1.0, 0.7, 1.3])}
    bits = rng.choice([32, 8])
    # the clipped 8-bit step is drawn at small totals: its norm is summed in another order by every
    # implementation, and the last bit of the clip factor may move a scale to the next power of two
    clip = rng.choice([0.0, 0.5])
    return {'op': 'adamw', 'bits': bits, 'sizes': 'spread',
            'total': _log_int(rng, 20000, 1 << 20 if clip and bits == 8 else 96 << 20), 'tensors': _log_int(rng, 1, 200),
            'grad': rng.choice(['f32', 'bf16']), 'copies': rng.random() < 0.5, 'clip': clip}


# ---------------------------------------------------------------- inputs

def _sizes(case):
    """Element counts of a case's parameter tensors: the weight-decayed ones first, then the others."""
    if case['sizes'] == 'policy':  # conv 10-32-64-64, FC 3136-512, head 512-80, target head 64-9
        decayed = [32 * 90, 64 * 288, 64 * 576, 512 * 3136, 80 * 512, 2 * 16, 64 * 16, 9 * 64]
        return decayed, [32, 64, 64, 512, 80, 9, 512, 512, 28]
    total, count = case['total'], case['tensors']
    weights = [1 + (i * 7919) % 23 for i in range(count)]
    sizes = [max(1, total * w // sum(weights)) for w in weights]
    if count > 4:  # every fourth tensor is a vector: its elements go to the first tensor
        for i in range(3, count, 4):
            n = min(sizes[i], 1 + (i * 131) % 4099)
            sizes[0] += sizes[i] - n
            sizes[i] = n
    sizes[0] += max(0, total - sum(sizes))
    plain = sizes[3::4] if count > 4 else []
    return [s for i, s in enumerate(sizes) if count <= 4 or i % 4 != 3], plain


def _package():
    root = str(pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200')
    if root not in sys.path:
        sys.path.insert(0, root)


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, device='cuda', generator=g, dtype=torch.float32).mul_(scale).to(dtype)


def _prepare_ln(case, seed):
    g, rows, n, dtype = _generator(seed), case['rows'], case['n'], DTYPES[case['dtype']]
    s = {'x': (_randn(g, rows, n) + 0.5 * _randn(g, rows, 1)).to(dtype), 'weight': 1 + _randn(g, n, scale=0.1),
         'bias': _randn(g, n, scale=0.1)}
    if case['pass'] == 'bwd':
        x = s['x'].float()
        s['mean'] = x.mean(1)
        s['rstd'] = (x.var(1, correction=0) + EPS).rsqrt()
        s['dy'] = _randn(g, rows, n, dtype=dtype, scale=0.1)
    return s


def _prepare_lp(case, seed):
    g, rows, vocab, dtype = _generator(seed), case['rows'], case['vocab'], DTYPES[case['dtype']]
    s = {'logits': _randn(g, rows, vocab, scale=2.5).to(dtype), 'legal': None, 'top': case['top'],
         'temperature': case['temperature'], 'tokens': torch.randint(0, vocab, (rows,), device='cuda', generator=g)}
    row = torch.arange(rows, device='cuda')
    if case['legal']:  # three bits of four; one row of 61 has nothing left; most rows keep their token
        bits = torch.randint(0, 256, (rows, (vocab + 7) // 8), device='cuda', generator=g, dtype=torch.uint8)
        bits |= torch.randint(0, 256, bits.shape, device='cuda', generator=g, dtype=torch.uint8)
        at = (row, s['tokens'] // 8)
        kept = bits[at] | (1 << (s['tokens'] % 8)).to(torch.uint8)
        bits[at] = torch.where(row % 13 != 5, kept, bits[at])
        bits[row % 61 == 60] = 0
        s['legal'] = bits
    s['tokens'] = torch.where(row % 17 == 16, -1, s['tokens'])  # rows without a token (padding)
    if case['pass'] == 'bwd':
        f = _lp_forward(dict(s, top=0))
        s['stats'], s['entropy'] = f['stats'], f['entropy']
        s['dlogp'], s['dentropy'] = _randn(g, rows, scale=1.0 / rows), _randn(g, rows, scale=0.01 / rows)
    return s


def _prepare_adamw(case, seed):
    g, (decayed, plain) = _generator(seed), _sizes(case)
    padded = [(n + BLOCK - 1) // BLOCK * BLOCK for n in decayed + plain]  # every tensor starts a block
    offsets = [sum(padded[:i]) for i in range(len(padded))]
    at, split = sum(padded), sum(padded[:len(decayed)])
    pad = torch.ones(at, dtype=torch.bool, device='cuda')
    for o, n in zip(offsets, decayed + plain):
        pad[o:o + n] = False
    s = {'bits': case['bits'], 'clip': case['clip'], 'split': split, 'seed': 7}
    # gradients differ by a factor from block to block, as the layers' do
    level = torch.exp(_randn(g, at // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-3
    s['param'] = _randn(g, at, scale=0.05).masked_fill_(pad, 0)
    s['grad'] = (_randn(g, at) * level).masked_fill_(pad, 0).to(DTYPES[case['grad']])
    m = (_randn(g, at, scale=0.3) * level).masked_fill_(pad, 0)
    v = (torch.rand(at, device='cuda', generator=g).add_(0.5) * level * level).masked_fill_(pad, 0)
    del level
    if case['bits'] == 8:
        s['m_scale'] = torch.exp2(torch.floor(torch.log2(m.view(-1, BLOCK).abs().amax(1).clamp(min=1e-30))) - 7)
        s['v_scale'] = torch.exp2(torch.floor(torch.log2(v.view(-1, BLOCK).amax(1).clamp(min=1e-30))) - 14)
        s['m'] = (m.view(-1, BLOCK) / s['m_scale'][:, None]).to(torch.float8_e4m3fn).view(-1)
        s['v'] = (v.view(-1, BLOCK) / s['v_scale'][:, None]).to(torch.float8_e5m2).view(-1)
    else:
        s['m'], s['v'] = m, v
    s['copy'] = s['param'].to(torch.bfloat16) if case['copies'] else None
    s['steps'], s['places'] = AGE, list(zip(offsets, decayed + plain))
    s['decay'] = [DECAY] * len(decayed) + [0.0] * len(plain)
    return s


def _adamw_handle(s):
    """The optimizer object that a program keeps, over the same parameters, gradients and state."""
    _package()
    from d1.adamw import AdamW

    def views(t):
        return [t[o:o + n] for o, n in s['places']]

    s['opt'] = AdamW(views(s['param']), views(s['grad']), lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=s['decay'],
                     state_bits=s['bits'], max_norm=s['clip'], copies=None if s['copy'] is None else views(s['copy']),
                     seed=s['seed'])
    state = {k: s[k] for k in ('m', 'v', 'm_scale', 'v_scale') if k in s}
    s['opt'].load_state_dict(dict(state, step=AGE))
    for k in state:
        s[k] = getattr(s['opt'], k)


def _inputs(case, seed):
    s = {'ln': _prepare_ln, 'lp': _prepare_lp, 'adamw': _prepare_adamw}[case['op']](case, seed)
    s['op'], s['pass'] = case['op'], case.get('pass')
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and s['op'] == 'adamw':
        _adamw_handle(s)
    return s


# ---------------------------------------------------------------- plain forms, in 32 bits

def _ln_forward(s):
    x = s['x'].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    y = c * rstd * s['weight'] + s['bias']
    return {'y': y.to(s['x'].dtype), 'mean': mean[:, 0], 'rstd': rstd[:, 0]}


def _ln_backward(s):
    dy = s['dy'].float()
    xhat = (s['x'].float() - s['mean'][:, None]) * s['rstd'][:, None]
    g = dy * s['weight']
    dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s['rstd'][:, None]
    return {'dx': dx.to(s['x'].dtype), 'dweight': (dy * xhat).sum(0), 'dbias': dy.sum(0)}


def _masked(s):
    """The logits in 32 bits, -inf where a legal bit is clear."""
    x = s['logits'].float()
    if s['legal'] is not None:
        i = torch.arange(x.shape[1], device=x.device)
        bit = (s['legal'][:, i >> 3] >> (i & 7).to(torch.uint8)) & 1
        x = x.masked_fill(bit == 0, -math.inf)
    return x


def _token_column(s, vocab):
    """(has a token, its index or 0) of every row."""
    has = s['tokens'] >= 0
    return has, torch.where(has, s['tokens'], 0)[:, None]


def _lp_forward(s):
    x = _masked(s)
    top_of = x.amax(1)
    empty = top_of == -math.inf
    z = (x - torch.where(empty, 0.0, top_of)[:, None]) * (1.0 / s['temperature'])
    e = torch.exp(z)
    total = e.sum(1)
    log_sum = torch.log(total)
    entropy = log_sum - (e * z.masked_fill(z == -math.inf, 0)).sum(1) / total
    has, col = _token_column(s, x.shape[1])
    logp = torch.where(empty, -math.inf, z.gather(1, col)[:, 0] - log_sum)
    out = {'logp': torch.where(has, logp, 0.0), 'entropy': torch.where(empty, 0.0, entropy),
           'stats': torch.stack((top_of, log_sum), 1)}
    if s['top']:
        # one 64-bit key per token: its logit in whole-number order, then the lower index first
        key = (x + 0.0).view(torch.int32)
        key = torch.where(key < 0, key ^ 0x7fffffff, key).to(torch.int64) << 32
        key -= torch.arange(x.shape[1], device=x.device)
        top = key.topk(s['top'], 1).indices
        value = z.gather(1, top)
        none = value == -math.inf
        out['top_tokens'] = torch.where(none | empty[:, None], -1, top)
        out['top_logp'] = torch.where(none | empty[:, None], -math.inf, value - log_sum[:, None])
    return out


def _lp_backward(s):
    x = _masked(s)
    top_of, log_sum = s['stats'][:, :1], s['stats'][:, 1:]
    empty = top_of == -math.inf
    logp = (x - torch.where(empty, 0.0, top_of)) * (1.0 / s['temperature']) - torch.where(empty, 0.0, log_sum)
    p = torch.exp(logp)
    has, col = _token_column(s, x.shape[1])
    alive = has & ~empty[:, 0] & (logp.gather(1, col)[:, 0] > -math.inf)
    a = torch.where(alive, s['dlogp'], 0.0)[:, None]
    b = s['dentropy'][:, None]
    d = -p * (a + b * (logp.masked_fill(logp == -math.inf, 0) + s['entropy'][:, None]))
    d.scatter_add_(1, col, a)
    return {'dlogits': (d * (1.0 / s['temperature'])).masked_fill(empty, 0).to(s['logits'].dtype)}


def _mix(z):
    """The splitmix64 output function of a 64-bit tensor (products wrap; shifts are logical)."""
    z = z + -7046029254386353131
    z = (z ^ ((z >> 30) & 0x3ffffffff)) * -4658895280553007687
    z = (z ^ ((z >> 27) & 0x1fffffffff)) * -7723592293110705685
    return z ^ ((z >> 31) & 0x1ffffffff)


def _dither(n, seed, step, device):
    """16 random bits for each of n elements (n a multiple of 4), from the optimizer's seed and step: a 64-bit
    word per four elements, its lowest 16 bits for the first."""
    start = _mix(_mix(torch.tensor(seed, dtype=torch.int64, device=device)) + step)
    word = _mix(start + torch.arange(n // 4, device=device))
    return torch.stack([(word >> k) & 0xffff for k in (0, 16, 32, 48)], 1).view(-1).to(torch.int32)


def _scale_of(top, field):
    """Powers of two that bring each block's largest magnitude to [2^field, 2^(field + 1))."""
    e = torch.clamp((top.view(torch.int32) >> 23) - 127, min=-100)
    return ((e - field + 127) << 23).view(torch.float32), ((field - e + 127) << 23).view(torch.float32)


def _to_8_bits(x, dither, field, bias, drop):
    """(codes, scales): x >= 0 in blocks, rounded up with the probability of its distance (the dither's) to an
    8-bit float that keeps 23 - drop mantissa bits."""
    scale, inverse = _scale_of(x.amax(1), field)
    y = (x * inverse[:, None]) * 2.0 ** (bias - 127)
    low = (dither << (drop - 16)) + (1 << (drop - 17))
    return (y.view(torch.int32) + low) >> drop, scale


def _adamw(s):
    s['steps'] += 1
    (b1, b2), t, p = BETAS, s['steps'], s['param']
    g = s['grad'].float()
    if s['clip']:
        norm = torch.sqrt((g * g).sum())
        g = g * torch.clamp(s['clip'] / (norm + 1e-6), max=1.0)
    if s['bits'] == 8:
        m = (s['m'].float().view(-1, BLOCK) * s['m_scale'][:, None]).view(-1)
        v = (s['v'].float().view(-1, BLOCK) * s['v_scale'][:, None]).view(-1)
    else:
        m, v = s['m'], s['v']
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    if s['bits'] == 8:
        d = _dither(m.numel(), s['seed'], t, m.device).view(-1, BLOCK)
        code, s['m_scale'] = _to_8_bits(m.abs().view(-1, BLOCK), d, 7, 7, 20)
        code |= (m.view(-1, BLOCK) < 0).to(torch.int32) << 7
        s['m'] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)
        code, s['v_scale'] = _to_8_bits(v.view(-1, BLOCK), d, 14, 15, 21)
        code = torch.maximum(code, (v.view(-1, BLOCK) > 0).to(torch.int32))  # never a zero in place of a small v
        s['v'] = code.to(torch.uint8).view(torch.float8_e5m2).view(-1)
    else:
        s['m'], s['v'] = m, v
    p[:s['split']] *= 1 - LR * DECAY
    denom = torch.sqrt(v) / math.sqrt(1 - b2 ** t) + ADAM_EPS
    p -= (LR / (1 - b1 ** t)) * (m / denom)
    if s['copy'] is not None:
        s['copy'].copy_(p)
    return _adamw_out(s)


def _adamw_out(s):
    return {k: s[k] for k in ('param', 'm', 'v', 'm_scale', 'v_scale', 'copy') if s.get(k) is not None}


def run(s):
    if own:
        return _run_own(s)
    if s['op'] == 'ln':
        return _ln_forward(s) if s['pass'] == 'fwd' else _ln_backward(s)
    if s['op'] == 'lp':
        return _lp_forward(s) if s['pass'] == 'fwd' else _lp_backward(s)
    return _adamw(s)


def _run_own(s):
    _package()
    if s['op'] == 'ln':
        from d1.layer_norm import layer_norm, layer_norm_backward
        if s['pass'] == 'fwd':
            y, mean, rstd = layer_norm(s['x'], s['weight'], s['bias'], eps=EPS)
            return {'y': y, 'mean': mean, 'rstd': rstd}
        dx, dweight, dbias = layer_norm_backward(s['dy'], s['x'], s['mean'], s['rstd'], s['weight'])
        return {'dx': dx, 'dweight': dweight, 'dbias': dbias}
    if s['op'] == 'lp':
        from d1.token_logprob import token_logprob, token_logprob_backward
        if s['pass'] == 'fwd':
            r = token_logprob(s['logits'], s['tokens'], legal=s['legal'], temperature=s['temperature'], top=s['top'])
            out = {'logp': r.logp, 'entropy': r.entropy, 'stats': r.stats}
            return dict(out, top_tokens=r.top_tokens, top_logp=r.top_logp) if s['top'] else out
        return {'dlogits': token_logprob_backward(s['logits'], s['tokens'], s['stats'], s['entropy'], s['dlogp'],
                                                  s['dentropy'], legal=s['legal'], temperature=s['temperature'])}
    s['opt'].step()
    return _adamw_out(s)


# ---------------------------------------------------------------- the definitions, in 64 bits

def _exact_ln(case, s):
    x, w, b = s['x'].double(), s['weight'].double(), s['bias'].double()
    if case['pass'] == 'fwd':
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS) ** -0.5
        return {'y': w * (x - mean[:, None]) * rstd[:, None] + b, 'mean': mean, 'rstd': rstd}
    dy, n = s['dy'].double(), case['n']
    mean, rstd = s['mean'].double()[:, None], s['rstd'].double()[:, None]
    dxhat = dy * w
    c = x - mean
    inner = (dxhat * c).sum(1, keepdim=True) * rstd ** 3 / n
    return {'dx': dxhat * rstd - (dxhat.sum(1, keepdim=True) / n) * rstd - c * inner,
            'dweight': torch.einsum('rn,rn,r->n', dy, c, rstd[:, 0]), 'dbias': torch.einsum('rn->n', dy)}


def _exact_lp(case, s):
    rows, vocab = s['logits'].shape
    x = s['logits'].double()
    if s['legal'] is not None:
        bits = torch.stack([s['legal'].bitwise_right_shift(k) % 2 for k in range(8)], 2).view(rows, -1)[:, :vocab]
        x[bits == 0] = -math.inf
        del bits
    top_of = x.max(1).values
    dead = torch.isinf(top_of)
    x -= torch.where(dead, torch.zeros_like(top_of), top_of)[:, None]
    x /= s['temperature']
    log_sum = torch.logsumexp(x, 1)
    x -= torch.where(dead, torch.zeros_like(log_sum), log_sum)[:, None]
    rows_with = (s['tokens'] >= 0).nonzero()[:, 0]
    at = s['tokens'][rows_with]
    p = x.exp()
    surprise = torch.where(p > 0, -p * x, torch.zeros_like(p))
    entropy = surprise.sum(1)
    del surprise
    if case['pass'] == 'fwd':
        logp = torch.zeros(rows, dtype=torch.float64, device=x.device)
        logp[rows_with] = x[rows_with, at]
        out = {'logp': logp, 'entropy': entropy, 'stats': torch.stack((top_of, log_sum), 1)}
        if case['top']:
            best = x.topk(case['top'], 1).values
            out.update(top_tokens=None, top_logp=best)
        return out
    a = torch.zeros(rows, dtype=torch.float64, device=x.device)
    a[rows_with] = torch.where(torch.isinf(x[rows_with, at]), 0.0, s['dlogp'].double()[rows_with])
    b = s['dentropy'].double()
    d = p * (-a - b * entropy)[:, None]
    x.masked_fill_(p == 0, 0)
    d -= p * x * b[:, None]
    d[rows_with, at] += a[rows_with]
    d[dead] = 0
    return {'dlogits': d / s['temperature']}


def _exact_adamw(case, s):
    (b1, b2), t = BETAS, AGE + 1
    g = s['grad'].double()
    if case['clip']:
        g = g * min(1.0, case['clip'] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    m, v = s['m'].double(), s['v'].double()
    if case['bits'] == 8:
        m = m * s['m_scale'].double().repeat_interleave(BLOCK)
        v = v * s['v_scale'].double().repeat_interleave(BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    decay = torch.ones(g.numel(), dtype=torch.float64, device=g.device)
    decay[:s['split']] = 1 - LR * DECAY
    p = s['param'].double() * decay - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + ADAM_EPS)
    out = {'param': p, 'm': m, 'v': v}
    if case['bits'] == 8:
        d = (_dither(g.numel(), s['seed'], t, g.device).double() + 0.5) / 65536
        for name, x, field, mantissa, lowest in (('m', m, 7, 3, -6), ('v', v, 14, 2, -14)):
            top = x.abs().view(-1, BLOCK).amax(1)
            exponent = torch.frexp(top)[1].double() - 1
            exponent = torch.where(top == 0, -100.0, exponent).clamp(min=-100)
            out[name + '_scale'] = torch.exp2(exponent - field)
            y = x.abs() / out[name + '_scale'].repeat_interleave(BLOCK)
            spacing = torch.exp2((torch.frexp(y)[1].double() - 1).clamp(min=lowest) - mantissa)
            q = torch.floor(y / spacing + d) * spacing
            if name == 'v':
                q = torch.where(y > 0, q.clamp(min=2.0 ** -16), q)
            out[name] = q * torch.sign(x)
    if s['copy'] is not None:
        out['copy'] = p
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {'ln': _exact_ln, 'lp': _exact_lp, 'adamw': _exact_adamw}[case['op']](case, s)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case['op'] == 'ln':
        size, e = case['rows'] * case['n'], BYTES[case['dtype']]
        if case['pass'] == 'fwd':  # x in, y out; weight and bias in; mean and rstd out
            return {'bytes': 2 * size * e + 8 * case['n'] + 8 * case['rows'], 'flops': 7 * size}
        # x and dy in, dx out; weight in, both gradients out; mean and rstd in
        return {'bytes': 3 * size * e + 12 * case['n'] + 8 * case['rows'], 'flops': 12 * size}
    if case['op'] == 'lp':
        rows, size = case['rows'], case['rows'] * case['vocab']
        once = size * BYTES[case['dtype']] + (rows * ((case['vocab'] + 7) // 8) if case['legal'] else 0)
        if case['pass'] == 'fwd':  # logits and bits in; token in; logp, entropy and stats out; alternatives out
            return {'bytes': once + rows * (8 + 16 + 12 * case['top']), 'flops': 5 * size}
        return {'bytes': once + size * BYTES[case['dtype']] + rows * (8 + 20), 'flops': 7 * size}
    n = sum(a for part in _sizes(case) for a in part)
    state = 16 if case['bits'] == 32 else 4 + 16 / BLOCK  # both moments (and their scales), read and written
    return {'bytes': n * (8 + state + BYTES[case['grad']] + (2 if case['copies'] else 0)), 'flops': 16 * n}
