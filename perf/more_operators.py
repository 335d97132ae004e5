"""Cases, plain forms and 64-bit values of the operators that train a policy with a memory by reinforcement:
a gated linear recurrence over rollouts and long sequences (forward, one step, backward), the clipped policy
loss with KL and entropy terms and its gradient, and Muon (momentum, Newton-Schulz orthogonalisation, update).

A case is a dict of plain values; prepare() makes its inputs on the GPU from a seed, run() makes one call of the
operator (with `own`, through the package; else in elementary torch operations in 32 bits), exact() computes the
same outputs in 64 bits, and work() counts the bytes and operations no implementation can do without.
"""
import functools
import math
import pathlib
import sys
import types

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
LOW, HIGH, KL, ENT = 0.2, 0.28, 0.05, 0.01          # the policy loss's clip range and coefficients
LR, MOMENTUM, DECAY = 3e-4, 0.95, 0.01
PAD = 128                                           # elements between which Muon's tensors start
STEPS, NS = 5, (3.4445, -4.7750, 2.0315)            # Newton-Schulz steps and the quintic's coefficients
MAX_SCAN, MAX_TOKENS, MAX_FLOPS = 128 * 4096 * 512, 128 * 65536, 5e12


def listed():
    return [
        # one decision of 64 environments with 256 channels of memory: latency
        {'name': 'scan_step', 'op': 'scan', 'pass': 'fwd', 'T': 1, 'B': 64, 'D': 256, 'dtype': 'bf16',
         'form': 'average', 'reset': True},
        # a rollout of 128 steps by 4,096 environments, 512 channels, episodes ending inside it
        {'name': 'scan_fwd_rollout', 'op': 'scan', 'pass': 'fwd', 'T': 128, 'B': 4096, 'D': 512, 'dtype': 'bf16',
         'form': 'average', 'reset': True},
        # the gradient over a rollout of 64 steps
        {'name': 'scan_bwd_rollout', 'op': 'scan', 'pass': 'bwd', 'T': 64, 'B': 4096, 'D': 512, 'dtype': 'bf16',
         'form': 'average', 'reset': True},
        # one long sequence of few channels
        {'name': 'scan_fwd_long', 'op': 'scan', 'pass': 'fwd', 'T': 131072, 'B': 1, 'D': 256, 'dtype': 'bf16',
         'form': 'average', 'reset': False},
        # odd sizes, in 32 bits: three long sequences whose decay is given by its logarithm
        {'name': 'scan_bwd_odd', 'op': 'scan', 'pass': 'bwd', 'T': 50021, 'B': 3, 'D': 111, 'dtype': 'f32',
         'form': 'sum', 'reset': True},
        # a PPO minibatch of 16,384 decisions with the entropy term
        {'name': 'loss_minibatch', 'op': 'loss', 'rows': 1, 'length': 16384, 'per_row': False, 'ref': False,
         'entropy': True, 'mask': False, 'mean': 'token'},
        # sequences of odd length, an advantage for each, a KL term, padding, every sequence counting the same
        {'name': 'loss_sequences', 'op': 'loss', 'rows': 512, 'length': 4099, 'per_row': True, 'ref': True,
         'entropy': False, 'mask': True, 'mean': 'row'},
        # a whole rollout of 128 steps by 65,536 environments with every term
        {'name': 'loss_rollout', 'op': 'loss', 'rows': 128, 'length': 65536, 'per_row': False, 'ref': True,
         'entropy': True, 'mask': True, 'mean': 'token'},
        # the weight matrices of the conv policy with a memory of 512 channels, with bf16 copies: latency
        {'name': 'muon_policy', 'op': 'muon', 'sizes': 'policy', 'grad': 'f32', 'copies': True},
        # twelve layers of four square, one tall and one wide matrix, bf16 gradients
        {'name': 'muon_layers', 'op': 'muon', 'sizes': 'layers', 'layers': 12, 'width': 1024, 'grad': 'bf16',
         'copies': True},
        # one large square matrix
        {'name': 'ortho_square', 'op': 'ortho', 'batch': 1, 'm': 8192, 'n': 8192, 'dtype': 'bf16'},
        # a stack of odd matrices, taller than wide, in 32 bits (the result has 16)
        {'name': 'ortho_odd', 'op': 'ortho', 'batch': 7, 'm': 1777, 'n': 1003, 'dtype': 'f32'},
    ]


def _log_int(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['scan', 'scan', 'loss', 'muon', 'ortho'])
    if op == 'scan':
        d = _log_int(rng, 1, 2048)
        t = _log_int(rng, 1, 131072)
        b = max(1, min(_log_int(rng, 1, 65536), MAX_SCAN // (4 * d * t)))
        return {'op': 'scan', 'pass': rng.choice(['fwd', 'bwd']), 'T': max(1, min(t, MAX_SCAN // (4 * d * b))), 'B': b,
                'D': d, 'dtype': rng.choice(['f32', 'bf16', 'f16']), 'form': rng.choice(['average', 'sum']),
                'reset': rng.random() < 0.7}
    if op == 'loss':
        length = _log_int(rng, 1, 131072)
        return {'op': 'loss', 'rows': max(1, min(_log_int(rng, 1, 65536), MAX_TOKENS // length)), 'length': length,
                'per_row': rng.random() < 0.5, 'ref': rng.random() < 0.5, 'entropy': rng.random() < 0.5,
                'mask': rng.random() < 0.7, 'mean': rng.choice(['token', 'row'])}
    if op == 'muon':
        return {'op': 'muon', 'sizes': 'spread', 'count': rng.randint(1, 8), 'm': _log_int(rng, 1, 2048),
                'n': _log_int(rng, 8, 4096), 'grad': rng.choice(['f32', 'bf16']), 'copies': rng.random() < 0.5}
    m, n = _log_int(rng, 1, 4096), _log_int(rng, 8, 8192)
    flops = _ns_flops(m, n)
    return {'op': 'ortho', 'batch': max(1, min(rng.randint(1, 16), int(MAX_FLOPS / flops))), 'm': m, 'n': n,
            'dtype': rng.choice(['f32', 'bf16', 'f16'])}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, device='cuda', generator=g, dtype=torch.float32).mul_(scale).to(dtype)


def _prepare_scan(case, seed):
    g, shape, dtype = _generator(seed), (case['T'], case['B'], case['D']), DTYPES[case['dtype']]
    average = case['form'] == 'average'
    s = {'form': case['form'], 'x': _randn(g, *shape, dtype=dtype), 'h0': _randn(g, *shape[1:])}
    # gates: time constants from a few steps to a few hundred, of each channel its own
    level = _randn(g, case['D'], scale=1.5) + 3
    gate = _randn(g, *shape)
    s['gate'] = (gate.add_(level) if average else gate.mul_(0.3).sub_(level).exp_().neg_()).to(dtype)
    del gate
    s['reset'] = torch.rand(shape[:2], device='cuda', generator=g) < 1 / 64 if case['reset'] else None
    if case['pass'] == 'bwd':
        s['y'] = _scan_forward(s)['y']
        s['dy'], s['dlast'] = _randn(g, *shape, dtype=dtype, scale=0.1), _randn(g, *shape[1:], scale=0.1)
    return s


def _prepare_loss(case, seed):
    g, shape = _generator(seed), (case['rows'], case['length'])
    s = {'old_logp': -_randn(g, *shape).abs_(), 'ref_logp': None, 'entropy': None, 'mask': None, 'mean': case['mean']}
    # the policy has moved a little since the rollout; every eighth token has not moved
    moved = _randn(g, *shape, scale=0.15)
    moved[torch.rand(shape, device='cuda', generator=g) < 0.125] = 0
    s['logp'] = s['old_logp'] + moved
    s['advantage'] = _randn(g, *shape[:1]) if case['per_row'] else _randn(g, *shape)
    if case['ref']:
        s['ref_logp'] = s['old_logp'] + _randn(g, *shape, scale=0.2)
    if case['entropy']:
        s['entropy'] = _randn(g, *shape).abs_()
    if case['mask']:  # sequences end somewhere, some at once; what lies behind holds anything
        ends = torch.randint(0, case['length'] + 1, shape[:1], device='cuda', generator=g)
        s['mask'] = torch.arange(case['length'], device='cuda') < ends[:, None]
        s['logp'].masked_fill_(~s['mask'], -math.inf)
    return s


def _shapes(case):
    """The shapes of a Muon case's parameters."""
    if case['sizes'] == 'policy':  # conv 10-32-64-64, FC 3136-512, the memory's gate and input, the joint head
        return [(32, 90), (64, 288), (64, 576), (512, 3136), (1024, 512), (28, 512)]
    if case['sizes'] == 'layers':
        w = case['width']
        return [s for _ in range(case['layers']) for s in [(w, w)] * 4 + [(4 * w, w), (w, 4 * w)]]
    m, n = case['m'], case['n']
    some = [(m, n), (n, m), (1 + m // 2, n), (m, 1 + n // 3), (2, 3, 1 + m // 4, 1 + n // 4), (m, m), (1, n), (n, 1)]
    return some[:case['count']]


def _gradient(g, *shape):
    """A gradient as training has it: a few strong directions of different strength over noise."""
    *lead, m, n = shape
    k = max(1, min(m, n) // 8)
    strength = 1.0 / torch.arange(1, k + 1, device='cuda')
    return (_randn(g, *lead, m, k) * strength) @ _randn(g, *lead, k, n) + _randn(g, *shape, scale=0.2)


def _views(flat, shapes):
    """Tensors of these shapes in one buffer, each starting at a multiple of 128 elements."""
    sizes = [math.prod(t) for t in shapes]
    starts = [sum(-(-n // PAD) * PAD for n in sizes[:i]) for i in range(len(sizes))]
    return [flat[o:o + n].view(t) for o, n, t in zip(starts, sizes, shapes)]


def _prepare_muon(case, seed):
    g, shapes = _generator(seed), _shapes(case)
    total = sum(-(-math.prod(t) // PAD) * PAD for t in shapes)
    s = {'param': torch.zeros(total, device='cuda'), 'momentum': torch.zeros(total, device='cuda'), 'copy': None}
    s['params'], s['momenta'] = _views(s['param'], shapes), _views(s['momentum'], shapes)
    for p, m in zip(s['params'], s['momenta']):
        p.copy_(_randn(g, *p.shape, scale=0.05))
        m.copy_(_gradient(g, *p.shape)).mul_(1e-2)
    s['grads'] = [_gradient(g, *t).mul_(1e-3).to(DTYPES[case['grad']]) for t in shapes]
    if case['copies']:
        s['copy'] = s['param'].to(torch.bfloat16)
        s['copies'] = _views(s['copy'], shapes)
    return s


def _prepare_ortho(case, seed):
    return {'x': _gradient(_generator(seed), case['batch'], case['m'], case['n']).to(DTYPES[case['dtype']])}


def _inputs(case, seed):
    s = {'scan': _prepare_scan, 'loss': _prepare_loss, 'muon': _prepare_muon, 'ortho': _prepare_ortho}[case['op']](
        case, seed)
    s['op'], s['pass'] = case['op'], case.get('pass')
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and s['op'] == 'muon':  # the optimizer object that a program keeps
        s['opt'] = _package().Muon(s['params'], s['grads'], lr=LR, momentum=MOMENTUM, weight_decay=DECAY,
                                   steps=STEPS, copies=s.get('copies'))
        s['opt'].load_state_dict({'momentum': s['momentum']})
        s['momentum'] = s['opt'].momentum
    return s


# ---------------------------------------------------------------- plain forms, in 32 bits

def _decay(s):
    """(a, the input's factor) of every step, the factor None where it is 1."""
    g = s['gate'].float()
    if s['form'] == 'sum':
        return torch.exp(g), None
    e = torch.exp(-g.abs())
    small, large = e / (1 + e), 1 / (1 + e)
    return torch.where(g < 0, small, large), torch.where(g < 0, large, small)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first dimension from h = 0, in place of b, by doubling."""
    d = 1
    while d < a.shape[0]:
        b[d:] = b[d:] + a[d:] * b[:-d]
        a[d:] = a[d:] * a[:-d]
        d *= 2
    return b


def _scan_forward(s):
    a, w = _decay(s)
    b = s['x'].float() if w is None else s['x'].float() * w
    b = b.clone() if b.data_ptr() == s['x'].data_ptr() else b
    if s['reset'] is not None:
        a = a.masked_fill(s['reset'][:, :, None], 0)
    b[0] = b[0] + a[0] * s['h0']
    h = _scan(a, b)
    return {'y': h.to(s['x'].dtype), 'last': h[-1].clone()}


def _scan_backward(s):
    a, w = _decay(s)
    before = torch.cat((s['h0'][None], s['y'][:-1].float()))
    kept = a
    if s['reset'] is not None:
        before = before.masked_fill(s['reset'][:, :, None], 0)
        kept = a.masked_fill(s['reset'][:, :, None], 0)
    d = s['dy'].float().flip(0)
    d[0] = d[0] + s['dlast']
    behind = torch.cat((torch.zeros_like(kept[:1]), kept[1:].flip(0)))  # a_{t+1} for t = T-1, T-2, ..., 0
    d = _scan(behind, d).flip(0)
    dx = d if w is None else d * w
    dgate = d * before * a if w is None else d * (before - s['x'].float()) * a * w
    return {'dx': dx.to(s['x'].dtype), 'dgate': dgate.to(s['x'].dtype), 'dh0': kept[0] * d[0]}


def _weights(mask, shape, mean, dtype):
    """Every token's weight in the mean."""
    keep = torch.ones(shape, dtype=dtype, device='cuda') if mask is None else mask.to(dtype)
    if mean == 'token':
        return keep / keep.sum().clamp(min=1)
    count = keep.sum(1, keepdim=True)
    return keep / count.clamp(min=1) / (count > 0).sum().clamp(min=1)


def _loss(s):
    logp, adv = s['logp'], s['advantage']
    shape, mask = logp.shape, s['mask']
    adv = adv[:, None] if adv.dim() == 1 else adv
    out = torch.zeros(shape, dtype=torch.bool, device='cuda') if mask is None else ~mask
    w = _weights(mask, shape, s['mean'], torch.float32)
    wide = logp.double() - s['old_logp'].double()  # 64 bits: which side of the clip range a ratio lies on
    delta = wide.float().masked_fill(out, 0)
    over, under = wide > math.log1p(HIGH), wide < math.log1p(-LOW)
    clipped = ((over & (adv > 0)) | (under & (adv < 0))) & ~out
    r = torch.exp(delta)
    limit = torch.where(over, 1 + HIGH, torch.where(under, 1 - LOW, r))
    policy = -torch.where(clipped, limit, r) * adv
    dlogp = torch.where(clipped, 0.0, -adv * r)
    policy, dlogp = policy.masked_fill(out, 0), dlogp.masked_fill(out, 0)
    wide_w = w.double()  # sums over many tokens, whose terms cancel, in 64 bits
    none = torch.zeros_like(wide_w[0, 0])
    stats = [(policy * wide_w).sum(), none, none, (clipped * wide_w).sum(),
             ((torch.expm1(delta) - delta) * wide_w).sum()]
    loss = stats[0]
    if s['ref_logp'] is not None:
        d = (s['ref_logp'].double() - logp.double()).masked_fill(out, 0)  # e^d - d - 1 cancels near 0
        grown = torch.expm1(d)
        stats[1] = ((grown - d) * wide_w).sum()
        loss = loss + KL * stats[1]
        dlogp = dlogp - KL * grown.float()
    found = {'dlogp': dlogp * w}
    if s['entropy'] is not None:
        stats[2] = (s['entropy'].masked_fill(out, 0) * wide_w).sum()
        loss = loss - ENT * stats[2]
        found['dentropy'] = -ENT * w
    return dict(found, loss=loss.float(), stats=torch.stack(stats).float())


def _newton_schulz(u):
    """u's directions with singular values near 1, in 32 bits."""
    a, b, c = NS
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    norm = torch.sqrt((x * x).sum((-2, -1), keepdim=True))
    x = x / torch.where(norm > 0, norm, 1)
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _ortho(s):
    return {'y': _newton_schulz(s['x'].float()).to(_result_type(s['x'].dtype))}


def _result_type(dtype):
    return torch.bfloat16 if dtype == torch.float32 else dtype


def _muon(s):
    for p, g, m in zip(s['params'], s['grads'], s['momenta']):
        g = g.float()
        m.mul_(MOMENTUM).add_(g)
        x = _newton_schulz(g + MOMENTUM * m)
        p.mul_(1 - LR * DECAY).sub_(x * (LR * 0.2 * math.sqrt(max(p.shape[-2:]))))
    if s['copy'] is not None:
        s['copy'].copy_(s['param'])
    return _muon_out(s)


def _muon_out(s):
    return {k: s[k] for k in ('param', 'momentum', 'copy') if s[k] is not None}


def run(s):
    if own:
        return _run_own(s)
    if s['op'] == 'scan':
        return _scan_forward(s) if s['pass'] == 'fwd' else _scan_backward(s)
    return {'loss': _loss, 'muon': _muon, 'ortho': _ortho}[s['op']](s)


@functools.lru_cache(None)
def _package():
    root = str(pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200')
    if root not in sys.path:
        sys.path.insert(0, root)
    from d1.gated_scan import gated_scan, gated_scan_backward
    from d1.muon import Muon, orthogonalize
    from d1.policy_loss import policy_loss
    return types.SimpleNamespace(gated_scan=gated_scan, gated_scan_backward=gated_scan_backward, Muon=Muon,
                                 orthogonalize=orthogonalize, policy_loss=policy_loss)


def _run_own(s):
    d1 = _package()
    if s['op'] == 'scan':
        if s['pass'] == 'fwd':
            y, last = d1.gated_scan(s['x'], s['gate'], s['h0'], reset=s['reset'], form=s['form'])
            return {'y': y, 'last': last}
        dx, dgate, dh0 = d1.gated_scan_backward(s['dy'], s['x'], s['gate'], s['y'], s['h0'], reset=s['reset'],
                                                dlast=s['dlast'], form=s['form'])
        return {'dx': dx, 'dgate': dgate, 'dh0': dh0}
    if s['op'] == 'loss':
        r = d1.policy_loss(s['logp'], s['old_logp'], s['advantage'], ref_logp=s['ref_logp'], entropy=s['entropy'],
                           mask=s['mask'], clip=(LOW, HIGH), kl_coef=KL, ent_coef=ENT, mean=s['mean'])
        out = {'loss': r.loss, 'stats': r.stats, 'dlogp': r.dlogp}
        return out if r.dentropy is None else dict(out, dentropy=r.dentropy)
    if s['op'] == 'ortho':
        return {'y': d1.orthogonalize(s['x'], steps=STEPS)}
    s['opt'].step()
    return _muon_out(s)


# ---------------------------------------------------------------- the definitions, in 64 bits

def _exact_steps(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0, step by step: within 256 pieces of the time side by side, then over the pieces."""
    steps = a.shape[0]
    size = -(-steps // min(256, steps))
    pad = -steps % size
    a = torch.cat((a, a.new_ones(pad, *a.shape[1:]))).view(-1, size, *a.shape[1:])
    b = torch.cat((b, b.new_zeros(pad, *b.shape[1:]))).view(-1, size, *b.shape[1:])
    for t in range(1, size):
        b[:, t].addcmul_(a[:, t], b[:, t - 1])
    if a.shape[0] > 1:
        a = a.cumprod(1)
        for p in range(1, a.shape[0]):
            b[p].addcmul_(a[p], b[p - 1, -1])
    return b.view(-1, *b.shape[2:])[:steps]


def _exact_scan(case, s):
    g, average = s['gate'].double(), case['form'] == 'average'
    a = torch.sigmoid(g) if average else g.exp()
    keep = a if s['reset'] is None else torch.where(s['reset'][..., None], 0.0, a)
    h0 = s['h0'].double()
    if case['pass'] == 'fwd':
        b = s['x'].double()
        if average:
            b *= torch.sigmoid(-g)
        del g, a
        b[0] += keep[0] * h0
        h = _exact_steps(keep, b)
        return {'y': h, 'last': h[-1]}
    d = s['dy'].double()
    d[-1] += s['dlast'].double()
    later = torch.cat((keep[1:], torch.zeros_like(keep[:1])))
    d = _exact_steps(later.flip(0), d.flip(0)).flip(0)
    del later
    dh0 = keep[0] * d[0]
    del keep
    h = torch.cat((h0[None], s['y'][:-1].double()))
    if s['reset'] is not None:
        h[s['reset']] = 0
    if average:
        h -= s['x'].double()
        dx = d * torch.sigmoid(-g)
        return {'dx': dx, 'dgate': h.mul_(dx).mul_(a), 'dh0': dh0}
    return {'dx': d, 'dgate': h.mul_(d).mul_(a), 'dh0': dh0}


def _exact_loss(case, s):
    logp, old = s['logp'].double(), s['old_logp'].double()
    adv = s['advantage'].double()
    adv = adv.unsqueeze(1).expand_as(logp) if case['per_row'] else adv
    m = torch.ones_like(logp) if s['mask'] is None else s['mask'].double()
    if case['mean'] == 'token':
        w = m / max(1.0, float(m.sum()))
    else:
        lengths = m.sum(1)
        w = m / lengths.clamp(min=1)[:, None] / max(1, int((lengths > 0).sum()))
    at = w > 0
    logp, old, adv, w = logp[at], old[at], adv[at], w[at]
    ratio = (logp - old).exp()
    plain, bounded = ratio * adv, ratio.clamp(1 - LOW, 1 + HIGH) * adv
    cut = bounded < plain
    terms = [torch.dot(w, -torch.minimum(plain, bounded)), w.new_zeros(()), w.new_zeros(()), w[cut].sum(),
             torch.dot(w, ratio - 1 - ratio.log())]
    d = torch.where(cut, 0.0, -plain)
    if s['ref_logp'] is not None:
        away = s['ref_logp'].double()[at] - logp
        terms[1] = torch.dot(w, torch.expm1(away) - away)
        d = d + KL * (1 - away.exp())
    if s['entropy'] is not None:
        terms[2] = torch.dot(w, s['entropy'].double()[at])
    dlogp = torch.zeros_like(m)
    dlogp[at] = d * w
    out = {'loss': terms[0] + KL * terms[1] - ENT * terms[2], 'stats': torch.stack(terms), 'dlogp': dlogp}
    if s['entropy'] is not None:
        out['dentropy'] = torch.zeros_like(m).masked_scatter_(at, -ENT * w)
    return out


def _exact_polar(u):
    """The same polynomial of u's singular values, on the smaller side's Gram matrix."""
    a, b, c = NS
    x = u.double()
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=1e-300)
    one = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        wide = x.shape[-2] <= x.shape[-1]
        gram = torch.matmul(x, x.transpose(-1, -2)) if wide else torch.matmul(x.transpose(-1, -2), x)
        factor = a * one + torch.matmul(gram, b * one + c * gram)
        x = torch.matmul(factor, x) if wide else torch.matmul(x, factor)
    return x


def _exact_muon(case, s):
    out = {'param': torch.zeros_like(s['param'], dtype=torch.float64)}
    out['momentum'] = torch.zeros_like(out['param'])
    for p, m, g, p0, m0 in zip(*(_views(out[k], _shapes(case)) for k in ('param', 'momentum')), s['grads'], s['params'],
                               s['momenta']):
        m.copy_(MOMENTUM * m0.double() + g.double())
        x = _exact_polar(MOMENTUM * m + g.double())
        p.copy_(p0.double() * (1 - LR * DECAY) - 0.2 * LR * max(p.shape[-2:]) ** 0.5 * x)
    return dict(out, copy=out['param']) if case['copies'] else out


def exact(case, seed):
    s = _inputs(case, seed)
    if case['op'] == 'ortho':
        return {'y': _exact_polar(s['x'])}
    return {'scan': _exact_scan, 'loss': _exact_loss, 'muon': _exact_muon}[case['op']](case, s)


# ---------------------------------------------------------------- what a pass cannot do without

def _ns_flops(m, n):
    """Of one matrix: half of the two symmetric products, all of the third."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    if case['op'] == 'scan':
        size, e, lanes = case['T'] * case['B'] * case['D'], BYTES[case['dtype']], case['B'] * case['D']
        flags = case['T'] * case['B'] if case['reset'] else 0
        if case['pass'] == 'fwd':  # x and gate in, y out; the first state in, the last out
            return {'bytes': 3 * size * e + 8 * lanes + flags, 'flops': 8 * size}
        # dy, x (where the input has a factor), gate and y in, dx and dgate out; h0 and dlast in, dh0 out
        return {'bytes': (6 if case['form'] == 'average' else 5) * size * e + 12 * lanes + flags, 'flops': 14 * size}
    if case['op'] == 'loss':
        size = case['rows'] * case['length']
        each = 12 + (0 if case['per_row'] else 4) + 4 * case['ref'] + 8 * case['entropy'] + case['mask']
        return {'bytes': size * each + (4 * case['rows'] if case['per_row'] else 0) + 24, 'flops': 20 * size}
    if case['op'] == 'ortho':
        size = case['batch'] * case['m'] * case['n']
        return {'bytes': size * (BYTES[case['dtype']] + 2), 'flops': case['batch'] * _ns_flops(case['m'], case['n'])}
    total = flops = 0
    for *lead, m, n in _shapes(case):
        total += math.prod(lead) * m * n
        flops += math.prod(lead) * _ns_flops(m, n)
    # parameter and momentum in and out, the gradient in, the copy out
    return {'bytes': total * (16 + BYTES[case['grad']] + (2 if case['copies'] else 0)), 'flops': flops}
