"""The recurrent joint-action head (d1.recurrent): GEMMs, gated recurrence, layer norm, log-probabilities, policy
loss, Muon and AdamW together, on features of the conv policy and its own draws."""
import pytest
import torch

pytestmark = pytest.mark.gpu
T, N = 6, 640


@pytest.fixture(scope='module')
def rollout():
    """Features of T steps of the conv policy's environments, with the head's own actions."""
    from d1.conv_policy import ENV_ACTION, ConvPolicy
    from d1.recurrent import RecurrentHead
    from d1.spec_env import SpecEnv
    env, pol, head = SpecEnv(N, seed=3, observe=False), ConvPolicy(seed=1, chunk=N), RecurrentHead(seed=2)
    buf, g = pol.buffers(N), torch.Generator(device='cuda').manual_seed(4)
    to_env = torch.tensor(ENV_ACTION, device='cuda')
    state, reset = head.state(N), torch.zeros(N, dtype=torch.bool, device='cuda')
    first, rows = state, []
    for _ in range(T):
        pol.encode(env.state, N, buf)
        pol.features(buf, N)
        joint, logp, state = head.act(buf['h'], env.legal, state, reset=reset, generator=g)
        rows.append((buf['h'].clone(), joint, env.legal.clone(), logp, reset))
        near = (env.legal.to(torch.int32) >> 10) & 1 == 1
        env.step(torch.where((joint == 17) & near, 10, to_env[joint]))
        reset = torch.rand(N, device='cuda', generator=g) < 0.1
    h, joint, legal, logp, reset = (torch.stack(v) for v in zip(*rows))
    adv = torch.randn(T, N, device='cuda', generator=g)
    live = torch.rand(T, N, device='cuda', generator=g) < 0.9
    return dict(h=h, joint=joint, legal=legal, logp=logp, reset=reset, adv=adv, live=live, first=first, last=state)


def test_actions_are_legal(rollout):
    from d1.imitation import joint_legal
    bits = joint_legal(rollout['legal'].view(-1))
    assert ((bits >> rollout['joint'].view(-1).to(torch.int32)) & 1 == 1).all()


def test_the_rollout_again(rollout):
    """The same memory and log-probabilities over all steps at once as one decision after the other: the same operators on
    the same rows, whose sums do not depend on the rows beside them."""
    from d1.imitation import joint_legal
    from d1.recurrent import RecurrentHead
    from d1.token_logprob import token_logprob
    head = RecurrentHead(seed=2)
    logits, last, _ = head.forward(rollout['h'], rollout['first'], rollout['reset'])
    r = token_logprob(logits, rollout['joint'].view(-1), legal=joint_legal(rollout['legal'].view(-1)))
    assert (r.logp.view(T, N) - rollout['logp']).abs().max() <= 1e-5
    assert (last - rollout['last']).abs().max() <= 1e-5


def test_gradients_against_autograd(rollout):
    """Against torch's autograd in fp32 on the same bf16 operands; the kernels round the projections, states, normed states,
    logits and all of their gradients to bf16 (2^-9 each, of sums of terms of both signs): 3e-2 of each gradient's norm."""
    from d1.imitation import JOINT, joint_legal
    from d1.policy_loss import policy_loss
    from d1.recurrent import RecurrentHead
    from d1.token_logprob import token_logprob
    head, s = RecurrentHead(seed=2, ent_coef=0.05), rollout
    old = s['logp'] + 0.05 * torch.randn(T, N, device='cuda', generator=torch.Generator(device='cuda').manual_seed(9))
    logits, _, saved = head.forward(s['h'], s['first'] + 0.1, s['reset'])
    bits, flat = joint_legal(s['legal'].view(-1)), s['joint'].view(-1)
    r = token_logprob(logits, flat, legal=bits)
    loss = policy_loss(r.logp.view(T, N), old, s['adv'], entropy=r.entropy.view(T, N), mask=s['live'], clip=0.2, ent_coef=0.05)
    dh, dstate = head.backward(logits, flat, bits, r, loss, saved)
    p = {k: t.clone().requires_grad_() for k, t in head.params.items()}
    x, first = s['h'].float().requires_grad_(), (s['first'] + 0.1).requires_grad_()
    exact = {k: p[k] + (head.w[k].float() - p[k]).detach() for k in ('in', 'out')}
    proj = x @ exact['in'].view(-1, 512).T + p['in_b']
    a, hs, state = torch.sigmoid(proj[..., :256]), [], first
    for t in range(T):
        state = torch.where(s['reset'][t][:, None], 0.0, state)
        state = a[t] * state + (1 - a[t]) * proj[t, :, 256:]
        hs.append(state)
    z = torch.nn.functional.layer_norm(torch.stack(hs), (256,), p['norm_w'], p['norm_b'])
    lg = (z @ exact['out'].T + p['out_b'])[..., :JOINT].reshape(-1, JOINT)
    on = (bits[:, None] >> torch.arange(JOINT, device='cuda', dtype=torch.int32)) & 1 == 1
    lp = lg.masked_fill(~on, -1e9).log_softmax(1)
    ent = -(lp.exp() * lp).sum(1).view(T, N)
    took = lp.gather(1, flat[:, None])[:, 0].view(T, N)
    ratio = (took - old).exp()
    # the clipped tokens are the kernel's: a ratio next to a border may lie on its other side here
    cut = (loss.dlogp == 0) & s['live']
    each = torch.where(cut, 0.0, -ratio * s['adv']) - 0.05 * ent
    (each * s['live']).sum().div(s['live'].sum()).backward()
    assert (r.logp.view(T, N) - took).abs().max() < 0.05
    for k in p:
        assert (head.grads[k] - p[k].grad).norm() <= 3e-2 * p[k].grad.norm(), k
    assert (dh.float() - x.grad).norm() <= 3e-2 * x.grad.norm()
    assert (dstate - first.grad).norm() <= 3e-2 * first.grad.norm()


def test_update_moves_every_parameter(rollout):
    from d1.muon import muon_error
    from d1.recurrent import RecurrentHead
    head, s = RecurrentHead(seed=2, kl_coef=0.1), rollout
    before = {k: p.clone() for k, p in head.params.items()}
    for _ in range(3):
        loss = head.update(s['h'], s['joint'], s['legal'], s['logp'], s['adv'], s['first'], s['reset'], s['live'], ref_logp=s['logp'])
    assert torch.isfinite(loss.loss) and torch.isfinite(loss.stats).all() and muon_error() == 0
    for k, p in head.params.items():
        assert torch.isfinite(p).all() and not torch.equal(p, before[k]), k
        if k in head.w:
            assert torch.equal(head.w[k], p.to(torch.bfloat16))
    assert (head.params['out'][28:] == 0).all()


def test_update_as_a_graph(rollout):
    """An update captured into a CUDA graph, with its optimizers, goes on as the eager ones do."""
    from d1.recurrent import RecurrentHead
    s, heads = rollout, [RecurrentHead(seed=2) for _ in range(2)]
    step = lambda head: head.update(s['h'], s['joint'], s['legal'], s['logp'], s['adv'][:, 0], s['first'], s['reset'])
    for head in heads:
        step(head)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(heads[0])
    for _ in range(2):
        graph.replay()
        eager = step(heads[1])
    assert torch.equal(captured.loss, eager.loss)
    for k in heads[0].params:
        assert torch.equal(heads[0].params[k], heads[1].params[k]), k


def test_refusals():
    from d1.recurrent import RecurrentHead
    for memory in (0, 12, -8):
        with pytest.raises(ValueError):
            RecurrentHead(memory=memory)
