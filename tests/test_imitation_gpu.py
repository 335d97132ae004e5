"""The joint-action head (d1.imitation): layer norm, GEMM, log-probabilities and
AdamW together, on features of the conv policy and actions of its own head."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def rows():
    from d1.conv_policy import ConvPolicy
    from d1.spec_env import SpecEnv
    n = 2048
    env, pol = SpecEnv(n, seed=3, observe=False), ConvPolicy(seed=1, chunk=1024)
    buf = pol.buffers(n)
    for step in range(20):
        out = pol.act(env.state, env.legal, n, buf, 5, step)
        if step < 19:
            env.step(out['env_action'])
    return buf['h'].clone(), out['joint'].clone(), env.legal.clone()


def test_joint_legal_bits_cover_the_drawn_actions(rows):
    from d1.conv_policy import ENV_ACTION
    from d1.imitation import joint_legal
    h, joint, legal = rows
    bits = joint_legal(legal)
    assert ((bits >> joint.to(torch.int32)) & 1 == 1).all()
    for j, a in enumerate(ENV_ACTION):
        on = (bits >> j) & 1 == 1
        if a < 0:
            assert not on.any()
        else:
            assert ((legal[on].to(torch.int32) >> a) & 1 == 1).all()


def test_gradients_against_autograd(rows):
    """Against torch autograd in fp32 on the same bf16 operands; the kernels round y, the logits, dlogits and dy to
    bf16 (2^-9 each, of sums of terms of both signs): 2e-2 of each gradient's norm."""
    from d1.imitation import JOINT, JointHead, joint_legal
    h, joint, legal = rows
    head = JointHead(seed=2, ent_coef=0.05)
    n = h.shape[0]
    r, saved = head.forward(h, joint, legal, top=3)
    dlogp = torch.full((n,), -1.0 / n, device='cuda')
    dh = head.backward(r, saved, dlogp, torch.full((n,), -0.05 / n, device='cuda'))
    x = h.float().requires_grad_()
    p = {k: t.clone().requires_grad_() for k, t in head.params.items()}
    y = torch.nn.functional.layer_norm(x, (512,), p['norm_w'], p['norm_b'])
    logits = y @ (p['w'] + (head.w.float() - p['w']).detach()).T + p['b']
    bits = joint_legal(legal)[:, None] >> torch.arange(JOINT, device='cuda', dtype=torch.int32)
    lp = logits[:, :JOINT].masked_fill(bits & 1 == 0, -1e9).log_softmax(1)
    ent = -(lp.exp() * lp).sum(1)
    took = lp.gather(1, joint[:, None])[:, 0]
    assert (r.logp - took).abs().max() < 0.05 and (r.entropy - ent).abs().max() < 0.05
    (-took.mean() - 0.05 * ent.mean()).backward()
    for k in p:
        assert (head.grads[k] - p[k].grad).norm() <= 2e-2 * p[k].grad.norm(), k
    assert (dh.float() - x.grad).norm() <= 2e-2 * x.grad.norm()
    tokens, logp = head.alternatives(h, legal, 3)
    assert torch.equal(tokens, r.top_tokens) and torch.equal(logp, r.top_logp)
    assert (logp[:, 0] >= r.logp - 1e-6).all()


@pytest.mark.parametrize('bits', [8, 32])
def test_it_learns_the_actions(rows, bits):
    from d1.imitation import JointHead
    h, joint, legal = rows
    head = JointHead(seed=4, lr=3e-3, state_bits=bits)
    first = float(head.update(h, joint, legal)[0].mean())
    for _ in range(150):
        last = head.update(h, joint, legal)[0]
    last = float(last.mean())
    assert last > first + 0.3, (first, last)
    assert all(t.isfinite().all() for t in head.params.values())
    assert torch.equal(head.w, head.params['w'].bfloat16()) and (head.params['w'][28:] == 0).all()
